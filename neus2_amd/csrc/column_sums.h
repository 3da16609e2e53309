// Sums over the rows of a matrix of fp32 partial sums, one row from each workgroup of the launch before: the last step of the gradients
// of weights that every row shares.  The order is that of the sizes, whoever comes first.
#pragma once
#include "layer_types.h"

// 16 columns (64 bytes of a row) by 64 rows to a workgroup: with up to 1024 rows every lane has at most sixteen loads, all under way
// at once, and what the launch takes is its latency.
constexpr uint32_t N2_SUM_COLUMNS = 16, N2_SUM_ROWS = 64;

// A run of columns of the partial sums and where their sums go.
struct N2ColumnOutput {
	void* out;           // [columns] of dtype, or null: nothing is stored
	uint32_t first, columns, dtype;
};

template <typename P>
__device__ __forceinline__ void n2_store_sum(P* out, float sum, int accumulate) {
	*out = (P)(accumulate ? (float)*out + sum : sum);
}

// partial: [rows][pitch]; the outputs' columns do not overlap
template <int N_OUT>
__global__ void __launch_bounds__(N2_SUM_COLUMNS* N2_SUM_ROWS) n2_column_sums_kernel(const float* __restrict__ partial, uint32_t rows, uint64_t pitch, uint32_t columns,
                                                                                      N2ColumnOutput first, N2ColumnOutput second, int accumulate) {
	__shared__ float part[N2_SUM_ROWS][N2_SUM_COLUMNS + 1];
	const uint32_t x = threadIdx.x % N2_SUM_COLUMNS, y = threadIdx.x / N2_SUM_COLUMNS, column = blockIdx.x * N2_SUM_COLUMNS + x;
	float sum = 0.f;
	if (column < columns) {
#pragma unroll 16
		for (uint32_t r = y; r < rows; r += N2_SUM_ROWS) sum += partial[r * pitch + column];
	}
	part[y][x] = sum;
	__syncthreads();
	for (uint32_t half = N2_SUM_ROWS / 2; half > 0; half /= 2) {
		if (y < half) part[y][x] += part[y + half][x];
		__syncthreads();
	}
	if (y != 0 || column >= columns) return;
	const N2ColumnOutput o = N_OUT > 1 && column >= second.first ? second : first;
	if (o.out == nullptr || column < o.first || column >= o.first + o.columns) return;
	const uint32_t at = column - o.first;
	if (o.dtype == N2_DTYPE_F16) n2_store_sum(static_cast<n2_f16*>(o.out) + at, part[0][x], accumulate);
	else if (o.dtype == N2_DTYPE_BF16) n2_store_sum(static_cast<n2_bf16*>(o.out) + at, part[0][x], accumulate);
	else n2_store_sum(static_cast<float*>(o.out) + at, part[0][x], accumulate);
}
