// Sums over the rows of a matrix of fp32 partial sums, one row from each workgroup of the launch before: the last step of the gradients
// of weights that every row shares.  The order is that of the sizes, whoever comes first.
#pragma once
#include "layer_types.h"

// A run of columns of the partial sums and where their sums go.
struct N2ColumnOutput {
	void* out;           // [columns] of dtype, or null: nothing is stored
	uint32_t first, columns, dtype;
};

template <typename P>
__device__ __forceinline__ void n2_store_sum(P* out, float sum, int accumulate) {
	*out = (P)(accumulate ? (float)*out + sum : sum);
}

// partial: [rows][columns]; the outputs' columns follow each other.  A workgroup takes LANES * WIDE columns by ROWS rows.
template <int N_OUT, uint32_t LANES, uint32_t WIDE, uint32_t ROWS>
__global__ void __launch_bounds__(LANES* ROWS) n2_column_sums_kernel(const float* __restrict__ partial, uint32_t rows, uint32_t columns, N2ColumnOutput first, N2ColumnOutput second,
                                                                      int accumulate) {
	__shared__ float part[ROWS > 1u ? ROWS : 1u][LANES * WIDE + 1u];
	const uint32_t x = threadIdx.x % LANES * WIDE, y = threadIdx.x / LANES, column = blockIdx.x * LANES * WIDE + x;
	float sum[WIDE] = {};
	const uint32_t valid = column < columns ? min(columns - column, WIDE) : 0u;
#pragma unroll 16
	for (uint32_t r = y; r < rows; r += ROWS) {
		float v[WIDE] = {};
		const float* p = partial + (uint64_t)r * columns + column;
		if (valid == WIDE) {
			__builtin_memcpy(v, p, sizeof(v));
		} else {
#pragma unroll
			for (uint32_t i = 0; i < WIDE; ++i) v[i] = i < valid ? p[i] : 0.f;
		}
#pragma unroll
		for (uint32_t i = 0; i < WIDE; ++i) sum[i] += v[i];
	}
	if constexpr (ROWS > 1u) {
#pragma unroll
		for (uint32_t i = 0; i < WIDE; ++i) part[y][x + i] = sum[i];
		__syncthreads();
		for (uint32_t half = ROWS / 2u; half > 0u; half /= 2u) {
			if (y < half)
#pragma unroll
				for (uint32_t i = 0; i < WIDE; ++i) part[y][x + i] += part[y + half][x + i];
			__syncthreads();
		}
		if (y != 0u) return;
#pragma unroll
		for (uint32_t i = 0; i < WIDE; ++i) sum[i] = part[0][x + i];
	}
#pragma unroll
	for (uint32_t i = 0; i < WIDE; ++i) {
		if (i >= valid) break;
		const N2ColumnOutput o = N_OUT > 1 && column + i >= second.first ? second : first;
		const uint32_t at = column + i - o.first;
		if (o.dtype == N2_DTYPE_F16) n2_store_sum(static_cast<n2_f16*>(o.out) + at, sum[i], accumulate);
		else if (o.dtype == N2_DTYPE_BF16) n2_store_sum(static_cast<n2_bf16*>(o.out) + at, sum[i], accumulate);
		else n2_store_sum(static_cast<float*>(o.out) + at, sum[i], accumulate);
	}
}

// Few columns: 64 bytes of a row by 64 rows to a workgroup, with up to 1024 rows at most sixteen loads to a lane, all under way at once; the
// launch takes its latency.  Many columns: 16 bytes a lane, sixteen rows at a time; few rows of them: a lane takes its columns' sums alone.
template <int N_OUT>
static inline int n2_column_sums(hipStream_t s, const float* partial, uint32_t rows, uint32_t columns, const N2ColumnOutput& first, const N2ColumnOutput& second, int accumulate) {
	if (rows <= 16u && columns >= 4096u)
		n2_column_sums_kernel<N_OUT, 256, 4, 1><<<dim3(n2_ceil_div(columns, 1024u)), dim3(256), 0, s>>>(partial, rows, columns, first, second, accumulate);
	else if (columns >= 16384u)
		n2_column_sums_kernel<N_OUT, 16, 4, 16><<<dim3(n2_ceil_div(columns, 64u)), dim3(256), 0, s>>>(partial, rows, columns, first, second, accumulate);
	else
		n2_column_sums_kernel<N_OUT, 16, 1, 64><<<dim3(n2_ceil_div(columns, 16u)), dim3(1024), 0, s>>>(partial, rows, columns, first, second, accumulate);
	N2_LAUNCH_CHECK();
	return N2_OK;
}
