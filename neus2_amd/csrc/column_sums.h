// Sums over the rows of a matrix of fp32 partial sums, one row from each workgroup of the launch before: the last step of the gradients
// of weights that every row shares.  The order is that of the sizes, whoever comes first.
#pragma once
#include "layer_types.h"

template <typename P>
__device__ __forceinline__ void n2_store_sum(P* out, float sum, int accumulate) {
	*out = (P)(accumulate ? (float)*out + sum : sum);
}

// One workgroup of COLUMNS * ROWS lanes: run number `block` of COLUMNS columns of partial [rows][columns].  store(column, sum) is called by one
// lane for each column.
template <uint32_t COLUMNS, uint32_t ROWS, typename F>
__device__ __forceinline__ void n2_column_sums_block(const float* __restrict__ partial, uint32_t rows, uint32_t columns, uint32_t block, F&& store) {
	__shared__ float part[ROWS][COLUMNS + 1u];
	const uint32_t x = threadIdx.x % COLUMNS, y = threadIdx.x / COLUMNS, column = block * COLUMNS + x;
	float sum = 0.f;
#pragma unroll 16
	for (uint32_t r = y; r < rows; r += ROWS) sum += column < columns ? partial[(uint64_t)r * columns + column] : 0.f;
	part[y][x] = sum;
	__syncthreads();
	for (uint32_t half = ROWS / 2u; half > 0u; half /= 2u) {
		if (y < half) part[y][x] += part[y + half][x];
		__syncthreads();
	}
	if (y == 0u && column < columns) store(column, part[0][x]);
}

__device__ __forceinline__ void n2_store_sum(void* out, uint32_t dtype, uint32_t at, float sum, int accumulate) {
	if (dtype == N2_DTYPE_F16) n2_store_sum(static_cast<n2_f16*>(out) + at, sum, accumulate);
	else if (dtype == N2_DTYPE_BF16) n2_store_sum(static_cast<n2_bf16*>(out) + at, sum, accumulate);
	else n2_store_sum(static_cast<float*>(out) + at, sum, accumulate);
}

// columns [0, width) go to `first`, the `width` behind them to `second`
template <uint32_t COLUMNS, uint32_t ROWS>
__global__ void __launch_bounds__(COLUMNS* ROWS) n2_column_sums_kernel(const float* __restrict__ partial, uint32_t rows, uint32_t width, void* first, void* second, uint32_t dtype, int accumulate) {
	n2_column_sums_block<COLUMNS, ROWS>(partial, rows, 2u * width, blockIdx.x, [&](uint32_t column, float sum) {
		n2_store_sum(column < width ? first : second, dtype, column < width ? column : column - width, sum, accumulate);
	});
}

// Two gradients of `width` columns each, side by side in a row of sums.  64 bytes of a row by 64 rows to a workgroup, with up to 1024 rows at
// most sixteen loads to a lane, all under way at once; the launch takes its latency.  (16 bytes a lane and sixteen rows took 24 us more with 1024 rows
// of 2 x 1001 columns, 7 more with 512 of 2 x 4096, as long with 256 of 2 x 8192 and 4 less of 84 with 256 of 2 x 16 384.)
static inline int n2_column_sums(hipStream_t s, const float* partial, uint32_t rows, uint32_t width, void* first, void* second, uint32_t dtype, int accumulate) {
	n2_column_sums_kernel<16, 64><<<dim3(n2_ceil_div(2u * width, 16u)), dim3(1024), 0, s>>>(partial, rows, width, first, second, dtype, accumulate);
	N2_LAUNCH_CHECK();
	return N2_OK;
}
