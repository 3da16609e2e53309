// Layer norm over rows of 1 to 16384 values, forward and backward.
// What bounds it is memory: forward reads a row and writes one, backward reads two (three with a skip connection) and writes one.  A row
// stays in the registers of the 8 to 1024 lanes that share it, so mean, variance (from the centred values: no cancellation) and result
// come of one reading.
#include "column_sums.h"

#include <cmath>

namespace {

// LANES lanes share a row, each with CHUNKS vectors of it, LANES vectors apart.
template <uint32_t LANES>
constexpr uint32_t threads_of() { return LANES > 256u ? LANES : 256u; }

// sum over the lanes of a row, in all of them
template <uint32_t LANES, uint32_t N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*shared)[N]) {
#pragma unroll
	for (uint32_t o = min(LANES, 64u) / 2u; o > 0u; o /= 2u)
#pragma unroll
		for (uint32_t k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], (int)o);
	if constexpr (LANES > 64u) {
		constexpr uint32_t WAVES = LANES / 64u;
		__syncthreads();  // (the sums before are read)
		if ((threadIdx.x & 63u) == 0u)
#pragma unroll
			for (uint32_t k = 0; k < N; ++k) shared[threadIdx.x >> 6][k] = v[k];
		__syncthreads();
#pragma unroll
		for (uint32_t k = 0; k < N; ++k) {
			float s = 0.f;
#pragma unroll
			for (uint32_t w = 0; w < WAVES; ++w) s += shared[w][k];
			v[k] = s;
		}
	}
}

// sum / width to the last bit, where sum * (1 / width) is a step off: rows of equal values have no variance
__device__ __forceinline__ float mean_of(float sum, float width, float inv) {
	const float m = sum * inv;
	return fmaf(fmaf(-m, width, sum), inv, m);
}

template <typename T, typename P, uint32_t LANES, uint32_t CHUNKS>
__global__ void __launch_bounds__(threads_of<LANES>()) layer_norm_forward_kernel(uint32_t n_rows, uint32_t width, float epsilon, const P* __restrict__ scale, const P* __restrict__ shift,
                                                                                  const T* x, uint64_t x_stride, T* y, uint64_t y_stride, float* __restrict__ mean_out,
                                                                                  float* __restrict__ rstd_out) {
	constexpr uint32_t VEC = N2Vec<T>::SIZE, ROWS = threads_of<LANES>() / LANES;
	__shared__ float shared[LANES > 64u ? LANES / 64u : 1u][1];
	const uint32_t lane = threadIdx.x % LANES;
	const float inv = 1.f / (float)width;
	for (uint64_t row = (uint64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row - threadIdx.x / LANES < n_rows; row += (uint64_t)gridDim.x * ROWS) {
		const bool live = row < n_rows;  // (the lanes of a workgroup's last rows stay for the barriers)
		float v[CHUNKS][VEC], sum[1] = {0.f};
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC, n = live ? n2_left<T>(width, at) : 0u;
			const N2Vec<T> in = n2_load_vec(x + row * x_stride + at, n);
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) v[c][i] = (float)in.v[i], sum[0] += v[c][i];
		}
		row_sums<LANES>(sum, shared);
		const float mean = mean_of(sum[0], (float)width, inv);
		sum[0] = 0.f;
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC;
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				v[c][i] = at + i < width ? v[c][i] - mean : 0.f;
				sum[0] += v[c][i] * v[c][i];
			}
		}
		row_sums<LANES>(sum, shared);
		const float rstd = rsqrtf(sum[0] * inv + epsilon);
		if (live && lane == 0u) {
			if (mean_out != nullptr) mean_out[row] = mean;
			if (rstd_out != nullptr) rstd_out[row] = rstd;
		}
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC, n = live ? n2_left<T>(width, at) : 0u;
			N2Vec<T> out;
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) out.v[i] = i < n ? (T)(v[c][i] * rstd * (float)scale[at + i] + (float)shift[at + i]) : (T)0.f;
			n2_store_vec(y + row * y_stride + at, out, n);
		}
	}
}

// Backward: a workgroup takes rows gridDim.x apart and keeps the weights' gradients of its columns in registers; each leaves one row of
// fp32 sums, [blocks][2][width], for n2_column_sums_kernel.
template <typename T, typename P, uint32_t LANES, uint32_t CHUNKS>
__global__ void __launch_bounds__(threads_of<LANES>()) layer_norm_backward_kernel(uint32_t n_rows, uint32_t width, const P* __restrict__ scale, const T* __restrict__ x, uint64_t x_stride,
                                                                                   const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ dy, uint64_t dy_stride,
                                                                                   const T* skip, uint64_t skip_stride, T* dx, uint64_t dx_stride, float* __restrict__ partial) {
	constexpr uint32_t VEC = N2Vec<T>::SIZE, THREADS = threads_of<LANES>(), ROWS = THREADS / LANES, COLUMNS = LANES * CHUNKS * VEC;
	__shared__ float shared[LANES > 64u ? LANES / 64u : 1u][2];
	const uint32_t lane = threadIdx.x % LANES;
	const float inv = 1.f / (float)width;
	float dscale[CHUNKS][VEC] = {}, dshift[CHUNKS][VEC] = {};
	for (uint64_t row = (uint64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row - threadIdx.x / LANES < n_rows; row += (uint64_t)gridDim.x * ROWS) {
		const bool live = row < n_rows;
		const float m = live ? mean[row] : 0.f, r = live ? rstd[row] : 0.f;
		float xh[CHUNKS][VEC], h[CHUNKS][VEC], sum[2] = {0.f, 0.f};
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC, n = live ? n2_left<T>(width, at) : 0u;
			const N2Vec<T> in = n2_load_vec(x + row * x_stride + at, n), g = n2_load_vec(dy + row * dy_stride + at, n);
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				xh[c][i] = i < n ? ((float)in.v[i] - m) * r : 0.f;
				h[c][i] = (float)g.v[i];
				dscale[c][i] += h[c][i] * xh[c][i];
				dshift[c][i] += h[c][i];
				h[c][i] *= i < n ? (float)scale[at + i] : 0.f;
				sum[0] += h[c][i];
				sum[1] += h[c][i] * xh[c][i];
			}
		}
		if (dx == nullptr) continue;
		row_sums<LANES>(sum, shared);
		const float a = sum[0] * inv, b = sum[1] * inv;
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC, n = live ? n2_left<T>(width, at) : 0u;
			N2Vec<T> out = {}, add = {};
			if (skip != nullptr) add = n2_load_vec(skip + row * skip_stride + at, n);
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) out.v[i] = (T)(r * (h[c][i] - a - xh[c][i] * b) + (float)add.v[i]);
			n2_store_vec(dx + row * dx_stride + at, out, n);
		}
	}
	if (partial == nullptr) return;
	// the workgroup's rows of lanes, one after the other, in one row of sums
	__shared__ float fold[ROWS > 1u ? COLUMNS : 1u];
#pragma unroll
	for (uint32_t k = 0; k < 2u; ++k) {
		float(&mine)[CHUNKS][VEC] = k == 0u ? dscale : dshift;
		if constexpr (ROWS > 1u) {
			for (uint32_t turn = ROWS - 1u; turn > 0u; --turn) {
				if (threadIdx.x / LANES == turn)
#pragma unroll
					for (uint32_t c = 0; c < CHUNKS; ++c)
#pragma unroll
						for (uint32_t i = 0; i < VEC; ++i) {
							float& f = fold[(c * LANES + lane) * VEC + i];
							f = turn == ROWS - 1u ? mine[c][i] : f + mine[c][i];
						}
				__syncthreads();
			}
		}
		if (threadIdx.x / LANES == 0u)
#pragma unroll
			for (uint32_t c = 0; c < CHUNKS; ++c)
#pragma unroll
				for (uint32_t i = 0; i < VEC; ++i) {
					const uint32_t at = (c * LANES + lane) * VEC + i;
					if (at < width) partial[((uint64_t)blockIdx.x * 2u + k) * width + at] = ROWS > 1u ? mine[c][i] + fold[at] : mine[c][i];
				}
		if constexpr (ROWS > 1u) __syncthreads();
	}
}

struct Row {
	uint32_t lanes, chunks;
};
// the fewest lanes that hold a row, one vector each up to 64 lanes, then up to four
Row row_of(uint32_t width, uint32_t vec) {
	for (uint32_t lanes = 8; lanes <= 64; lanes *= 2)
		if (width <= lanes * vec) return {lanes, 1};
	for (uint32_t lanes : {64u, 256u, 1024u})
		for (uint32_t chunks : {2u, 4u})
			if (width <= lanes * chunks * vec) return {lanes, chunks};
	return {0, 0};
}

template <typename F>
void with_row(Row row, F&& f) {
	using std::integral_constant;
	auto go = [&](auto lanes, auto chunks) { if (row.lanes == lanes() && row.chunks == chunks()) f(lanes, chunks); };
	go(integral_constant<uint32_t, 8>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 16>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 32>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 64>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 64>{}, integral_constant<uint32_t, 2>{});
	go(integral_constant<uint32_t, 64>{}, integral_constant<uint32_t, 4>{});
	go(integral_constant<uint32_t, 256>{}, integral_constant<uint32_t, 2>{});
	go(integral_constant<uint32_t, 256>{}, integral_constant<uint32_t, 4>{});
	go(integral_constant<uint32_t, 1024>{}, integral_constant<uint32_t, 2>{});
	go(integral_constant<uint32_t, 1024>{}, integral_constant<uint32_t, 4>{});
}

template <typename F>
void with_types(n2_dtype dtype, n2_dtype weights, F&& f) {
	if (dtype == N2_DTYPE_F16 && weights == N2_DTYPE_F16) f(n2_f16{}, n2_f16{});
	if (dtype == N2_DTYPE_F16 && weights == N2_DTYPE_F32) f(n2_f16{}, float{});
	if (dtype == N2_DTYPE_BF16 && weights == N2_DTYPE_BF16) f(n2_bf16{}, n2_bf16{});
	if (dtype == N2_DTYPE_BF16 && weights == N2_DTYPE_F32) f(n2_bf16{}, float{});
	if (dtype == N2_DTYPE_F32) f(float{}, float{});
}

constexpr uint32_t MAX_WIDTH = 16384;

bool known(n2_dtype t) { return t == N2_DTYPE_F16 || t == N2_DTYPE_BF16 || t == N2_DTYPE_F32; }

}  // namespace

#define NORM_CHECKS(name)                                                                                                                                       \
	N2_REQUIRE(known(dtype) && (weights_dtype == dtype || weights_dtype == N2_DTYPE_F32), name ": rows of type %d with weights of type %d", (int)dtype, (int)weights_dtype); \
	N2_REQUIRE(width >= 1 && width <= MAX_WIDTH, name ": width %u outside [1, %u]", width, MAX_WIDTH)

N2_API int n2_layer_norm_forward(n2_stream_t stream, n2_dtype dtype, n2_dtype weights_dtype, uint32_t n_rows, uint32_t width, float epsilon, const void* d_scale,
                                 const void* d_shift, const void* d_input, uint64_t input_stride, void* d_output, uint64_t output_stride, float* d_mean, float* d_rstd) {
	NORM_CHECKS("n2_layer_norm_forward");
	N2_REQUIRE(std::isfinite(epsilon) && epsilon > 0.f, "n2_layer_norm_forward: epsilon %g must be positive", (double)epsilon);
	if (n_rows == 0) return N2_OK;
	N2_REQUIRE(d_scale && d_shift && d_input && d_output, "n2_layer_norm_forward: null buffer");
	N2_REQUIRE(n_rows == 1 || (input_stride >= width && output_stride >= width), "n2_layer_norm_forward: a row stride below the width %u", width);
	N2_REQUIRE(n_rows == 1 || (n2_rows_fit(n_rows, input_stride) && n2_rows_fit(n_rows, output_stride)), "n2_layer_norm_forward: a row stride beyond memory");
	const uint32_t bytes = n2_dtype_bytes(dtype), weight_bytes = n2_dtype_bytes(weights_dtype);
	const N2Rows written[3] = {n2_rows(d_output, n_rows, width, output_stride, bytes), n2_vector(d_mean, n_rows, 4), n2_vector(d_rstd, n_rows, 4)};
	const N2Rows read[3] = {n2_rows(d_input, n_rows, width, input_stride, bytes), n2_vector(d_scale, width, weight_bytes), n2_vector(d_shift, width, weight_bytes)};
	N2_REQUIRE(!n2_overlap(written, read), "n2_layer_norm_forward: an output overlaps another buffer");
	with_types(dtype, weights_dtype, [&](auto t, auto p) {
		using T = decltype(t);
		using P = decltype(p);
		with_row(row_of(width, N2Vec<T>::SIZE), [&](auto lanes, auto chunks) {
			constexpr uint32_t LANES = decltype(lanes)::value, THREADS = threads_of<LANES>(), ROWS = THREADS / LANES;
			const uint32_t blocks = n2_layer_norm_blocks(n_rows, ROWS, THREADS);
			layer_norm_forward_kernel<T, P, LANES, decltype(chunks)::value><<<dim3(blocks), dim3(THREADS), 0, n2_stream(stream)>>>(
				n_rows, width, epsilon, static_cast<const P*>(d_scale), static_cast<const P*>(d_shift), static_cast<const T*>(d_input), input_stride, static_cast<T*>(d_output),
				output_stride, d_mean, d_rstd);
		});
	});
	N2_LAUNCH_CHECK();
	return N2_OK;
}

N2_API uint64_t n2_layer_norm_workspace_bytes(n2_dtype dtype, uint32_t n_rows, uint32_t width) {
	if (!known(dtype) || width < 1 || width > MAX_WIDTH) return 0;
	const Row row = row_of(width, 16u / n2_dtype_bytes(dtype));
	const uint32_t threads = row.lanes > 256u ? row.lanes : 256u;
	return 8ull * width * n2_layer_norm_blocks(n_rows, threads / row.lanes, threads);
}

N2_API int n2_layer_norm_backward(n2_stream_t stream, n2_dtype dtype, n2_dtype weights_dtype, uint32_t n_rows, uint32_t width, const void* d_scale, const void* d_input,
                                  uint64_t input_stride, const float* d_mean, const float* d_rstd, const void* d_dL_doutput, uint64_t dL_doutput_stride,
                                  const void* d_dL_dskip, uint64_t dL_dskip_stride, void* d_dL_dinput, uint64_t dL_dinput_stride, void* d_dL_dscale, void* d_dL_dshift,
                                  n2_grad_mode mode, void* d_workspace, uint64_t workspace_bytes) {
	NORM_CHECKS("n2_layer_norm_backward");
	N2_REQUIRE(mode == N2_GRAD_IGNORE || mode == N2_GRAD_OVERWRITE || mode == N2_GRAD_ACCUMULATE, "n2_layer_norm_backward: gradient mode %d", (int)mode);
	const bool weights = mode != N2_GRAD_IGNORE;
	const uint32_t bytes = n2_dtype_bytes(dtype), weight_bytes = n2_dtype_bytes(weights_dtype);
	if (weights) N2_REQUIRE(d_dL_dscale && d_dL_dshift, "n2_layer_norm_backward: null weight gradients");
	if (n_rows > 0) {
		N2_REQUIRE(d_scale && d_input && d_mean && d_rstd && d_dL_doutput, "n2_layer_norm_backward: null buffer");
		N2_REQUIRE(n_rows == 1 || (input_stride >= width && dL_doutput_stride >= width && (!d_dL_dskip || dL_dskip_stride >= width) && (!d_dL_dinput || dL_dinput_stride >= width)),
		           "n2_layer_norm_backward: a row stride below the width %u", width);
		N2_REQUIRE(n_rows == 1 || (n2_rows_fit(n_rows, input_stride) && n2_rows_fit(n_rows, dL_doutput_stride) && (!d_dL_dskip || n2_rows_fit(n_rows, dL_dskip_stride)) &&
		                           (!d_dL_dinput || n2_rows_fit(n_rows, dL_dinput_stride))),
		           "n2_layer_norm_backward: a row stride beyond memory");
	}
	const uint64_t needed = n2_layer_norm_workspace_bytes(dtype, n_rows, width);
	if (weights && n_rows > 0)
		N2_REQUIRE(d_workspace && reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0 && workspace_bytes >= needed, "n2_layer_norm_backward: needs a 16-byte aligned workspace of %llu bytes, got %llu",
		           (unsigned long long)needed, (unsigned long long)workspace_bytes);
	const bool skip_in_place = d_dL_dskip == d_dL_dinput && (n_rows <= 1 || dL_dskip_stride == dL_dinput_stride);
	const N2Rows written[4] = {n2_rows(d_dL_dinput, n_rows, width, dL_dinput_stride, bytes), n2_vector(weights ? d_dL_dscale : nullptr, width, weight_bytes),
	                           n2_vector(weights ? d_dL_dshift : nullptr, width, weight_bytes), n2_vector(weights ? d_workspace : nullptr, needed, 1)};
	const N2Rows read[6] = {n2_rows(d_input, n_rows, width, input_stride, bytes), n2_rows(d_dL_doutput, n_rows, width, dL_doutput_stride, bytes), n2_vector(d_scale, width, weight_bytes),
	                        n2_vector(d_mean, n_rows, 4), n2_vector(d_rstd, n_rows, 4), n2_rows(skip_in_place ? nullptr : d_dL_dskip, n_rows, width, dL_dskip_stride, bytes)};
	N2_REQUIRE(!n2_overlap(written, read), "n2_layer_norm_backward: an output overlaps another buffer");
	hipStream_t s = n2_stream(stream);
	uint32_t blocks = 0;
	if (n_rows > 0 && (weights || d_dL_dinput != nullptr)) {
		with_types(dtype, weights_dtype, [&](auto t, auto p) {
			using T = decltype(t);
			using P = decltype(p);
			with_row(row_of(width, N2Vec<T>::SIZE), [&](auto lanes, auto chunks) {
				constexpr uint32_t LANES = decltype(lanes)::value, THREADS = threads_of<LANES>(), ROWS = THREADS / LANES;
				blocks = n2_layer_norm_blocks(n_rows, ROWS, THREADS);
				layer_norm_backward_kernel<T, P, LANES, decltype(chunks)::value><<<dim3(blocks), dim3(THREADS), 0, s>>>(
					n_rows, width, static_cast<const P*>(d_scale), static_cast<const T*>(d_input), input_stride, d_mean, d_rstd, static_cast<const T*>(d_dL_doutput), dL_doutput_stride,
					static_cast<const T*>(d_dL_dskip), dL_dskip_stride, static_cast<T*>(d_dL_dinput), dL_dinput_stride, weights ? static_cast<float*>(d_workspace) : nullptr);
			});
		});
		N2_LAUNCH_CHECK();
	}
	if (!weights) return N2_OK;
	const N2ColumnOutput scale_out = {d_dL_dscale, 0, width, (uint32_t)weights_dtype}, shift_out = {d_dL_dshift, width, width, (uint32_t)weights_dtype};
	return n2_column_sums<2>(s, static_cast<const float*>(d_workspace), blocks, 2u * width, scale_out, shift_out, mode == N2_GRAD_ACCUMULATE ? 1 : 0);
}
