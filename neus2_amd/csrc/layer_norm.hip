// Layer norm over rows of 1 to 16384 values, forward and backward.
// What bounds it is memory: forward reads a row and writes one, backward reads two (three with a skip connection) and writes one.  A row
// stays in the registers of the 8 to 1024 lanes that share it, so mean, variance (from the centred values: no cancellation) and result
// come of one reading.  fp16 on an MI355X: 262 144 x 256 forward 49 us (5.5 TB/s, some of it from the last-level cache; a large copy has 4.8), backward with
// a skip connection 107 (5.0), 65 536 x 1024 47 and 115 (5.7, 4.7), 2000 x 16 384 33 and 89 (4.0, 2.9: one workgroup to a CU, whose waves load, wait for the
// row's sums and store together, and sums of 256 rows to join; fp32 52 and 127: 5.0, 4.1).
#include "column_sums.h"

#include <cmath>

namespace {

// LANES lanes share a row, each with CHUNKS vectors of it, LANES vectors apart, one row at a time: with few registers the other waves keep
// memory busy.  (Four rows under way in a lane took, forward, 4.8 us for 3.3 at 300 x 256, 12 for 9.3 at 20 000 x 512, 52.6 for 49 at 262 144 x 256; two,
// backward, 120 for 91 at 65 536 x 1024 and as long at 262 144 x 256.)
template <uint32_t LANES>
constexpr uint32_t threads_of() { return LANES > 256u ? LANES : 256u; }
// sums over the lanes of a row, in all of them
template <uint32_t LANES, uint32_t N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*shared)[N]) {
#pragma unroll
	for (uint32_t k = 0; k < N; ++k) v[k] = n2_lane_sum<(LANES < 64u ? LANES : 64u)>(v[k]);
	if constexpr (LANES > 64u) {
		constexpr uint32_t WAVES = LANES / 64u;
		__syncthreads();  // (the sums before are read)
		if ((threadIdx.x & 63u) == 0u)
#pragma unroll
			for (uint32_t k = 0; k < N; ++k) shared[threadIdx.x >> 6][k] = v[k];
		__syncthreads();
#pragma unroll
		for (uint32_t k = 0; k < N; ++k) {
			if constexpr (WAVES >= 8u) {  // (one value to a lane: sixteen waves' sums of both at once are 32 registers)
				v[k] = n2_lane_sum<WAVES>(shared[threadIdx.x / LANES * WAVES + threadIdx.x % WAVES][k]);
			} else {
				float s = 0.f;
#pragma unroll
				for (uint32_t w = 0; w < WAVES; ++w) s += shared[threadIdx.x / LANES * WAVES + w][k];
				v[k] = s;
			}
		}
	}
}

template <typename T>
__device__ __forceinline__ void as_loaded(N2Vec<T>& v) {
	n2_u32x4 u = __builtin_bit_cast(n2_u32x4, v);
	asm("" : "+v"(u));
	v = __builtin_bit_cast(N2Vec<T>, u);
}

// sum / width to the last bit, where sum * (1 / width) is a step off: rows of equal values have no variance.  (An infinite sum leaves no
// remainder to correct by.)
__device__ __forceinline__ float mean_of(float sum, float width, float inv) {
	const float m = sum * inv;
	return isinf(m) ? m : fmaf(fmaf(-m, width, sum), inv, m);
}

// a lane's weights, zero past the width
template <typename P, uint32_t LANES, uint32_t CHUNKS, uint32_t VEC>
struct Weights {
	P v[CHUNKS][VEC];
	__device__ __forceinline__ Weights(const P* __restrict__ p, uint32_t width, uint32_t lane) {
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC;
			if (at + VEC <= width) {
				__builtin_memcpy(v[c], p + at, sizeof(v[c]));
			} else {
#pragma unroll
				for (uint32_t i = 0; i < VEC; ++i) v[c][i] = at + i < width ? p[at + i] : (P)0.f;
			}
		}
	}
};

template <typename T, typename P, uint32_t LANES, uint32_t CHUNKS>
__global__ void __launch_bounds__(threads_of<LANES>()) layer_norm_forward_kernel(uint32_t n_rows, uint32_t width, float epsilon, const P* __restrict__ scale, const P* __restrict__ shift,
                                                                                  const T* x, uint64_t x_stride, T* y, uint64_t y_stride, float* __restrict__ mean_out,
                                                                                  float* __restrict__ rstd_out) {
	constexpr uint32_t VEC = N2Vec<T>::SIZE, ROWS = threads_of<LANES>() / LANES;
	__shared__ float shared[LANES > 64u ? threads_of<LANES>() / 64u : 1u][1];
	const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
	const float inv = 1.f / (float)width;
	const uint64_t end = (uint64_t)(n_rows - 1u) * x_stride + width;
	const Weights<P, LANES, CHUNKS, VEC> g(scale, width, lane), b(shift, width, lane);
	// (the lanes of a workgroup's last rows stay for the barriers)
	for (uint64_t first = (uint64_t)blockIdx.x * ROWS; first < n_rows; first += (uint64_t)gridDim.x * ROWS) {
		const uint64_t row = first + group;
		N2Vec<T> in[CHUNKS];
		float sum[1] = {0.f};
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC;
			in[c] = n2_load_row(x, row * x_stride + at, end, row < n_rows ? n2_left<T>(width, at) : 0u);
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) sum[0] += (float)in[c].v[i];
		}
		row_sums<LANES>(sum, shared);
		const float mean = mean_of(sum[0], (float)width, inv);
		sum[0] = 0.f;
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c)
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				const float d = (c * LANES + lane) * VEC + i < width ? (float)in[c].v[i] - mean : 0.f;
				sum[0] += d * d;
			}
		row_sums<LANES>(sum, shared);
		const float rstd = rsqrtf(sum[0] * inv + epsilon);
		if (row < n_rows && lane == 0u) {
			if (mean_out != nullptr) mean_out[row] = mean;
			if (rstd_out != nullptr) rstd_out[row] = rstd;
		}
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC;
			N2Vec<T> out;
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) out.v[i] = (T)(((float)in[c].v[i] - mean) * rstd * (float)g.v[c][i] + (float)b.v[c][i]);
			n2_store_vec(y + row * y_stride + at, out, row < n_rows ? n2_left<T>(width, at) : 0u);
		}
	}
}

// Backward: a workgroup takes groups of rows gridDim.x apart and keeps the weights' gradients of its columns in registers; each leaves one
// row of fp32 sums, [blocks][2][width], for n2_column_sums.
template <typename T, typename P, uint32_t LANES, uint32_t CHUNKS>
__global__ void __launch_bounds__(threads_of<LANES>(), LANES <= 512u ? 4 : 1) layer_norm_backward_kernel(uint32_t n_rows, uint32_t width, const P* __restrict__ scale, const T* __restrict__ x, uint64_t x_stride,
                                                                                   const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ dy, uint64_t dy_stride,
                                                                                   const T* skip, uint64_t skip_stride, T* dx, uint64_t dx_stride, float* __restrict__ partial) {
	constexpr uint32_t VEC = N2Vec<T>::SIZE, THREADS = threads_of<LANES>(), ROWS = THREADS / LANES, COLUMNS = LANES * CHUNKS * VEC;
	__shared__ float shared[LANES > 64u ? THREADS / 64u : 1u][2];
	const uint32_t lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
	const float inv = 1.f / (float)width;
	const uint64_t end_x = (uint64_t)(n_rows - 1u) * x_stride + width, end_dy = (uint64_t)(n_rows - 1u) * dy_stride + width, end_skip = (uint64_t)(n_rows - 1u) * skip_stride + width;
	const Weights<P, LANES, CHUNKS, VEC> w(scale, width, lane);
	// (four vectors of weights to a lane do not fit beside their gradients' sums: LDS holds them, each lane's own)
	constexpr bool IN_LDS = CHUNKS > 2u;
	__shared__ alignas(16) P kept[IN_LDS ? CHUNKS : 1u][LANES][VEC];
	if constexpr (IN_LDS)
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) __builtin_memcpy(kept[c][lane], w.v[c], sizeof(w.v[c]));
	auto weights = [&](uint32_t c) __attribute__((always_inline)) -> const P* { return IN_LDS ? kept[c][lane] : w.v[c]; };
	float dscale[CHUNKS][VEC] = {}, dshift[CHUNKS][VEC] = {};
	for (uint64_t first = (uint64_t)blockIdx.x * ROWS; first < n_rows; first += (uint64_t)gridDim.x * ROWS) {
		const uint64_t row = first + group;
		const bool live = row < n_rows;
		const float m = live ? mean[row] : 0.f, s = live ? rstd[row] : 0.f;
		N2Vec<T> in[CHUNKS], g[CHUNKS], early[CHUNKS];
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC, n = live ? n2_left<T>(width, at) : 0u;
			in[c] = n2_load_row(x, row * x_stride + at, end_x, n);
			g[c] = n2_load_row(dy, row * dy_stride + at, end_dy, n);
			early[c] = N2Vec<T>{};  // (of more than one vector the skip connection's come behind the sums: in place too, a lane writes only what it has read)
			if (CHUNKS == 1u && skip != nullptr) early[c] = n2_load_row(skip, row * skip_stride + at, end_skip, n);
		}
		float sum[2] = {0.f, 0.f};
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			// Past the width, and for rows past the last, dy is zero and so is the scale.  The row's values are zero there, too, and mean * rstd may leave fp32
			// where no value's own does: equal values, 1e34 with an epsilon of 1e-12.
			const uint32_t n = n2_left<T>(width, (c * LANES + lane) * VEC);
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				const float xh = i < n ? ((float)in[c].v[i] - m) * s : 0.f, d = (float)g[c].v[i], h = d * (float)weights(c)[i];
				dscale[c][i] += d * xh;
				dshift[c][i] += d;
				sum[0] += h;
				sum[1] += h * xh;
			}
		}
		if (dx == nullptr) continue;
		row_sums<LANES>(sum, shared);
		// (the second half takes the rows' values from the registers they came in: kept as fp32 they would halve the waves, or not fit)
		if constexpr (LANES <= 256u || CHUNKS > 1u)
#pragma unroll
			for (uint32_t c = 0; c < CHUNKS; ++c) as_loaded(in[c]), as_loaded(g[c]);
		const float a = sum[0] * inv, b = sum[1] * inv;
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c) {
			const uint32_t at = (c * LANES + lane) * VEC;
			N2Vec<T> add = early[c];
			if (CHUNKS > 1u && skip != nullptr) add = n2_load_row(skip, row * skip_stride + at, end_skip, live ? n2_left<T>(width, at) : 0u);
			N2Vec<T> out;
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				const float xh = ((float)in[c].v[i] - m) * s, h = (float)g[c].v[i] * (float)weights(c)[i];
				out.v[i] = (T)(s * (h - a - xh * b) + (float)add.v[i]);
			}
			n2_store_vec(dx + row * dx_stride + at, out, live ? n2_left<T>(width, at) : 0u);
		}
	}
	if (partial == nullptr) return;
	// the workgroup's groups of lanes in one row of sums: those of a wave by exchange, the waves through LDS
	if constexpr (ROWS > 1u) {
		constexpr uint32_t PARTS = LANES < 64u ? THREADS / 64u : ROWS;
		__shared__ float fold[PARTS][COLUMNS];
#pragma unroll
		for (uint32_t k = 0; k < 2u; ++k) {
			float(&mine)[CHUNKS][VEC] = k == 0u ? dscale : dshift;
#pragma unroll
			for (uint32_t c = 0; c < CHUNKS; ++c)
#pragma unroll
				for (uint32_t i = 0; i < VEC; ++i) {
#pragma unroll
					for (uint32_t o = LANES; o < 64u; o *= 2u) mine[c][i] += __shfl_xor(mine[c][i], (int)o);
					if (threadIdx.x % 64u < LANES) fold[LANES < 64u ? threadIdx.x / 64u : group][(c * LANES + lane) * VEC + i] = mine[c][i];
				}
			__syncthreads();
			for (uint32_t at = threadIdx.x; at < min(COLUMNS, width); at += THREADS) {
				float sum = 0.f;
#pragma unroll
				for (uint32_t p = 0; p < PARTS; ++p) sum += fold[p][at];
				partial[((uint64_t)blockIdx.x * 2u + k) * width + at] = sum;
			}
			__syncthreads();
		}
	} else {
#pragma unroll
		for (uint32_t c = 0; c < CHUNKS; ++c)
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				const uint32_t at = (c * LANES + lane) * VEC + i;
				if (at >= width) continue;
				partial[(uint64_t)blockIdx.x * 2u * width + at] = dscale[c][i];
				partial[((uint64_t)blockIdx.x * 2u + 1u) * width + at] = dshift[c][i];
			}
	}
}

constexpr uint32_t MAX_WIDTH = 16384;

struct Row {
	uint32_t lanes, chunks;
};
// The fewest lanes that hold a row in one vector each, or in two or four where there are no more lanes to take.  With half the lanes and two vectors
// in each, forward and backward took 59 and 361 us for 53 and 87 at 262 144 x 256, 10.5 and 43 for 8.8 and 18 at 5003 x 1001, 4.7 and 8.0 for 4.6 and 8.0 at
// 1000 x 64 (fp16).
Row row_of(uint32_t width, uint32_t vec) {
	constexpr Row rows[] = {{8, 1}, {16, 1}, {32, 1}, {64, 1}, {128, 1}, {256, 1}, {512, 1}, {1024, 1}, {1024, 2}, {1024, 4}};
	for (const Row& row : rows)
		if (width <= row.lanes * row.chunks * vec) return row;
	return {0, 0};
}

// f(lanes, vectors) for rows in vectors of VEC values
template <uint32_t VEC, typename F>
void with_row(Row row, F&& f) {
	using std::integral_constant;
	auto go = [&](auto lanes, auto chunks) { if (row.lanes == lanes() && row.chunks == chunks()) f(lanes, chunks); };
	go(integral_constant<uint32_t, 8>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 16>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 32>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 64>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 128>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 256>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 512>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 1024>{}, integral_constant<uint32_t, 1>{});
	go(integral_constant<uint32_t, 1024>{}, integral_constant<uint32_t, 2>{});
	if constexpr (1024u * 2u * VEC < MAX_WIDTH) go(integral_constant<uint32_t, 1024>{}, integral_constant<uint32_t, 4>{});
}

template <typename F>
void with_types(n2_dtype dtype, n2_dtype weights, F&& f) {
	if (dtype == N2_DTYPE_F16 && weights == N2_DTYPE_F16) f(n2_f16{}, n2_f16{});
	if (dtype == N2_DTYPE_F16 && weights == N2_DTYPE_F32) f(n2_f16{}, float{});
	if (dtype == N2_DTYPE_BF16 && weights == N2_DTYPE_BF16) f(n2_bf16{}, n2_bf16{});
	if (dtype == N2_DTYPE_BF16 && weights == N2_DTYPE_F32) f(n2_bf16{}, float{});
	if (dtype == N2_DTYPE_F32) f(float{}, float{});
}

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
		with_row<N2Vec<T>::SIZE>(row_of(width, N2Vec<T>::SIZE), [&](auto lanes, auto chunks) {
			constexpr uint32_t LANES = decltype(lanes)::value, THREADS = threads_of<LANES>(), ROWS = THREADS / LANES;
			const uint32_t blocks = n2_layer_norm_forward_blocks(n_rows, ROWS, THREADS);
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
	uint64_t blocks = 0;
	auto count = [&](auto lanes, auto) {
		constexpr uint32_t LANES = decltype(lanes)::value, THREADS = threads_of<LANES>();
		blocks = n2_layer_norm_backward_blocks(n_rows, THREADS / LANES, THREADS);
	};
	if (dtype == N2_DTYPE_F32) with_row<4>(row_of(width, 4), count);
	else with_row<8>(row_of(width, 8), count);
	return 8ull * width * blocks;
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
			with_row<N2Vec<T>::SIZE>(row_of(width, N2Vec<T>::SIZE), [&](auto lanes, auto chunks) {
				constexpr uint32_t LANES = decltype(lanes)::value, THREADS = threads_of<LANES>(), ROWS = THREADS / LANES;
				blocks = n2_layer_norm_backward_blocks(n_rows, ROWS, THREADS);
				layer_norm_backward_kernel<T, P, LANES, decltype(chunks)::value><<<dim3(blocks), dim3(THREADS), 0, s>>>(
					n_rows, width, static_cast<const P*>(d_scale), static_cast<const T*>(d_input), input_stride, d_mean, d_rstd, static_cast<const T*>(d_dL_doutput), dL_doutput_stride,
					static_cast<const T*>(d_dL_dskip), dL_dskip_stride, static_cast<T*>(d_dL_dinput), dL_dinput_stride, weights ? static_cast<float*>(d_workspace) : nullptr);
			});
		});
		N2_LAUNCH_CHECK();
	}
	if (!weights) return N2_OK;
	return n2_column_sums(s, static_cast<const float*>(d_workspace), blocks, width, d_dL_dscale, d_dL_dshift, weights_dtype, mode == N2_GRAD_ACCUMULATE ? 1 : 0);
}
