// The norm over the gradients of many tensors and their clipping: two launches whatever the number of tensors.
// The host cuts the tensors into pieces, about as many as there are workgroups at a time; a launch's workgroups take pieces in turn.  What
// bounds both launches is memory: the first reads every gradient, the second reads and writes it, from the last pieces to the first, so that
// what the first launch read last is still in the caches.  On an MI355X the norm of 139 MB in 60 fp32 tensors takes 24 us (5.8 TB/s), of 800 MB
// in two 142 (5.6); clipping 50 MB into other tensors 28 us for three times as many bytes (5.5), clipping in place where nothing is clipped
// little more than the norm (26 and 146 us); four tensors of 1000 values 4.6 us, the launches.
#include "layer_types.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <new>
#include <vector>

namespace {

struct Piece {
	const void* in;
	void* out;
	uint32_t n, dtype;
	uint64_t unused;
};
static_assert(sizeof(Piece) == 32, "pieces are read by 16 bytes");

constexpr uint32_t THREADS = 256, MAX_BLOCKS = N2_GRADIENTS_WORKSPACE_BYTES / sizeof(double);
// Bytes to a piece: 4 to 64 KB, so that up to 128 MB each of the 2048 workgroups has one piece; beyond, a piece's entry in the table costs little.  Clipping in
// place with pieces up to 16, 32, 64 and 256 KB, us: 60 fp32 tensors, 139 MB, 27.4, 27.3, 26.4, 26.7; 8 fp16 tensors, 160 MB, 30.9, 29.9, 29.6, 29.8; 2 fp32
// tensors, 800 MB, 150, 145, 146, 140.
constexpr uint64_t PIECE_STEP = THREADS * 16, MOST_STEPS = 16;

// Squares are summed in fp64: those of fp32 and bf16 leave fp32's range long before the values do.
template <typename T>
__device__ __forceinline__ double squares(const N2Vec<T>& v) {
	double s = 0.;
#pragma unroll
	for (uint32_t i = 0; i < N2Vec<T>::SIZE; ++i) s = fma((double)(float)v.v[i], (double)(float)v.v[i], s);
	return s;
}

// f(vector, place, valid values) for a lane's vectors of a piece, four loads under way at a time.  (The norm with two, four and eight, us: 40
// fp16 tensors, 8 MB, 6.8, 6.8, 7.6; 60 fp32 tensors, 139 MB, 24.5, 23.7, 23.6; 4 fp32 tensors, 50 MB, 11.8, 12.8, 14.4: the loads of a piece's end are made
// one by one.)
template <typename T, typename F>
__device__ __forceinline__ void each_vector(const Piece& p, F&& f) {
	constexpr uint32_t VEC = N2Vec<T>::SIZE, STEP = THREADS * VEC;
	const T* in = static_cast<const T*>(p.in);
	uint32_t at = threadIdx.x * VEC;
	for (; at + 3u * STEP + VEC <= p.n; at += 4u * STEP) {
		N2Vec<T> v[4];
#pragma unroll
		for (uint32_t i = 0; i < 4u; ++i) __builtin_memcpy(&v[i], in + at + i * STEP, 16);
#pragma unroll
		for (uint32_t i = 0; i < 4u; ++i) f(v[i], at + i * STEP, VEC);
	}
#pragma unroll
	for (uint32_t i = 0; i < 4u; ++i, at += STEP)
		if (at < p.n) f(n2_load_vec(in + at, n2_left<T>(p.n, at)), at, n2_left<T>(p.n, at));
}

template <typename T>
__device__ __forceinline__ double piece_squares(const Piece& p) {
	double s = 0.;
	each_vector<T>(p, [&](const N2Vec<T>& v, uint32_t, uint32_t) __attribute__((always_inline)) { s += squares(v); });
	return s;
}

// times factor * 2^exponent
template <typename T>
__device__ __forceinline__ void piece_scale(const Piece& p, float factor, int exponent) {
	each_vector<T>(p, [&](N2Vec<T> v, uint32_t at, uint32_t n) __attribute__((always_inline)) {
#pragma unroll
		for (uint32_t i = 0; i < N2Vec<T>::SIZE; ++i) v.v[i] = (T)__builtin_amdgcn_ldexpf((float)v.v[i] * factor, exponent);
		n2_store_vec(static_cast<T*>(p.out) + at, v, n);
	});
}

// sum over the workgroup, in all of its lanes
__device__ __forceinline__ double block_sum(double s) {
	__shared__ double part[THREADS / 64];
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
	__syncthreads();
	if ((threadIdx.x & 63u) == 0u) part[threadIdx.x >> 6] = s;
	__syncthreads();
	return (part[0] + part[1]) + (part[2] + part[3]);
}

__global__ void __launch_bounds__(THREADS) gradient_squares_kernel(const Piece* __restrict__ pieces, uint32_t n_pieces, double* __restrict__ partial) {
	double s = 0.;
	for (uint32_t i = blockIdx.x; i < n_pieces; i += gridDim.x) {
		const Piece p = pieces[i];
		s += p.dtype == N2_DTYPE_F16 ? piece_squares<n2_f16>(p) : p.dtype == N2_DTYPE_BF16 ? piece_squares<n2_bf16>(p) : piece_squares<float>(p);
	}
	s = block_sum(s);
	if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double norm_of(const double* __restrict__ partial, uint32_t n_partial, double loss_scale) {
	double s = 0.;
#pragma unroll
	for (uint32_t k = 0; k < MAX_BLOCKS / THREADS; ++k) {
		const uint32_t i = k * THREADS + threadIdx.x;
		s += i < n_partial ? partial[i] : 0.;
	}
	return sqrt(block_sum(s)) / loss_scale;
}

__global__ void __launch_bounds__(THREADS) gradient_norm_kernel(const double* __restrict__ partial, uint32_t n_partial, float loss_scale, float* __restrict__ norm) {
	const double n = norm_of(partial, n_partial, (double)loss_scale);
	if (threadIdx.x == 0) *norm = (float)n;
}

// Every workgroup forms the norm itself, from the same sums in the same order.
__global__ void __launch_bounds__(THREADS) gradient_clip_kernel(const Piece* __restrict__ pieces, uint32_t n_pieces, const double* __restrict__ partial, uint32_t n_partial, float max_norm,
                                                                float loss_scale, float* __restrict__ norm) {
	const double n = norm_of(partial, n_partial, (double)loss_scale), ratio = (double)max_norm / (n + 1e-6);
	float factor = ratio > 1. ? 1.f : (float)ratio;  // (no number stays none)
	int exponent = 0;
	if (factor < FLT_MIN && ratio > 0.) factor = (float)frexp(ratio, &exponent);  // (no normal number of fp32, where its products may be)
	if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
	for (uint32_t i = blockIdx.x; i < n_pieces; i += gridDim.x) {
		const Piece p = pieces[n_pieces - 1u - i];
		if (p.in == p.out && factor == 1.f) continue;
		if (p.dtype == N2_DTYPE_F16) piece_scale<n2_f16>(p, factor, exponent);
		else if (p.dtype == N2_DTYPE_BF16) piece_scale<n2_bf16>(p, factor, exponent);
		else piece_scale<float>(p, factor, exponent);
	}
}

// values to a piece of a tensor of this type where all tensors have so many bytes
uint64_t piece_values(uint64_t all_bytes, uint32_t dtype) {
	const uint64_t steps = std::min<uint64_t>(std::max<uint64_t>((all_bytes + MAX_BLOCKS * PIECE_STEP - 1) / (MAX_BLOCKS * PIECE_STEP), 1), MOST_STEPS);
	return steps * PIECE_STEP / n2_dtype_bytes(dtype);
}
uint64_t all_bytes_of(uint32_t n_tensors, const n2_gradient_tensor* tensors) {
	uint64_t bytes = 0;
	for (uint32_t i = 0; i < n_tensors; ++i) bytes += std::min<uint64_t>(tensors[i].n, 1ull << 38) * n2_dtype_bytes(tensors[i].dtype);
	return bytes;
}

}  // namespace

struct n2_gradients {
	const Piece* table = nullptr;
	uint32_t n_pieces = 0, blocks = 0;
};

N2_API uint64_t n2_gradients_table_bytes(uint32_t n_tensors, const n2_gradient_tensor* tensors) {
	if (n_tensors > 0 && tensors == nullptr) return 0;
	uint64_t pieces = 0;
	const uint64_t all = all_bytes_of(n_tensors, tensors);
	for (uint32_t i = 0; i < n_tensors; ++i) {
		const uint64_t values = piece_values(all, tensors[i].dtype);
		pieces += tensors[i].n / values + (tensors[i].n % values != 0);
	}
	return std::max<uint64_t>(pieces, 1) * sizeof(Piece);
}

N2_API int n2_gradients_create(n2_stream_t stream, uint32_t n_tensors, const n2_gradient_tensor* tensors, void* d_table, uint64_t table_bytes, n2_gradients_t** out) {
	N2_REQUIRE(out != nullptr, "n2_gradients_create: out is null");
	*out = nullptr;
	N2_REQUIRE(n_tensors == 0 || tensors != nullptr, "n2_gradients_create: null tensors");
	N2_REQUIRE(n_tensors < (1u << 24), "n2_gradients_create: %u tensors", n_tensors);
	try {
		struct Range { uintptr_t begin, end; };
		std::vector<Range> ranges;
		std::vector<Piece> pieces;
		const uint64_t all = all_bytes_of(n_tensors, tensors);
		for (uint32_t i = 0; i < n_tensors; ++i) {
			const n2_gradient_tensor& t = tensors[i];
			N2_REQUIRE(t.dtype <= N2_DTYPE_F32, "n2_gradients_create: tensor %u has type %u", i, t.dtype);
			if (t.n == 0) continue;
			const uint64_t bytes = n2_dtype_bytes(t.dtype);
			N2_REQUIRE(t.d_gradients && t.d_out, "n2_gradients_create: tensor %u is null", i);
			N2_REQUIRE(t.n < (1ull << 38), "n2_gradients_create: tensor %u has %llu values", i, (unsigned long long)t.n);
			N2_REQUIRE((reinterpret_cast<uintptr_t>(t.d_gradients) | reinterpret_cast<uintptr_t>(t.d_out)) % bytes == 0, "n2_gradients_create: tensor %u is not aligned to its type", i);
			const uintptr_t in = reinterpret_cast<uintptr_t>(t.d_gradients), to = reinterpret_cast<uintptr_t>(t.d_out);
			ranges.push_back({in, in + t.n * bytes});
			if (to != in) ranges.push_back({to, to + t.n * bytes});
			const uint64_t values = piece_values(all, t.dtype);
			for (uint64_t at = 0; at < t.n; at += values)
				pieces.push_back({static_cast<const char*>(t.d_gradients) + at * bytes, static_cast<char*>(t.d_out) + at * bytes, (uint32_t)std::min<uint64_t>(values, t.n - at), t.dtype, 0});
		}
		std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
		for (size_t i = 1; i < ranges.size(); ++i) N2_REQUIRE(ranges[i].begin >= ranges[i - 1].end, "n2_gradients_create: two of the tensors overlap");
		const uint64_t needed = std::max<uint64_t>(pieces.size(), 1) * sizeof(Piece);
		N2_REQUIRE(pieces.size() < (1ull << 31), "n2_gradients_create: too many values");
		N2_REQUIRE(d_table && reinterpret_cast<uintptr_t>(d_table) % 16 == 0 && table_bytes >= needed, "n2_gradients_create: needs a 16-byte aligned table of %llu bytes, got %llu",
		           (unsigned long long)needed, (unsigned long long)table_bytes);
		if (!pieces.empty()) {
			hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
			N2_HIP(hipStreamIsCapturing(n2_stream(stream), &capturing));
			N2_REQUIRE(capturing == hipStreamCaptureStatusNone, "n2_gradients_create: the stream is being captured");
		}
		n2_gradients* g = new n2_gradients();
		g->table = static_cast<const Piece*>(d_table);
		g->n_pieces = (uint32_t)pieces.size();
		g->blocks = std::min<uint32_t>(g->n_pieces, MAX_BLOCKS);
		if (!pieces.empty()) {
			hipError_t e = hipMemcpyAsync(d_table, pieces.data(), needed, hipMemcpyHostToDevice, n2_stream(stream));
			if (e == hipSuccess) e = hipStreamSynchronize(n2_stream(stream));
			if (e != hipSuccess) {
				delete g;
				n2_set_error("n2_gradients_create: %s", hipGetErrorString(e));
				return N2_ERR_HIP;
			}
		}
		*out = g;
		return N2_OK;
	} catch (const std::bad_alloc&) {
		n2_set_error("n2_gradients_create: out of host memory");
		return N2_ERR_INVALID_ARGUMENT;
	}
}

N2_API void n2_gradients_destroy(n2_gradients_t* gradients) { delete gradients; }

static int launch_squares(const n2_gradients_t* g, n2_stream_t stream, float loss_scale, float* d_norm, void* d_workspace, uint64_t workspace_bytes, const char* name) {
	N2_REQUIRE(g != nullptr && d_norm != nullptr, "%s: null argument", name);
	N2_REQUIRE(std::isfinite(loss_scale) && loss_scale > 0.f, "%s: loss_scale must be positive", name);
	N2_REQUIRE(d_workspace && reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0 && workspace_bytes >= N2_GRADIENTS_WORKSPACE_BYTES, "%s: needs a 16-byte aligned workspace of %u bytes, got %llu",
	           name, N2_GRADIENTS_WORKSPACE_BYTES, (unsigned long long)workspace_bytes);
	if (g->blocks > 0) {
		gradient_squares_kernel<<<dim3(g->blocks), dim3(THREADS), 0, n2_stream(stream)>>>(g->table, g->n_pieces, static_cast<double*>(d_workspace));
		N2_LAUNCH_CHECK();
	}
	return N2_OK;
}

N2_API int n2_gradients_norm(const n2_gradients_t* gradients, n2_stream_t stream, float loss_scale, float* d_norm, void* d_workspace, uint64_t workspace_bytes) {
	if (const int rc = launch_squares(gradients, stream, loss_scale, d_norm, d_workspace, workspace_bytes, "n2_gradients_norm")) return rc;
	gradient_norm_kernel<<<dim3(1), dim3(THREADS), 0, n2_stream(stream)>>>(static_cast<const double*>(d_workspace), gradients->blocks, loss_scale, d_norm);
	N2_LAUNCH_CHECK();
	return N2_OK;
}

N2_API int n2_gradients_clip(const n2_gradients_t* gradients, n2_stream_t stream, float max_norm, float loss_scale, float* d_norm, void* d_workspace, uint64_t workspace_bytes) {
	N2_REQUIRE(max_norm >= 0.f, "n2_gradients_clip: max_norm %g must not be negative", (double)max_norm);
	if (const int rc = launch_squares(gradients, stream, loss_scale, d_norm, d_workspace, workspace_bytes, "n2_gradients_clip")) return rc;
	gradient_clip_kernel<<<dim3(std::max(gradients->blocks, 1u)), dim3(THREADS), 0, n2_stream(stream)>>>(gradients->table, gradients->n_pieces, static_cast<const double*>(d_workspace),
		gradients->blocks, max_norm, loss_scale, d_norm);
	N2_LAUNCH_CHECK();
	return N2_OK;
}
