// Linear layers of any width: y = act(x W^T + b) + r, and the two products of the backward pass, dx = dz W and dW = dz^T x.
// One kernel serves the three products, C[m][n] = sum_k A(m, k) B(n, k), with each operand either contiguous in k (rows of x, W, dz as they
// stand) or in its own index (W in dx, dz and x in dW): such a tile goes into LDS as it stands in memory and is turned around on the way
// into the registers (ds_read_b64_tr_b16), so nothing is transposed in memory.
#include "column_sums.h"

#include <type_traits>

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(n2_f16, s16x8 a, s16x8 b, f32x4 c) {
	return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(n2_bf16, s16x8 a, s16x8 b, f32x4 c) {
	return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// exp2 and the reciprocal are the hardware's, within a step of fp32; what the exponent's rounding adds to exp(-|z|) is below 2^-24 |z| of it.
// exp(-|z|) is a square, since exp2 gives zero below 2^-126 (|z| above 87.3), where z times it is a number of bf16 still (down to -92, and less exactly to -97).  (Without the square
// 2^18 x 256 x 256 takes 73.5 us for 75.5, backward 198 for 200.)
__device__ __forceinline__ float exp_minus_abs(float z) {
	const float h = __builtin_amdgcn_exp2f(fabsf(z) * -0.72134752044448170f);
	return h * h;
}
// erfc(|z| / sqrt(2)) / 2 = q g^2 with g = exp(-z^2 / 4), squared last: exp2 gives zero below 2^-126, where the values are still bf16's.  q = t P(t), t = 1 / (1 + 0.305 |z|); P is
// the polynomial of degree 7 whose largest relative error on 0 <= |z| <= 14.6 is the least, 8.9e-8 (by linear programming over 3000 Chebyshev points of t; degree 6: 1.2e-6); with
// fp32's roundings q is within ten half steps.  So the negative tail is as exact as its own size asks for, where an approximation of erf itself, within 1.5e-7 of 1, was nine
// steps of bf16 off at -12.  16 384 x 2048 x 2048 with GELU and saved values takes 151 us, with that approximation (degree 5, one exponential too) 150.  (The mathematical
// library's erff took 50 us more, three times the product's own epilogue.)
struct Tail {
	float q, g;
};
__device__ __forceinline__ Tail normal_tail(float z) {
	const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.305f, 1.f));
	const float p = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.0363750011f, -0.151774764f), 0.18384853f), -0.0364459902f), 0.120301656f), 0.103615142f), 0.122438982f), 0.121641368f);
	return {t * p, __builtin_amdgcn_exp2f(z * -0.36067376022224085f * z)};
}
__device__ __forceinline__ float activation(float z, int kind) {
	if (kind == N2_ACTIVATION_RELU) return z > 0.f ? z : 0.f;
	if (kind == N2_ACTIVATION_SILU) {
		const float u = exp_minus_abs(z), r = __builtin_amdgcn_rcpf(1.f + u);
		return z * (z < 0.f ? u * r : r);
	}
	if (kind == N2_ACTIVATION_GELU) {
		const Tail a = normal_tail(z);
		const float below = a.q * a.g * a.g;
		return z * (z < 0.f ? below : 1.f - below);
	}
	return z;
}
__device__ __forceinline__ float activation_slope(float z, int kind) {
	if (kind == N2_ACTIVATION_SILU) {
		// s + z s (1 - s), s the logistic function, by u = exp(-|z|): 1 - s is formed without the difference, whose half step z would multiply
		const float u = exp_minus_abs(z), r = __builtin_amdgcn_rcpf(1.f + u), ur = u * r;
		return fmaf(z * ur, r, z < 0.f ? ur : r);
	}
	if (kind == N2_ACTIVATION_GELU) {
		const Tail a = normal_tail(z);
		return fmaf(fmaf(z, 0.39894228040143268f, z < 0.f ? a.q : -a.q) * a.g, a.g, z < 0.f ? 0.f : 1.f);
	}
	return 1.f;
}

__device__ __forceinline__ float slope_times(float dy, float z, int kind) {
	if (kind == N2_ACTIVATION_NONE) return dy;
	if (kind == N2_ACTIVATION_RELU) return z > 0.f ? dy : 0.f;
	return dy * activation_slope(z, kind);
}

// Eight values in each of sixteen lanes, i their number: the sum of value i % 8 over all lanes.  Each step keeps the half of the values that the
// lane's next bit names and takes the partner's: 8, 4, 2 and 1 are left.
__device__ __forceinline__ float sum_of_sixteen(float (&v)[8], uint32_t i) {
	auto dpp = [](float x, auto control) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(control)::value, 0xf, 0xf, true)); };
	auto half = [&](uint32_t n, uint32_t bit, auto control) __attribute__((always_inline)) {
#pragma unroll
		for (uint32_t j = 0; j < n; ++j) {
			const float low = v[j], high = v[j + n];
			v[j] = ((i & bit) != 0u ? high : low) + dpp((i & bit) != 0u ? low : high, control);
		}
	};
	half(4u, 4u, std::integral_constant<int, 0x141>{});  // row_half_mirror: lane i ^ 7
	half(2u, 2u, std::integral_constant<int, 0x1B>{});   // quad_perm 3 2 1 0: i ^ 3
	half(1u, 1u, std::integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2: i ^ 1
	return v[0] + dpp(v[0], std::integral_constant<int, 0x128>{});  // row_ror 8: i ^ 8
}

// -------------------------------------------------------------------------------------------------------------------------------------
// tiles
// -------------------------------------------------------------------------------------------------------------------------------------
constexpr uint32_t BK = 64;

struct Operand {
	const void* p;
	uint64_t ld;
	bool padded;  // what stands between a row's end and the next multiple of eight values is zero
};

// A tile of R indices by BK in LDS, 16 bytes (eight values) at a time.  Contiguous in k: R rows of eight pieces.  Contiguous in its own
// index: BK rows of R / 8 pieces.  Pieces of a row are permuted so that the lanes that read one column of pieces meet different banks.
template <bool KC, uint32_t R, uint32_t RUN>
__device__ __forceinline__ uint32_t place(uint32_t row, uint32_t piece) {
	if constexpr (KC) {
		// the 16 rows of a fragment: consecutive ones, or four runs of four that stand eight apart
		const uint32_t f = RUN == 4u ? row % 8u : row % 4u + row / RUN % 2u * 4u;
		return row * (BK / 8u) + (piece ^ f);
	} else {
		// a half wave reads 32 bytes of each of the rows k .. k + 3 and k + 8 .. k + 11
		const uint32_t f = 2u * (row % 4u) + (R >= 128u ? row / 8u % 2u * 8u : 0u);
		return row * (R / 8u) + (piece ^ f);
	}
}

// A tile of an operand that may start at any element, on its way through registers: load() asks for the one from index `first` and k0 on, put()
// writes it to LDS, zero past the extent and past K.  Every piece is one load of 16 bytes inside the matrix, moved back from its end where it
// would go beyond, and only put(), a stage later, shifts and cuts it: nothing waits for a load before that.  (Loaded and put at once, element by
// element at the rows' ends, a product took, forward, 56 us for 36 at 6836 x 3385 x 109, 70 for 60 at 139 043 x 255 x 111, 12 for 10.2 at 300 x 333 x 77,
// backward with ReLU 45 for 40 at 12 783 x 279 x 216, 177 for 141 at 139 043 x 255 x 111.)
template <typename T, bool KC, uint32_t R, uint32_t RUN, uint32_t THREADS>
struct RegisterTile {
	static constexpr uint32_t LOADS = R * BK / 8u / THREADS, ROW = KC ? BK / 8u : R / 8u;
	const T* p;
	uint64_t ld, end;  // the matrix is [p, p + end)
	uint32_t first, extent;
	uint4 v[LOADS];

	__device__ __forceinline__ RegisterTile(const Operand& o, uint32_t from, uint32_t n, uint32_t k)
		: p(static_cast<const T*>(o.p)), ld(o.ld), end(KC ? (uint64_t)(n - 1u) * o.ld + k : (uint64_t)(k - 1u) * o.ld + n), first(from), extent(n) {}
	__device__ __forceinline__ uint64_t place_of(uint32_t i, uint32_t k0) const {
		const uint32_t at = i * THREADS + threadIdx.x, row = at / ROW, piece = at % ROW;
		return KC ? (uint64_t)(first + row) * ld + k0 + piece * 8u : (uint64_t)(k0 + row) * ld + first + piece * 8u;
	}
	__device__ __forceinline__ void load(uint32_t k0) {
		if (end < 8u) return;
#pragma unroll
		for (uint32_t i = 0; i < LOADS; ++i) __builtin_memcpy(&v[i], p + min(place_of(i, k0), end - 8u), 16);
	}
	__device__ __forceinline__ void put(uint4* __restrict__ lds, uint32_t k0, uint32_t k_end) {
#pragma unroll
		for (uint32_t i = 0; i < LOADS; ++i) {
			const uint32_t at = i * THREADS + threadIdx.x, row = at / ROW, piece = at % ROW;
			const uint32_t index = KC ? first + row : first + piece * 8u, k = KC ? k0 + piece * 8u : k0 + row;
			const uint32_t valid = index < extent && k < k_end ? min(KC ? k_end - k : extent - index, 8u) : 0u;
			if (end < 8u) {
				v[i] = __builtin_bit_cast(uint4, n2_load_vec(p + (valid != 0u ? place_of(i, k0) : 0u), valid));
			} else if (valid < 8u) {
				typedef unsigned __int128 Bits;
				const uint64_t from = place_of(i, k0), back = from + 8u > end ? from + 8u - end : 0u;
				Bits bits = __builtin_bit_cast(Bits, v[i]);
				bits = valid != 0u ? bits >> ((uint32_t)back * 16u) & ~(Bits)0 >> (128u - 16u * valid) : (Bits)0;
				v[i] = __builtin_bit_cast(uint4, bits);
			}
			lds[place<KC, R, RUN>(row, piece)] = v[i];
		}
	}
};

// Reads operands of matrix instructions: 16 indices by 32 values of k, lane l holding index l % 16 and the eight values from 8 * (l / 16)
// on.  The 16 indices are consecutive (RUN 4), or four runs of four, eight apart (RUN 8); number u begins at first + b_base(u).  The
// permutation of place() is the same for every u and kk, so a lane's address is one offset (two, for contiguous k) and constants.
template <uint32_t RUN>
__device__ __forceinline__ constexpr uint32_t b_base(uint32_t u) { return RUN == 4u ? u * 16u : u / 2u * 32u + u % 2u * 4u; }

template <bool KC, uint32_t R, uint32_t RUN>
struct Fragments {
	uint32_t offset[KC ? BK / 32u : 1u];  // bytes

	__device__ __forceinline__ explicit Fragments(uint32_t first) {
		const uint32_t lane = threadIdx.x & 63u, i = lane % 16u, g = lane / 16u;
		if constexpr (KC) {
#pragma unroll
			for (uint32_t kk = 0; kk < BK / 32u; ++kk) offset[kk] = 16u * place<KC, R, RUN>(first + i / 4u * RUN + i % 4u, kk * 4u + g);
		} else {
			static_assert(RUN == 4u, "");
			offset[0] = 16u * place<KC, R, RUN>(g * 8u + i / 4u, first / 8u + i % 4u / 2u) + i % 2u * 8u;
		}
	}
	__device__ __forceinline__ s16x8 read(const uint4* tile, uint32_t u, uint32_t kk) const {
		const char* lds = reinterpret_cast<const char*>(tile);
		if constexpr (KC) {
			return *reinterpret_cast<const s16x8*>(lds + offset[kk] + b_base<RUN>(u) * BK * 2u);
		} else {
			// (16 indices on: two pieces, whose number's bits the first one leaves free; four and 32 values of k on: rows of the same permutation)
			typedef __attribute__((address_space(3))) s16x4* Half;
			const char* p = lds + (offset[0] ^ u * 32u) + kk * 64u * R;
			const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Half)(p)), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Half)(p + 8u * R));
			return s16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
		}
	}
};

// -------------------------------------------------------------------------------------------------------------------------------------
// the product
// -------------------------------------------------------------------------------------------------------------------------------------
enum Epilogue { LAYER, STORE, GRADIENT };
// C, or the sums of one split of k: known where the kernel is built (a test in the epilogue costs large products 2 %), or by Product::partial
enum Output { WHOLE, SPLIT, EITHER };

struct Product {
	Operand a, b;
	uint32_t m, n, k;
	uint32_t extent_a, extent_b;  // indices that may be read (of an operand contiguous in them a multiple of eight)
	uint32_t tiles_m, tiles_n, splits, k_per_split;
	void* c;         // T [m][n]
	uint64_t ldc;
	float* partial;  // or null: the sums of the splits, [splits][m][n], instead of C
	// LAYER
	const void* bias;
	const void* residual;
	uint64_t ldr;
	void* pre;
	uint64_t ldp;
	int activation;
	int accumulate;  // GRADIENT
};

template <typename T, uint32_t N>
struct Run {
	T v[N];
};
// N consecutive values of row m from column n on, all of them inside
template <typename T, int EPI, int OUT, uint32_t N>
__device__ __forceinline__ void finish(const Product& q, uint32_t m, uint32_t n, uint32_t split, float (&v)[N]) {
	auto add = [&](const T* p) __attribute__((always_inline)) {
		Run<T, N> t;
		__builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
		for (uint32_t i = 0; i < N; ++i) v[i] += (float)t.v[i];
	};
	auto store = [&](auto* p) __attribute__((always_inline)) {
		Run<std::remove_pointer_t<decltype(p)>, N> t;
#pragma unroll
		for (uint32_t i = 0; i < N; ++i) t.v[i] = (std::remove_pointer_t<decltype(p)>)v[i];
		__builtin_memcpy(p, &t, sizeof(t));
	};
	if (OUT == SPLIT || (OUT == EITHER && q.partial != nullptr)) {
		store(q.partial + ((uint64_t)split * q.m + m) * q.n + n);
	} else {
		T* c = static_cast<T*>(q.c) + (uint64_t)m * q.ldc + n;
		if constexpr (EPI == LAYER) {
			if (q.bias != nullptr) add(static_cast<const T*>(q.bias) + n);
			if (q.pre != nullptr) store(static_cast<T*>(q.pre) + (uint64_t)m * q.ldp + n);
			if (q.activation != N2_ACTIVATION_NONE)
#pragma unroll
				for (uint32_t i = 0; i < N; ++i) v[i] = activation(v[i], q.activation);
			if (q.residual != nullptr) add(static_cast<const T*>(q.residual) + (uint64_t)m * q.ldr + n);
		}
		if constexpr (EPI == GRADIENT)
			if (q.accumulate) add(c);
		store(c);
	}
}

// The layer's epilogue for eight columns whose bias and residual are in registers.
template <typename T, bool RESIDUAL>
__device__ __forceinline__ void finish_with(const Product& q, uint32_t m, uint32_t n, float (&v)[8], const uint4& bias, const uint4& residual) {
	auto add = [&](const uint4& u) __attribute__((always_inline)) {
		const N2Vec<T> t = __builtin_bit_cast(N2Vec<T>, u);
#pragma unroll
		for (uint32_t i = 0; i < 8u; ++i) v[i] += (float)t.v[i];
	};
	auto store = [&](void* p, uint64_t ld) __attribute__((always_inline)) {
		N2Vec<T> t;
#pragma unroll
		for (uint32_t i = 0; i < 8u; ++i) t.v[i] = (T)v[i];
		__builtin_memcpy(static_cast<T*>(p) + (uint64_t)m * ld + n, &t, 16);
	};
	if (q.bias != nullptr) add(bias);
	if (q.pre != nullptr) store(q.pre, q.ldp);
	if (q.activation != N2_ACTIVATION_NONE)
#pragma unroll
		for (uint32_t i = 0; i < 8u; ++i) v[i] = activation(v[i], q.activation);
	if constexpr (RESIDUAL) add(residual);
	store(q.c, q.ldc);
}

// What a wave has of C, from (m0, n0) on.  Inside C a lane stores its runs of RUN columns; at an edge sixteen rows at a time go through LDS
// of the wave's own (16 rows of its columns) and are finished one by one, a row's columns side by side in the lanes.
template <typename T, int EPI, int OUT, uint32_t RUN, uint32_t S, uint32_t U>
__device__ __forceinline__ void finish_all(const Product& q, uint32_t m0, uint32_t n0, uint32_t split, const f32x4 (&acc)[S][U], float* lds) {
	constexpr uint32_t WIDTH = U * 16u;
	const uint32_t lane = threadIdx.x & 63u;
	if (m0 + S * 16u <= q.m && n0 + WIDTH <= q.n) {
#pragma unroll
		for (uint32_t s = 0; s < S; ++s)
#pragma unroll
			for (uint32_t u = 0; u < U; u += RUN / 4u) {
				float v[RUN];
#pragma unroll
				for (uint32_t r = 0; r < RUN; ++r) v[r] = acc[s][u + r / 4u][r % 4u];
				finish<T, EPI, OUT>(q, m0 + s * 16u + lane % 16u, n0 + b_base<RUN>(u) + lane / 16u * RUN, split, v);
			}
		return;
	}
	if (m0 >= q.m || n0 >= q.n) return;
	float* mine = lds + threadIdx.x / 64u * 16u * WIDTH;
#pragma unroll
	for (uint32_t s = 0; s < S; ++s) {
#pragma unroll
		for (uint32_t u = 0; u < U; ++u) *reinterpret_cast<f32x4*>(mine + lane % 16u * WIDTH + (b_base<RUN>(u) + lane / 16u * RUN)) = acc[s][u];
		__builtin_amdgcn_wave_barrier();
#pragma unroll 1
		for (uint32_t i = lane; i < 16u * WIDTH; i += 64u) {
			const uint32_t m = m0 + s * 16u + i / WIDTH, n = n0 + i % WIDTH;
			float v[1] = {mine[i]};
			if (m < q.m && n < q.n) finish<T, EPI, OUT>(q, m, n, split, v);
		}
		__builtin_amdgcn_wave_barrier();
	}
}

// BM x BN of C to a workgroup, WM x WN waves.  The matrix instruction's rows are n and its columns m, so that a lane's four values stand side
// by side in a row of C; where B is contiguous in k its rows are dealt to the instructions so that all of a lane's values do.
template <typename T, bool A_KC, bool B_KC, uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, int EPI, int OUT>
__device__ __forceinline__ void product(const Product& q, uint32_t block, uint4* __restrict__ tile_a, uint4* __restrict__ tile_b) {
	constexpr uint32_t THREADS = WM * WN * 64u, S = BM / WM / 16u, U = BN / WN / 16u, RUN = B_KC ? 8u : 4u;
	const uint32_t tile = block % (q.tiles_m * q.tiles_n), split = block / (q.tiles_m * q.tiles_n);
	const uint32_t m0 = tile / q.tiles_n * BM, n0 = tile % q.tiles_n * BN;
	const uint32_t wave = threadIdx.x / 64u, wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
	const uint32_t k_begin = split * q.k_per_split, k_end = min(q.k, k_begin + q.k_per_split);
	const Fragments<A_KC, BM, 4u> a_read(wm);
	const Fragments<B_KC, BN, RUN> b_read(wn);
	f32x4 acc[S][U] = {};
	RegisterTile<T, A_KC, BM, 4u, THREADS> a_tile(q.a, m0, q.m, q.k);
	RegisterTile<T, B_KC, BN, RUN, THREADS> b_tile(q.b, n0, q.n, q.k);
	if (k_begin < k_end) a_tile.load(k_begin), b_tile.load(k_begin);  // (of no rows there is nothing to load)
	for (uint32_t k0 = k_begin; k0 < k_end; k0 += BK) {
		a_tile.put(tile_a, k0, k_end);
		b_tile.put(tile_b, k0, k_end);
		__syncthreads();
		a_tile.load(k0 + BK), b_tile.load(k0 + BK);  // (past the end of k: the matrix's last values, not used)
#pragma unroll
		for (uint32_t kk = 0; kk < BK / 32u; ++kk) {
			s16x8 a[S], b[U];
#pragma unroll
			for (uint32_t s = 0; s < S; ++s) a[s] = a_read.read(tile_a, s, kk);
#pragma unroll
			for (uint32_t u = 0; u < U; ++u) b[u] = b_read.read(tile_b, u, kk);
#pragma unroll
			for (uint32_t s = 0; s < S; ++s)
#pragma unroll
				for (uint32_t u = 0; u < U; ++u) acc[s][u] = mfma(T{}, b[u], a[s], acc[s][u]);
		}
		__syncthreads();
	}
	finish_all<T, EPI, OUT, RUN>(q, m0 + wm, n0 + wn, split, acc, reinterpret_cast<float*>(tile_a));
}

// Such a tile straight from memory into LDS (no register in between): 16 bytes from each lane's address go to the wave's place and
// 16 bytes times the lane, so a lane asks for the piece that belongs there.  Rows and pieces past the extent are the last ones once more; what
// is computed from them is not stored.  Pieces past the end of k (a multiple of eight, for an operand contiguous in k) are zeros from g_zeros.
__device__ const uint4 g_zeros = {0u, 0u, 0u, 0u};

template <typename T, bool KC, uint32_t R, uint32_t RUN, uint32_t THREADS>
struct AsyncTile {
	static constexpr uint32_t LOADS = R * BK / 8u / THREADS, ROW = KC ? BK / 8u : R / 8u;
	uint32_t offset[LOADS], k_of;  // (k_of: the lane's first k in a tile; KC: the same for all loads)
	const char* base;
	uint64_t step;

	__device__ __forceinline__ AsyncTile(const Operand& o, uint32_t first, uint32_t extent, uint32_t k0) {
		const T* p = static_cast<const T*>(o.p);
		base = reinterpret_cast<const char*>(KC ? p + (uint64_t)first * o.ld + k0 : p + (uint64_t)k0 * o.ld + first);
		step = (KC ? (uint64_t)BK : BK * o.ld) * sizeof(T);
		static_assert(!KC || THREADS / ROW % 16u == 0u, "the permutation of place() repeats from load to load");
		k_of = KC ? place<KC, R, RUN>(threadIdx.x / ROW, threadIdx.x % ROW) % ROW * 8u : threadIdx.x / ROW;
#pragma unroll
		for (uint32_t i = 0; i < LOADS; ++i) {
			const uint32_t at = i * THREADS + threadIdx.x, row = at / ROW, piece = place<KC, R, RUN>(row, at % ROW) % ROW;
			offset[i] = KC ? min(row, extent - 1u - first) * (uint32_t)o.ld * 2u + piece * 16u : row * (uint32_t)o.ld * 2u + min(piece, (extent - first) / 8u - 1u) * 16u;
		}
	}
	// left: values of k from this tile's first on, none included
	__device__ __forceinline__ void load(uint4* lds, uint32_t i, uint32_t left) {
		const char* from = k_of + (KC ? 0u : i * (THREADS / ROW)) < left ? base + offset[i] : reinterpret_cast<const char*>(&g_zeros);
		__builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from, (__attribute__((address_space(3))) void*)(lds + i * THREADS + (threadIdx.x & ~63u)), 16, 0, 0);
	}
	__device__ __forceinline__ void advance() { base += step; }
};

// One stage of the product, in ta and tb, while the next one, of which `left` values of k are left, goes to next_a and next_b.  The matrix
// instructions come in steps of U, one fragment of A each, which is read two steps ahead; B's fragments of the second half are read while
// the first is computed; a load of the next stage is sent off with each step.  (That the four tiles do not overlap has to stand here: where
// the compiler takes a load into LDS for one that a later reading meets, it waits for all loads before that.)
template <typename T, bool A_KC, bool B_KC, uint32_t BM, uint32_t BN, uint32_t RUN, uint32_t THREADS, uint32_t S, uint32_t U>
__device__ __forceinline__ void product_stage(const uint4* __restrict__ ta, const uint4* __restrict__ tb, uint4* __restrict__ next_a, uint4* __restrict__ next_b, uint32_t left,
                                              const Fragments<A_KC, BM, 4u>& a_read, const Fragments<B_KC, BN, RUN>& b_read, AsyncTile<T, A_KC, BM, 4u, THREADS>& a_tile,
                                              AsyncTile<T, B_KC, BN, RUN, THREADS>& b_tile, f32x4 (&acc)[S][U]) {
	constexpr uint32_t STEPS = S * BK / 32u, AHEAD = 2u, LOADS_A = AsyncTile<T, A_KC, BM, 4u, THREADS>::LOADS, LOADS_B = AsyncTile<T, B_KC, BN, RUN, THREADS>::LOADS;
	// (smaller tiles read B's fragments of both halves at once)
	constexpr bool BOTH = S < U + AHEAD;
	static_assert(BK == 64u && LOADS_A + LOADS_B <= STEPS, "");
	s16x8 a[STEPS], b[2][U];
#pragma unroll
	for (uint32_t u = 0; u < U; ++u) b[0][u] = b_read.read(tb, u, 0u);
#pragma unroll
	for (uint32_t i = 0; i < AHEAD; ++i) a[i] = a_read.read(ta, i % S, i / S);
	if constexpr (BOTH) {
#pragma unroll
		for (uint32_t u = 0; u < U; ++u) b[1][u] = b_read.read(tb, u, 1u);
	}
#pragma unroll
	for (uint32_t i = 0; i < STEPS; ++i) {
		constexpr uint32_t B_FROM = BOTH ? 0u : S - U - AHEAD;
		if (i + AHEAD < STEPS) a[i + AHEAD] = a_read.read(ta, (i + AHEAD) % S, (i + AHEAD) / S);
		if (!BOTH && i >= B_FROM && i < B_FROM + U) b[1][i - B_FROM] = b_read.read(tb, i - B_FROM, 1u);
		if (i < LOADS_A) a_tile.load(next_a, i, left);
		else if (i < LOADS_A + LOADS_B) b_tile.load(next_b, i - LOADS_A, left);
#pragma unroll
		for (uint32_t u = 0; u < U; ++u) acc[i % S][u] = mfma(T{}, b[i / S][u], a[i], acc[i % S][u]);
		__builtin_amdgcn_sched_barrier(0);
	}
	a_tile.advance(), b_tile.advance();
}

// Two stages in LDS.  Tiles of 256 (128 KiB, eight waves of 128 x 64) read 96 of the 128 bytes that LDS gives in a clock under full matrix cores,
// those of 128 (four of 64 x 64) all of them, those of 64 (four of 32 x 32) twice that: half the rate at most.  bf16 on an MI355X: 8192 x 8192 x 8192 1310 TFLOP/s, 16 384 x 2048 x 2048 116 us (1180), plain, beside 1370 and 1208 for the
// library's product of that size; 2^18 x 256 x 256 is bound by memory.
template <typename T, bool A_KC, bool B_KC, uint32_t BM, uint32_t BN, uint32_t WM, uint32_t WN, int EPI, int OUT>
__device__ __forceinline__ void product_async(const Product& q, uint32_t block, uint32_t blocks, uint4* tile_a0, uint4* tile_a1, uint4* tile_b0, uint4* tile_b1) {
	constexpr uint32_t THREADS = WM * WN * 64u, S = BM / WM / 16u, U = BN / WN / 16u, RUN = B_KC ? 8u : 4u;
	const uint32_t tiles = q.tiles_m * q.tiles_n, work = n2_xcd_order(block, blocks), split = work / tiles;
	uint32_t tm, tn;
	n2_tile_order(work - split * tiles, q.tiles_m, q.tiles_n, tm, tn);
	const uint32_t m0 = tm * BM, n0 = tn * BN;
	const uint32_t wave = threadIdx.x / 64u, wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
	const uint32_t k_begin = split * q.k_per_split, k_end = min(q.k, k_begin + q.k_per_split);
	AsyncTile<T, A_KC, BM, 4u, THREADS> a_tile(q.a, m0, q.extent_a, k_begin);
	AsyncTile<T, B_KC, BN, RUN, THREADS> b_tile(q.b, n0, q.extent_b, k_begin);
	const Fragments<A_KC, BM, 4u> a_read(wm);
	const Fragments<B_KC, BN, RUN> b_read(wn);
	f32x4 acc[S][U] = {};
	uint32_t left = k_end - k_begin;  // values of k from the stage on that is asked for next
	const uint32_t stages = n2_ceil_div(left, BK);
	if (left > 0u) {
#pragma unroll
		for (uint32_t i = 0; i < a_tile.LOADS; ++i) a_tile.load(tile_a0, i, left);
#pragma unroll
		for (uint32_t i = 0; i < b_tile.LOADS; ++i) b_tile.load(tile_b0, i, left);
		a_tile.advance(), b_tile.advance();
	}
	// a stage is there once every wave's loads into LDS have arrived; the one before it has been read by then
	auto arrived = []() __attribute__((always_inline)) {
		__builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
		__syncthreads();
	};
	// (stages come in pairs: a branch out between the two would have the sums in other registers there)
	for (uint32_t pair = 0; pair < stages / 2u; ++pair) {
		left -= BK;
		arrived();
		product_stage<T, A_KC, B_KC, BM, BN, RUN, THREADS>(tile_a0, tile_b0, tile_a1, tile_b1, left, a_read, b_read, a_tile, b_tile, acc);
		left -= min(left, BK);
		arrived();
		product_stage<T, A_KC, B_KC, BM, BN, RUN, THREADS>(tile_a1, tile_b1, tile_a0, tile_b0, left, a_read, b_read, a_tile, b_tile, acc);
	}
	if (stages % 2u != 0u) {
		arrived();
		product_stage<T, A_KC, B_KC, BM, BN, RUN, THREADS>(tile_a0, tile_b0, tile_a1, tile_b1, 0u, a_read, b_read, a_tile, b_tile, acc);
	}
	arrived();
	finish_all<T, EPI, OUT, RUN>(q, m0 + wm, n0 + wn, split, acc, reinterpret_cast<float*>(tile_a0));
}

template <typename T, bool ASYNC, bool A_KC, bool B_KC, uint32_t B, uint32_t WM, uint32_t WN, int EPI, int OUT>
__global__ void __launch_bounds__(WM* WN * 64) product_kernel(Product q) {
	__shared__ uint4 a0[B * BK / 8u], b0[B * BK / 8u], a1[ASYNC ? B * BK / 8u : 1u], b1[ASYNC ? B * BK / 8u : 1u];
	if constexpr (ASYNC) product_async<T, A_KC, B_KC, B, B, WM, WN, EPI, OUT>(q, blockIdx.x, gridDim.x, a0, a1, b0, b1);
	else product<T, A_KC, B_KC, B, B, WM, WN, EPI, OUT>(q, blockIdx.x, a0, b0);
}

// Both products of a backward pass in one launch, where both come in tiles of 64: the first blocks_x workgroups are dx's.  Backward with ReLU, us, in one
// launch | in two: 300 x 512 x 512 13.7 | 18.3, 2000 x 64 x 64 13.5 | 16.4, 5003 x 320 x 257 24.4 | 26.9, 1000 x 1024 x 1024 26 | 34, 50 000 x 200 x 136 50 | 53, 20 000 x 512 x 512 68 | 68.
template <typename T, bool ASYNC>
__global__ void __launch_bounds__(256) product_pair_kernel(Product x, Product w, uint32_t blocks_x) {
	__shared__ uint4 a0[64u * BK / 8u], b0[64u * BK / 8u], a1[ASYNC ? 64u * BK / 8u : 1u], b1[ASYNC ? 64u * BK / 8u : 1u];
	if (blockIdx.x < blocks_x) {
		if constexpr (ASYNC) product_async<T, true, false, 64, 64, 2, 2, STORE, EITHER>(x, blockIdx.x, blocks_x, a0, a1, b0, b1);
		else product<T, true, false, 64, 64, 2, 2, STORE, EITHER>(x, blockIdx.x, a0, b0);
	} else {
		if constexpr (ASYNC) product_async<T, false, false, 64, 64, 2, 2, GRADIENT, EITHER>(w, blockIdx.x - blocks_x, gridDim.x - blocks_x, a0, a1, b0, b1);
		else product<T, false, false, 64, 64, 2, 2, GRADIENT, EITHER>(w, blockIdx.x - blocks_x, a0, b0);
	}
}

// The sums of the parts that k was dealt out to, finished: a lane takes four columns of a row, and of more than
// sixteen parts every sixteenth.  (With all of them in one lane the weights' gradient of 2^18 x 64 x 64 took 38 us for 30, of 2^18 x 128 x 128 65 for 52.)
constexpr uint32_t JOIN_ALONE = 16;
template <typename T, int EPI>
__device__ __forceinline__ void join(const Product& q, uint32_t block) {
	__shared__ f32x4 part[16][16];
	const bool alone = q.splits <= JOIN_ALONE;
	const uint32_t quads = n2_ceil_div(q.n, 4u), first = alone ? 0u : threadIdx.x / 16u, step = alone ? 1u : 16u;
	const uint64_t at = alone ? (uint64_t)block * 256u + threadIdx.x : (uint64_t)block * 16u + threadIdx.x % 16u, row = at / quads;
	const uint32_t m = (uint32_t)row, n = (uint32_t)(at - row * quads) * 4u, valid = row < q.m ? min(q.n - n, 4u) : 0u;
	f32x4 sum = {0.f, 0.f, 0.f, 0.f};
	const float* p = q.partial + row * q.n + n;
	const uint64_t pitch = (uint64_t)q.m * q.n;
	if (valid == 4u) {
#pragma unroll 8
		for (uint32_t i = first; i < q.splits; i += step) {
			f32x4 t;
			__builtin_memcpy(&t, p + i * pitch, 16);
			sum += t;
		}
	} else {
		for (uint32_t i = first; i < q.splits; i += step)
#pragma unroll
			for (uint32_t j = 0; j < 3u; ++j)
				if (j < valid) sum[j] += p[i * pitch + j];
	}
	if (!alone) {
		part[first][threadIdx.x % 16u] = sum;
		__syncthreads();
		if (first != 0u) return;
#pragma unroll
		for (uint32_t i = 1; i < 16u; ++i) sum += part[i][threadIdx.x];
	}
	if (valid == 4u) {
		float v[4] = {sum[0], sum[1], sum[2], sum[3]};
		finish<T, EPI, WHOLE>(q, m, n, 0u, v);
	} else {
#pragma unroll
		for (uint32_t j = 0; j < 3u; ++j) {
			float v[1] = {sum[j]};
			if (j < valid) finish<T, EPI, WHOLE>(q, m, n + j, 0u, v);
		}
	}
}
uint32_t join_blocks(const Product& q) { return q.partial != nullptr ? n2_ceil_div((uint64_t)q.m * n2_ceil_div(q.n, 4u), q.splits <= JOIN_ALONE ? 256u : 16u) : 0u; }

template <typename T>
__global__ void __launch_bounds__(256) join_kernel(Product q) { join<T, LAYER>(q, blockIdx.x); }

// What is left of a backward pass: dx's and dW's splits, and the bias's gradient from the column sums of sum_rows workgroups.
template <typename T>
__global__ void __launch_bounds__(256) join_backward_kernel(Product x, uint32_t blocks_x, Product w, uint32_t blocks_w, const float* __restrict__ sums, uint32_t sum_rows, uint32_t columns,
                                                            T* __restrict__ db, int accumulate) {
	const uint32_t block = blockIdx.x;
	if (block < blocks_x) join<T, STORE>(x, block);
	else if (block - blocks_x < blocks_w) join<T, GRADIENT>(w, block - blocks_x);
	else n2_column_sums_block<16, 16>(sums, sum_rows, columns, block - blocks_x - blocks_w, [&](uint32_t column, float sum) { n2_store_sum(db + column, sum, accumulate); });
}

// A layer of up to sixteen rows: what it takes is the weights' way from memory, so sixteen columns of C go to a workgroup and its sixteen
// waves take 32 values of k in turn, straight into the matrix instructions' registers; every wave's loads are under way at once.
template <typename T>
__global__ void __launch_bounds__(1024) few_rows_kernel(Product q) {
	constexpr uint32_t WAVES = 16u, AT_ONCE = 4u;
	__shared__ float part[WAVES][16u][16u];
	const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u, i = lane % 16u, g = lane / 16u, n0 = blockIdx.x * 16u;
	const T* w = static_cast<const T*>(q.b.p) + (uint64_t)min(n0 + i, q.n - 1u) * q.b.ld;
	const T* x = static_cast<const T*>(q.a.p) + (uint64_t)min(i, q.m - 1u) * q.a.ld;
	f32x4 acc = {};
	for (uint32_t k0 = wave * 32u; k0 < q.k; k0 += WAVES * 32u * AT_ONCE) {
		s16x8 b[AT_ONCE], a[AT_ONCE];
#pragma unroll
		for (uint32_t j = 0; j < AT_ONCE; ++j) {
			const uint32_t k = k0 + j * WAVES * 32u + g * 8u, valid = k < q.k ? min(q.k - k, 8u) : 0u;
			b[j] = __builtin_bit_cast(s16x8, n2_load_vec(w + k, valid));
			a[j] = __builtin_bit_cast(s16x8, n2_load_vec(x + k, valid));
		}
#pragma unroll
		for (uint32_t j = 0; j < AT_ONCE; ++j) acc = mfma(T{}, b[j], a[j], acc);
	}
	*reinterpret_cast<f32x4*>(&part[wave][i][g * 4u]) = acc;
	__syncthreads();
	const uint32_t m = threadIdx.x / 16u, n = threadIdx.x % 16u;
	if (m >= q.m || m >= 16u || n0 + n >= q.n) return;
	float v[1] = {0.f};
#pragma unroll
	for (uint32_t k = 0; k < WAVES; ++k) v[0] += part[k][m][n];
	finish<T, LAYER, WHOLE>(q, m, n0 + n, 0u, v);
}

// The weights of a narrow layer in LDS, as the matrix instructions take them: KT steps of 32 values of k, NT instructions of 16 columns, whose
// pairs leave eight consecutive columns of C in a lane.
template <typename T, uint32_t KT, uint32_t NT, bool B_KC>
__device__ __forceinline__ void fill_weights(const Product& q, uint4* weights) {
	const uint32_t lane = threadIdx.x & 63u, i = lane % 16u, g = lane / 16u;
	// (all of a lane's loads are under way at once)
	if constexpr (B_KC) {
		constexpr uint32_t FILL = (NT * KT * 64u + 1023u) / 1024u;
		uint4 fill[FILL];
	#pragma unroll
		for (uint32_t j = 0; j < FILL; ++j) {
			const uint32_t at = j * 1024u + threadIdx.x, u = at / 64u / KT, kk = at / 64u % KT, n = b_base<8>(u) + i / 4u * 8u + i % 4u, k = kk * 32u + g * 8u;
			fill[j] = *reinterpret_cast<const uint4*>(static_cast<const T*>(q.b.p) + (uint64_t)min(n, q.n - 1u) * q.b.ld + min(k, q.k - 8u));
			if (n >= q.n || k >= q.k) fill[j] = make_uint4(0u, 0u, 0u, 0u);
		}
	#pragma unroll
		for (uint32_t j = 0; j < FILL; ++j)
			if (j * 1024u + threadIdx.x < NT * KT * 64u) weights[j * 1024u + threadIdx.x] = fill[j];
	} else {
		// columns of W as rows: eight by eight values to a lane, turned around in its registers
		static_assert(NT * KT * 8u <= 1024u, "");
		const uint32_t n = threadIdx.x % (NT * 2u) * 8u, k = threadIdx.x / (NT * 2u) * 8u;
		N2Vec<T> in[8];
#pragma unroll
		for (uint32_t j = 0; j < 8u; ++j) {
			const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const T*>(q.b.p) + (uint64_t)min(k + j, q.k - 1u) * q.b.ld + min(n, q.n - 8u));
			in[j] = __builtin_bit_cast(N2Vec<T>, n < q.n && k + j < q.k ? u : make_uint4(0u, 0u, 0u, 0u));
		}
		if (k < KT * 32u)
#pragma unroll
			for (uint32_t e = 0; e < 8u; ++e) {
				N2Vec<T> out;
#pragma unroll
				for (uint32_t j = 0; j < 8u; ++j) out.v[j] = in[j].v[e];
				weights[((n / 32u * 2u + e / 4u) * KT + k / 32u) * 64u + k % 32u / 8u * 16u + n % 32u / 8u * 4u + e % 4u] = __builtin_bit_cast(uint4, out);
			}
	}
}

// A layer of many rows and few columns: memory bounds it, and tiles that load, multiply and store in turn leave memory idle.  Here the
// weights stay in LDS as the matrix instructions take them, and every wave passes over rows on its own, sixteen at a time: the next rows
// come into registers while these are multiplied, and nothing is waited for in common.  KT steps of 32 values of k, NT instructions of 16
// columns; widths and strides are multiples of eight, rows start at multiples of 16 bytes.  2^18 x 256 x 256: 4.2 TB/s, with a residual 4.1.
// (32 rows to a wave halve what is read from LDS, and were no faster: 64 and 105 us for 63 and 99.)
template <typename T, uint32_t KT, uint32_t NT, bool RESIDUAL>
__global__ void __launch_bounds__(1024) stream_rows_kernel(Product q) {
	__shared__ uint4 weights[NT * KT * 64u], bias[NT * 2u];
	const uint32_t lane = threadIdx.x & 63u, i = lane % 16u, g = lane / 16u;
	fill_weights<T, KT, NT, true>(q, weights);
	if (threadIdx.x < NT * 2u && threadIdx.x * 8u < q.n && q.bias != nullptr) bias[threadIdx.x] = *reinterpret_cast<const uint4*>(static_cast<const T*>(q.bias) + threadIdx.x * 8u);
	__syncthreads();
	const uint64_t tiles = n2_ceil_div(q.m, 16u), step = (uint64_t)gridDim.x * 16u;
	const T* x = static_cast<const T*>(q.a.p);
	const T* r = static_cast<const T*>(q.residual);
	auto load_x = [&](uint4 (&to)[KT], uint64_t tile) __attribute__((always_inline)) {
		const uint64_t row = min(tile * 16u + i, (uint64_t)q.m - 1u);
#pragma unroll
		for (uint32_t kk = 0; kk < KT; ++kk) {
			const uint32_t k = kk * 32u + g * 8u;
			to[kk] = k < q.k ? *reinterpret_cast<const uint4*>(x + row * q.a.ld + k) : make_uint4(0u, 0u, 0u, 0u);
		}
	};
	// (with a residual the registers hold its rows instead of the next ones of x)
	constexpr uint32_t AHEAD = NT / 2u < 4u ? NT / 2u : 4u;
	uint4 now[KT], next[RESIDUAL ? 1u : KT], add[RESIDUAL ? AHEAD : 1u];
	uint64_t tile = (uint64_t)blockIdx.x * 16u + threadIdx.x / 64u;
	if constexpr (!RESIDUAL)
		if (tile < tiles) load_x(next, tile);
	for (; tile < tiles; tile += step) {
		const uint64_t m = tile * 16u + i;
		auto load_r = [&](uint32_t u) __attribute__((always_inline)) {
			const uint32_t n = b_base<8>(u) + g * 8u;
			if (n < q.n) add[u / 2u % AHEAD] = *reinterpret_cast<const uint4*>(r + min(m, (uint64_t)q.m - 1u) * q.ldr + n);
		};
		if constexpr (RESIDUAL) {
			load_x(now, tile);
#pragma unroll
			for (uint32_t u = 0; u < 2u * AHEAD; u += 2u) load_r(u);
		} else {
#pragma unroll
			for (uint32_t kk = 0; kk < KT; ++kk) now[kk] = next[kk];
			if (tile + step < tiles) load_x(next, tile + step);
		}
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (uint32_t u = 0; u < NT; u += 2u) {
			f32x4 acc[2] = {};
#pragma unroll
			for (uint32_t kk = 0; kk < KT; ++kk)
#pragma unroll
				for (uint32_t h = 0; h < 2u; ++h)
					acc[h] = mfma(T{}, __builtin_bit_cast(s16x8, weights[((u + h) * KT + kk) * 64u + lane]), __builtin_bit_cast(s16x8, now[kk]), acc[h]);
			const uint32_t n = b_base<8>(u) + g * 8u;
			if (n < q.n && m < q.m) {
				float v[8];
#pragma unroll
				for (uint32_t j = 0; j < 8u; ++j) v[j] = acc[j / 4u][j % 4u];
				finish_with<T, RESIDUAL>(q, (uint32_t)m, n, v, bias[n / 8u], add[RESIDUAL ? u / 2u % AHEAD : 0u]);
			}
			if constexpr (RESIDUAL)
				if (u + 2u * AHEAD < NT) load_r(u + 2u * AHEAD);
			__builtin_amdgcn_sched_barrier(0);
		}
	}
}

// dx of a narrow layer of many rows in the same way.  q.a is dz, or dy, with z (or null, without an activation): then dz is formed in the
// registers that the matrix instructions take it from.  partial (or null): its column sums, one row of q.k from each workgroup.
template <typename T, uint32_t KT, uint32_t NT>
__global__ void __launch_bounds__(1024) stream_backward_kernel(Product q, const T* __restrict__ z, uint64_t ld_z, float* __restrict__ partial) {
	__shared__ uint4 weights[NT * KT * 64u];
	const uint32_t lane = threadIdx.x & 63u, i = lane % 16u, g = lane / 16u, wave = threadIdx.x / 64u;
	fill_weights<T, KT, NT, false>(q, weights);
	__syncthreads();
	const uint64_t tiles = n2_ceil_div(q.m, 16u), step = (uint64_t)gridDim.x * 16u;
	const T* dy = static_cast<const T*>(q.a.p);
	float sums[KT] = {};  // of column kk * 32 + g * 8 + i % 8, over the lanes of a row of sixteen
	for (uint64_t tile = (uint64_t)blockIdx.x * 16u + wave; tile < tiles; tile += step) {
		const uint64_t m = tile * 16u + i, row = min(m, (uint64_t)q.m - 1u);
		uint4 now[KT], pre[KT];
#pragma unroll
		for (uint32_t kk = 0; kk < KT; ++kk) {
			const uint32_t k = kk * 32u + g * 8u;
			now[kk] = pre[kk] = make_uint4(0u, 0u, 0u, 0u);
			if (k < q.k) {
				now[kk] = *reinterpret_cast<const uint4*>(dy + row * q.a.ld + k);
				if (z != nullptr) pre[kk] = *reinterpret_cast<const uint4*>(z + row * ld_z + k);
			}
		}
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (uint32_t kk = 0; kk < KT; ++kk) {
			if (z == nullptr && partial == nullptr) break;
			const N2Vec<T> d = __builtin_bit_cast(N2Vec<T>, now[kk]), p = __builtin_bit_cast(N2Vec<T>, pre[kk]);
			float v[8];
			N2Vec<T> out;
#pragma unroll
			for (uint32_t j = 0; j < 8u; ++j) {
				v[j] = slope_times((float)d.v[j], (float)p.v[j], z != nullptr ? q.activation : N2_ACTIVATION_NONE);
				out.v[j] = (T)v[j];
				v[j] = m < q.m ? v[j] : 0.f;
			}
			now[kk] = __builtin_bit_cast(uint4, out);
			if (partial != nullptr) sums[kk] += sum_of_sixteen(v, i);
		}
#pragma unroll
		for (uint32_t u = 0; u < NT; u += 2u) {
			f32x4 acc[2] = {};
#pragma unroll
			for (uint32_t kk = 0; kk < KT; ++kk)
#pragma unroll
				for (uint32_t h = 0; h < 2u; ++h)
					acc[h] = mfma(T{}, __builtin_bit_cast(s16x8, weights[((u + h) * KT + kk) * 64u + lane]), __builtin_bit_cast(s16x8, now[kk]), acc[h]);
			const uint32_t n = b_base<8>(u) + g * 8u;
			if (n < q.n && m < q.m) {
				N2Vec<T> out;
#pragma unroll
				for (uint32_t j = 0; j < 8u; ++j) out.v[j] = (T)acc[j / 4u][j % 4u];
				__builtin_memcpy(static_cast<T*>(q.c) + m * q.ldc + n, &out, 16);
			}
			__builtin_amdgcn_sched_barrier(0);
		}
	}
	if (partial == nullptr) return;
	__syncthreads();  // (the weights are read)
	float* all = reinterpret_cast<float*>(weights);
	static_assert(16u * KT * 32u * 4u <= sizeof(weights), "");
	if (i < 8u)
#pragma unroll
		for (uint32_t kk = 0; kk < KT; ++kk) all[wave * KT * 32u + kk * 32u + g * 8u + i] = sums[kk];
	__syncthreads();
	if (threadIdx.x < min(KT * 32u, q.k)) {
		float sum = 0.f;
#pragma unroll
		for (uint32_t w = 0; w < 16u; ++w) sum += all[w * KT * 32u + threadIdx.x];
		partial[(uint64_t)blockIdx.x * q.k + threadIdx.x] = sum;
	}
}

// -------------------------------------------------------------------------------------------------------------------------------------
// dz = dy * act'(z), and its column sums
// -------------------------------------------------------------------------------------------------------------------------------------
// dz is rounded to the type here, and where stream_backward_kernel forms it: the matrix instructions take both operands in one type.  ReLU's and no activation's is exact; with SiLU and
// GELU dx and dW are off by the square root of two times what their own rounding leaves (bf16, 5003 x 320 x 257: 2.35e-3 of the 2-norm for 1.66e-3).  What the rounding leaves as
// a second operand would double both products: 16 384 x 2048 x 2048 290 us to about 500.  The bias's gradient sums the values as they are in fp32.
// LANES lanes of eight values take a row (512 columns of it, where it is wider), rows as far apart as the launch has groups of lanes along
// them.  dz (or null) goes into rows of ld_dz values, a multiple of eight, zero behind the width; partial (or null): one row of sums from
// each workgroup.
template <typename T, uint32_t LANES, bool STREAM>
__global__ void __launch_bounds__(256) slope_kernel(uint32_t n_rows, uint32_t width, const T* __restrict__ dy, uint64_t ld_dy, const T* __restrict__ z, uint64_t ld_z, int kind,
                                                    T* __restrict__ dz, uint64_t ld_dz, float* __restrict__ partial) {
	constexpr uint32_t VEC = N2Vec<T>::SIZE, ROWS = 256u / LANES, COLUMNS = LANES * VEC;
	const uint32_t lane = threadIdx.x % LANES, column = blockIdx.x * COLUMNS + lane * VEC, group = threadIdx.x / LANES;
	const uint32_t n = n2_left<T>(width, column);
	float sum[VEC] = {};
	if (column < width) {
#pragma unroll 4
		for (uint64_t row = (uint64_t)blockIdx.y * ROWS + group; row < n_rows; row += (uint64_t)gridDim.y * ROWS) {
			const N2Vec<T> g = n2_load_vec_once<STREAM>(dy + row * ld_dy + column, n);
			N2Vec<T> out = {}, pre = {};
			if (kind != N2_ACTIVATION_NONE) pre = n2_load_vec_once<STREAM>(z + row * ld_z + column, n);
#pragma unroll
			for (uint32_t i = 0; i < VEC; ++i) {
				const float v = i < n ? slope_times((float)g.v[i], (float)pre.v[i], kind) : 0.f;
				sum[i] += v;
				out.v[i] = (T)v;
			}
			if (dz != nullptr) n2_store_vec(dz + row * ld_dz + column, out, VEC);
		}
	}
	if (partial == nullptr) return;
	__shared__ float fold[ROWS][COLUMNS + 4u];
#pragma unroll
	for (uint32_t i = 0; i < VEC; ++i) fold[group][lane * VEC + i] = sum[i];
	__syncthreads();
	for (uint32_t i = threadIdx.x; i < COLUMNS; i += 256u) {
		const uint32_t at = blockIdx.x * COLUMNS + i;
		float s = 0.f;
#pragma unroll
		for (uint32_t r = 0; r < ROWS; ++r) s += fold[r][i];
		if (at < width) partial[(uint64_t)blockIdx.y * width + at] = s;
	}
}

// an operand that can go into LDS without registers: pieces of 16 bytes at multiples of 16 bytes, offsets of a tile within 32 bits
bool async_operand(const Operand& o, bool kc, uint32_t extent, uint32_t k) {
	return reinterpret_cast<uintptr_t>(o.p) % 16 == 0 && o.ld % 8 == 0 && o.ld < (1u << 22) && (o.padded || (kc ? k : extent) % 8 == 0);
}

template <bool A_KC, bool B_KC>
bool async_product(const Product& q) { return async_operand(q.a, A_KC, q.extent_a, q.k) && async_operand(q.b, B_KC, q.extent_b, q.k); }

// how the product is cut, with `partial` for the sums of splits
void plan_product(Product& q, const N2LinearPlan& plan, float* partial) {
	if (q.extent_a == 0) q.extent_a = q.m;
	if (q.extent_b == 0) q.extent_b = q.n;
	q.tiles_m = n2_ceil_div(q.m, plan.tile), q.tiles_n = n2_ceil_div(q.n, plan.tile);
	q.splits = plan.splits, q.k_per_split = plan.k_per_split;
	q.partial = plan.splits > 1 ? partial : nullptr;
}
uint64_t blocks_of(const Product& q) { return (uint64_t)q.tiles_m * q.tiles_n * q.splits; }

template <typename T, bool A_KC, bool B_KC, int EPI>
int launch_product(hipStream_t s, const Product& all, uint32_t tile) {
	const auto launch_rows = [&](const Product& q) -> int {
		const dim3 grid((uint32_t)blocks_of(q));
		auto launch = [&](auto async, auto out) {
			constexpr bool ASYNC = decltype(async)::value;
			constexpr int OUT = decltype(out)::value;
			if (tile == 256) product_kernel<T, ASYNC, A_KC, B_KC, 256, 2, 4, EPI, OUT><<<grid, dim3(512), 0, s>>>(q);
			else if (tile == 128) product_kernel<T, ASYNC, A_KC, B_KC, 128, 2, 2, EPI, OUT><<<grid, dim3(256), 0, s>>>(q);
			else product_kernel<T, ASYNC, A_KC, B_KC, 64, 2, 2, EPI, OUT><<<grid, dim3(256), 0, s>>>(q);
		};
		auto with_out = [&](auto async) {
			if (q.partial != nullptr) launch(async, std::integral_constant<int, SPLIT>{});
			else launch(async, std::integral_constant<int, WHOLE>{});
		};
		if (async_product<A_KC, B_KC>(q)) with_out(std::true_type{});
		else with_out(std::false_type{});
		N2_LAUNCH_CHECK();
		return N2_OK;
	};
	// (where C's rows are widths, at most 65 536 of them, one launch takes all)
	const uint32_t most = A_KC ? n2_linear_launch_rows(all.m, tile, all.tiles_n, all.splits) : all.m;
	if (most >= all.m) return launch_rows(all);
	for (uint64_t first = 0; first < all.m; first += most) {
		Product q = all;
		q.m = q.extent_a = (uint32_t)(all.m - first < most ? all.m - first : most);
		q.tiles_m = n2_ceil_div(q.m, tile);
		q.a.p = static_cast<const T*>(all.a.p) + first * all.a.ld, q.c = static_cast<T*>(all.c) + first * all.ldc;
		if (all.residual != nullptr) q.residual = static_cast<const T*>(all.residual) + first * all.ldr;
		if (all.pre != nullptr) q.pre = static_cast<T*>(all.pre) + first * all.ldp;
		if (const int rc = launch_rows(q)) return rc;
	}
	return N2_OK;
}

// rows of whole vectors of eight values at multiples of 16 bytes (or nothing at all)
bool rows_of_vectors(const void* p, uint64_t stride, uint32_t width) { return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 8 == 0 && width % 8 == 0); }

// f(steps of 32 values of k, instructions of 16 columns) for widths up to 256
template <typename F>
void with_narrow(uint32_t k, uint32_t n, F&& f) {
	using std::integral_constant;
	auto with_n = [&](auto kt) {
		if (n <= 64u) f(kt, integral_constant<uint32_t, 4>{});
		else if (n <= 128u) f(kt, integral_constant<uint32_t, 8>{});
		else f(kt, integral_constant<uint32_t, 16>{});
	};
	if (k <= 64u) with_n(integral_constant<uint32_t, 2>{});
	else if (k <= 128u) with_n(integral_constant<uint32_t, 4>{});
	else with_n(integral_constant<uint32_t, 8>{});
}

template <typename F>
int with_type(n2_dtype dtype, F&& f) {
	return dtype == N2_DTYPE_F16 ? f(n2_f16{}) : f(n2_bf16{});
}

constexpr uint32_t MAX_WIDTH = 65536;

// what a backward pass keeps in its workspace, in this order
struct BackwardPlan {
	uint64_t ld_dz, dz_bytes, sums_bytes, partial_bytes, input_partial;
	uint32_t sum_blocks;
	N2LinearPlan input, weights;
};
BackwardPlan backward_plan(uint32_t n_rows, uint32_t in_width, uint32_t out_width) {
	BackwardPlan p = {};
	p.ld_dz = (uint64_t)n2_ceil_div(out_width, 8u) * 8u;
	p.dz_bytes = (n_rows * p.ld_dz * 2u + 15u) / 16u * 16u;
	p.sum_blocks = n2_linear_sum_blocks(n_rows, out_width);
	p.sums_bytes = ((uint64_t)p.sum_blocks * out_width * 4u + 15u) / 16u * 16u;
	p.input = n2_linear_plan(n_rows, in_width, out_width);
	p.weights = n2_linear_plan(out_width, in_width, n_rows);
	p.input_partial = n2_linear_partial_bytes(p.input, n_rows, in_width) / 4u;
	p.partial_bytes = p.input_partial * 4u + n2_linear_partial_bytes(p.weights, out_width, in_width);
	return p;
}

}  // namespace

#define LINEAR_CHECKS(name)                                                                                                                                \
	N2_REQUIRE(dtype == N2_DTYPE_F16 || dtype == N2_DTYPE_BF16, name ": type %d is neither fp16 nor bf16", (int)dtype);                                    \
	N2_REQUIRE((int)activation >= N2_ACTIVATION_NONE && (int)activation <= N2_ACTIVATION_GELU, name ": activation %d", (int)activation);                   \
	N2_REQUIRE(in_width >= 1 && in_width <= MAX_WIDTH && out_width >= 1 && out_width <= MAX_WIDTH, name ": widths %u, %u outside [1, %u]", in_width, out_width, MAX_WIDTH); \
	N2_REQUIRE(n_rows < (1u << 31), name ": %u rows, 2^31 - 1 are the most", n_rows)
#define STRIDE_CHECK(name, what, pointer, stride, width) \
	N2_REQUIRE((pointer) == nullptr || n_rows <= 1 || ((stride) >= (width) && n2_rows_fit(n_rows, stride)), name ": the stride of " what " is below the width %u or beyond memory", width)

N2_API uint64_t n2_linear_forward_workspace_bytes(uint32_t n_rows, uint32_t in_width, uint32_t out_width) {
	return n2_linear_few_rows(n_rows) || in_width == 0 || out_width == 0 ? 0u : n2_linear_partial_bytes(n2_linear_plan(n_rows, out_width, in_width), n_rows, out_width);
}

N2_API int n2_linear_forward(n2_stream_t stream, n2_dtype dtype, n2_activation activation, uint32_t n_rows, uint32_t in_width, uint32_t out_width, const void* d_weights,
                             const void* d_bias, const void* d_input, uint64_t input_stride, const void* d_residual, uint64_t residual_stride, void* d_output, uint64_t output_stride,
                             void* d_pre_activation, uint64_t pre_stride, void* d_workspace, uint64_t workspace_bytes) {
	LINEAR_CHECKS("n2_linear_forward");
	if (n_rows == 0) return N2_OK;
	N2_REQUIRE(d_weights && d_input && d_output, "n2_linear_forward: null buffer");
	STRIDE_CHECK("n2_linear_forward", "the input", d_input, input_stride, in_width);
	STRIDE_CHECK("n2_linear_forward", "the residual", d_residual, residual_stride, out_width);
	STRIDE_CHECK("n2_linear_forward", "the output", d_output, output_stride, out_width);
	STRIDE_CHECK("n2_linear_forward", "the saved values", d_pre_activation, pre_stride, out_width);
	const uint64_t needed = n2_linear_forward_workspace_bytes(n_rows, in_width, out_width);
	N2_REQUIRE(needed == 0 || (d_workspace && reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0 && workspace_bytes >= needed),
	           "n2_linear_forward: needs a 16-byte aligned workspace of %llu bytes, got %llu", (unsigned long long)needed, (unsigned long long)workspace_bytes);
	const bool in_place = d_residual == d_output && (n_rows == 1 || residual_stride == output_stride);
	const N2Rows written[3] = {n2_rows(d_output, n_rows, out_width, output_stride, 2), n2_rows(d_pre_activation, n_rows, out_width, pre_stride, 2), n2_vector(needed ? d_workspace : nullptr, needed, 1)};
	const N2Rows read[4] = {n2_vector(d_weights, (uint64_t)in_width * out_width, 2), n2_vector(d_bias, out_width, 2), n2_rows(d_input, n_rows, in_width, input_stride, 2),
	                        n2_rows(in_place ? nullptr : d_residual, n_rows, out_width, residual_stride, 2)};
	N2_REQUIRE(!n2_overlap(written, read), "n2_linear_forward: an output overlaps another buffer");
	Product q = {};
	q.a = {d_input, input_stride, false}, q.b = {d_weights, in_width, false};
	q.m = n_rows, q.n = out_width, q.k = in_width;
	q.c = d_output, q.ldc = output_stride;
	q.bias = d_bias, q.residual = d_residual, q.ldr = residual_stride, q.pre = d_pre_activation, q.ldp = pre_stride, q.activation = activation;
	const N2LinearPlan plan = n2_linear_few_rows(n_rows) ? N2LinearPlan{64, 1, in_width} : n2_linear_plan(n_rows, out_width, in_width);
	plan_product(q, plan, static_cast<float*>(d_workspace));
	return with_type(dtype, [&](auto t) -> int {
		using T = decltype(t);
		if (n2_linear_streams(n_rows, out_width, in_width) && async_product<true, true>(q) && rows_of_vectors(d_bias, 8, out_width) && rows_of_vectors(d_residual, residual_stride, out_width) &&
		    rows_of_vectors(d_output, output_stride, out_width) && rows_of_vectors(d_pre_activation, pre_stride, out_width)) {
			auto launch = [&](auto kt, auto nt) {
				constexpr uint32_t KT = decltype(kt)::value, NT = decltype(nt)::value;
				const dim3 grid(n2_linear_stream_blocks(n_rows, KT * NT * 1024u));
				if (d_residual != nullptr) stream_rows_kernel<T, KT, NT, true><<<grid, dim3(1024), 0, n2_stream(stream)>>>(q);
				else stream_rows_kernel<T, KT, NT, false><<<grid, dim3(1024), 0, n2_stream(stream)>>>(q);
			};
			with_narrow(in_width, out_width, launch);
			N2_LAUNCH_CHECK();
			return N2_OK;
		}
		if (n2_linear_few_rows(n_rows)) {
			few_rows_kernel<T><<<dim3(n2_ceil_div(out_width, 16u)), dim3(1024), 0, n2_stream(stream)>>>(q);
			N2_LAUNCH_CHECK();
			return N2_OK;
		}
		if (const int rc = launch_product<T, true, true, LAYER>(n2_stream(stream), q, plan.tile)) return rc;
		if (q.partial != nullptr) {
			join_kernel<T><<<dim3(join_blocks(q)), dim3(256), 0, n2_stream(stream)>>>(q);
			N2_LAUNCH_CHECK();
		}
		return N2_OK;
	});
}

N2_API uint64_t n2_linear_backward_workspace_bytes(uint32_t n_rows, uint32_t in_width, uint32_t out_width) {
	if (in_width < 1 || in_width > MAX_WIDTH || out_width < 1 || out_width > MAX_WIDTH) return 0;
	const BackwardPlan p = backward_plan(n_rows, in_width, out_width);
	return p.dz_bytes + p.sums_bytes + p.partial_bytes;
}

N2_API int n2_linear_backward(n2_stream_t stream, n2_dtype dtype, n2_activation activation, uint32_t n_rows, uint32_t in_width, uint32_t out_width, const void* d_weights,
                              const void* d_input, uint64_t input_stride, const void* d_pre_activation, uint64_t pre_stride, const void* d_dL_doutput, uint64_t dL_doutput_stride,
                              void* d_dL_dinput, uint64_t dL_dinput_stride, void* d_dL_dweights, void* d_dL_dbias, n2_grad_mode mode, void* d_workspace, uint64_t workspace_bytes) {
	LINEAR_CHECKS("n2_linear_backward");
	N2_REQUIRE(mode == N2_GRAD_IGNORE || mode == N2_GRAD_OVERWRITE || mode == N2_GRAD_ACCUMULATE, "n2_linear_backward: gradient mode %d", (int)mode);
	void* const dw = mode == N2_GRAD_IGNORE ? nullptr : d_dL_dweights;
	void* const db = mode == N2_GRAD_IGNORE ? nullptr : d_dL_dbias;
	if (activation == N2_ACTIVATION_NONE) d_pre_activation = nullptr;
	if (n_rows > 0) {
		N2_REQUIRE(d_weights && d_input && d_dL_doutput && (d_pre_activation || activation == N2_ACTIVATION_NONE), "n2_linear_backward: null buffer");
		STRIDE_CHECK("n2_linear_backward", "the input", d_input, input_stride, in_width);
		STRIDE_CHECK("n2_linear_backward", "the saved values", d_pre_activation, pre_stride, out_width);
		STRIDE_CHECK("n2_linear_backward", "the output's gradient", d_dL_doutput, dL_doutput_stride, out_width);
		STRIDE_CHECK("n2_linear_backward", "the input's gradient", d_dL_dinput, dL_dinput_stride, in_width);
	}
	const BackwardPlan p = backward_plan(n_rows, in_width, out_width);
	const uint64_t needed = p.dz_bytes + p.sums_bytes + p.partial_bytes;
	N2_REQUIRE(needed == 0 || (d_workspace && reinterpret_cast<uintptr_t>(d_workspace) % 16 == 0 && workspace_bytes >= needed),
	           "n2_linear_backward: needs a 16-byte aligned workspace of %llu bytes, got %llu", (unsigned long long)needed, (unsigned long long)workspace_bytes);
	const N2Rows written[4] = {n2_rows(d_dL_dinput, n_rows, in_width, dL_dinput_stride, 2), n2_vector(dw, (uint64_t)in_width * out_width, 2), n2_vector(db, out_width, 2),
	                           n2_vector(needed ? d_workspace : nullptr, needed, 1)};
	const N2Rows read[4] = {n2_vector(n_rows ? d_weights : nullptr, (uint64_t)in_width * out_width, 2), n2_rows(d_input, n_rows, in_width, input_stride, 2),
	                        n2_rows(d_pre_activation, n_rows, out_width, pre_stride, 2), n2_rows(d_dL_doutput, n_rows, out_width, dL_doutput_stride, 2)};
	N2_REQUIRE(!n2_overlap(written, read), "n2_linear_backward: an output overlaps another buffer");
	hipStream_t s = n2_stream(stream);
	const int accumulate = mode == N2_GRAD_ACCUMULATE ? 1 : 0;
	char* ws = static_cast<char*>(d_workspace);
	float* const sums = reinterpret_cast<float*>(ws + p.dz_bytes);
	float* const partial = reinterpret_cast<float*>(ws + p.dz_bytes + p.sums_bytes);
	return with_type(dtype, [&](auto t) -> int {
		using T = decltype(t);
		// dz: the output's gradient itself where there is no activation and its rows can go into LDS as they are
		const bool products = d_dL_dinput != nullptr || dw != nullptr, aligned = reinterpret_cast<uintptr_t>(d_dL_doutput) % 16 == 0 && dL_doutput_stride % 8 == 0 && out_width % 8 == 0;
		const bool writes = products && (activation != N2_ACTIVATION_NONE || !aligned);
		Operand dz = {d_dL_doutput, dL_doutput_stride, false};
		uint32_t sum_rows = n_rows > 0 ? p.sum_blocks : 0u;
		const bool has_x = d_dL_dinput != nullptr && n_rows > 0;
		// Narrow layers of many rows: dx by stream_backward_kernel.  It forms dz and sums its columns on the way where dz need not be stored; with the
		// store as well it took what two launches take (2^18 x 256 x 256 with ReLU 136 us for 73 and 62, 100 000 x 256 x 256 3 us more).  Where both
		// products fit one launch (product_pair_kernel) that is the faster way from a stored dz (50 000 x 200 x 136 45 us for 49).
		const bool small = p.input.tile == 64 && p.weights.tile == 64, forms_dz = activation == N2_ACTIVATION_NONE || dw == nullptr;
		const bool streams = has_x && n2_linear_streams(n_rows, in_width, out_width) && (forms_dz || !small) && rows_of_vectors(d_dL_doutput, dL_doutput_stride, out_width) &&
		                     rows_of_vectors(d_pre_activation, pre_stride, out_width) && rows_of_vectors(d_weights, in_width, in_width) && rows_of_vectors(d_dL_dinput, dL_dinput_stride, in_width);
		const bool forms = streams && forms_dz;
		if (!forms && n_rows > 0 && (writes || db != nullptr)) {
			if (writes) dz = {ws, p.ld_dz, true};
			const bool past_cache = writes && n2_linear_dz_streams(n_rows, in_width, out_width);
			auto launch = [&](auto lanes) {
				constexpr uint32_t LANES = decltype(lanes)::value;
				if (past_cache) slope_kernel<T, LANES, true><<<dim3(n2_ceil_div(out_width, LANES * 8u), p.sum_blocks), dim3(256), 0, s>>>(n_rows, out_width, static_cast<const T*>(d_dL_doutput), dL_doutput_stride,
					static_cast<const T*>(d_pre_activation), pre_stride, activation, writes ? reinterpret_cast<T*>(ws) : nullptr, p.ld_dz, db != nullptr ? sums : nullptr);
				else slope_kernel<T, LANES, false><<<dim3(n2_ceil_div(out_width, LANES * 8u), p.sum_blocks), dim3(256), 0, s>>>(n_rows, out_width, static_cast<const T*>(d_dL_doutput), dL_doutput_stride,
					static_cast<const T*>(d_pre_activation), pre_stride, activation, writes ? reinterpret_cast<T*>(ws) : nullptr, p.ld_dz, db != nullptr ? sums : nullptr);
			};
			if (out_width <= 64u) launch(std::integral_constant<uint32_t, 8>{});
			else if (out_width <= 128u) launch(std::integral_constant<uint32_t, 16>{});
			else if (out_width <= 256u) launch(std::integral_constant<uint32_t, 32>{});
			else launch(std::integral_constant<uint32_t, 64>{});
			N2_LAUNCH_CHECK();
		}
		if (streams) {
			Product q = {};
			q.a = dz, q.b = {d_weights, in_width, false};
			q.m = n_rows, q.n = in_width, q.k = out_width;
			q.c = d_dL_dinput, q.ldc = dL_dinput_stride, q.activation = activation;
			with_narrow(out_width, in_width, [&](auto kt, auto nt) {
				constexpr uint32_t KT = decltype(kt)::value, NT = decltype(nt)::value;
				const uint32_t blocks = n2_linear_stream_blocks(n_rows, KT * NT * 1024u);
				if (forms) sum_rows = blocks;
				stream_backward_kernel<T, KT, NT><<<dim3(blocks), dim3(1024), 0, s>>>(q, forms ? static_cast<const T*>(d_pre_activation) : nullptr, pre_stride, forms && db != nullptr ? sums : nullptr);
			});
			N2_LAUNCH_CHECK();
		}
		Product x = {}, w = {};
		if (has_x && !streams) {
			x.a = dz, x.b = {d_weights, in_width, false};
			x.m = n_rows, x.n = in_width, x.k = out_width;
			x.c = d_dL_dinput, x.ldc = dL_dinput_stride;
			plan_product(x, p.input, partial);
		}
		if (dw != nullptr) {
			w.a = dz, w.b = {d_input, input_stride, false};
			w.m = out_width, w.n = in_width, w.k = n_rows;
			if (dz.padded) w.extent_a = (uint32_t)p.ld_dz;
			w.c = dw, w.ldc = in_width, w.accumulate = accumulate;
			plan_product(w, p.weights, partial + p.input_partial);
		}
		const bool async = async_product<true, false>(x);
		if (has_x && !streams && dw != nullptr && small && async == async_product<false, false>(w) && blocks_of(x) + blocks_of(w) <= 0xFFFFFFFFull / 256u) {
			const dim3 grid((uint32_t)(blocks_of(x) + blocks_of(w)));
			if (async) product_pair_kernel<T, true><<<grid, dim3(256), 0, s>>>(x, w, (uint32_t)blocks_of(x));
			else product_pair_kernel<T, false><<<grid, dim3(256), 0, s>>>(x, w, (uint32_t)blocks_of(x));
			N2_LAUNCH_CHECK();
		} else {
			if (has_x && !streams)
				if (const int rc = launch_product<T, true, false, STORE>(s, x, p.input.tile)) return rc;
			if (dw != nullptr)
				if (const int rc = launch_product<T, false, false, GRADIENT>(s, w, p.weights.tile)) return rc;
		}
		const uint32_t blocks_x = join_blocks(x), blocks_w = join_blocks(w), blocks_b = db != nullptr ? n2_ceil_div(out_width, 16u) : 0u;
		if (blocks_x + blocks_w + blocks_b > 0) {
			join_backward_kernel<T><<<dim3(blocks_x + blocks_w + blocks_b), dim3(256), 0, s>>>(x, blocks_x, w, blocks_w, sums, sum_rows, out_width, static_cast<T*>(db), accumulate);
			N2_LAUNCH_CHECK();
		}
		return N2_OK;
	});
}
