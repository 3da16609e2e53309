// The layers' types: values of 16 or 32 bits in vectors of 16 bytes, and the sums over rows that their weights' gradients are.
#pragma once
#include "n2_common.h"

#include <type_traits>

typedef _Float16 n2_f16;
typedef __bf16 n2_bf16;

template <typename T>
struct N2Vec {
	static constexpr uint32_t SIZE = 16u / sizeof(T);
	T v[SIZE];
};

// Vectors that start at any element: the hardware takes 16 bytes from and to any address, so rows of odd widths and strides need no
// path of their own.  What a row's end leaves of a vector goes element by element.
template <typename T>
__device__ __forceinline__ N2Vec<T> n2_load_vec(const T* __restrict__ p, uint32_t valid) {
	N2Vec<T> r;
	if (valid >= N2Vec<T>::SIZE) {
		__builtin_memcpy(&r, p, 16);
	} else {
#pragma unroll
		for (uint32_t i = 0; i < N2Vec<T>::SIZE; ++i) r.v[i] = i < valid ? p[i] : (T)0.f;
	}
	return r;
}
template <typename T>
__device__ __forceinline__ void n2_store_vec(T* __restrict__ p, const N2Vec<T>& r, uint32_t valid) {
	if (valid >= N2Vec<T>::SIZE) {
		__builtin_memcpy(p, &r, 16);
	} else {
#pragma unroll
		for (uint32_t i = 0; i < N2Vec<T>::SIZE; ++i)
			if (i < valid) p[i] = r.v[i];
	}
}
typedef n2_u32x4 n2_u32x4_anywhere __attribute__((aligned(2)));
// n2_load_vec past the last-level cache (STREAM): for what is read once while something else is to stay there
template <bool STREAM, typename T>
__device__ __forceinline__ N2Vec<T> n2_load_vec_once(const T* __restrict__ p, uint32_t valid) {
	if (STREAM && valid >= N2Vec<T>::SIZE) return __builtin_bit_cast(N2Vec<T>, (n2_u32x4)__builtin_nontemporal_load(reinterpret_cast<const n2_u32x4_anywhere*>(p)));
	return n2_load_vec(p, valid);
}

// The vector at element `at` of a matrix whose last element is before `end`, zero from `valid` on.  Where a row's end leaves part of a vector
// the rest is read with it as long as the matrix goes on; a lane that reads element by element holds up its whole wave.
template <typename T>
__device__ __forceinline__ N2Vec<T> n2_load_row(const T* __restrict__ base, uint64_t at, uint64_t end, uint32_t valid) {
	if (at + N2Vec<T>::SIZE > end) return n2_load_vec(base + at, valid);
	N2Vec<T> r;
	__builtin_memcpy(&r, base + at, 16);
	if (valid < N2Vec<T>::SIZE) {
#pragma unroll
		for (uint32_t i = 0; i < N2Vec<T>::SIZE; ++i) r.v[i] = i < valid ? r.v[i] : (T)0.f;
	}
	return r;
}
// elements of a row of `width` from place `at` on, at most a vector
template <typename T>
__device__ __forceinline__ uint32_t n2_left(uint32_t width, uint32_t at) {
	return at < width ? min(width - at, N2Vec<T>::SIZE) : 0u;
}

// Sums over groups of 8, 16, 32 or 64 lanes, in all of them, without LDS: mirrors within the rows of 16 lanes, then whole rows change places.
template <uint32_t LANES>
__device__ __forceinline__ float n2_lane_sum(float x) {
	auto dpp = [](float v, auto control) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(control)::value, 0xf, 0xf, true)); };
	x += dpp(x, std::integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2
	x += dpp(x, std::integral_constant<int, 0x4E>{});   // quad_perm 2 3 0 1
	x += dpp(x, std::integral_constant<int, 0x141>{});  // row_half_mirror
	if constexpr (LANES >= 16u) x += dpp(x, std::integral_constant<int, 0x140>{});  // row_mirror
	auto sum = [](uint32_t a, uint32_t b) { return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b); };
	if constexpr (LANES >= 32u) {
		const uint32_t u = __builtin_bit_cast(uint32_t, x);
		const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
		x = sum(p[0], p[1]);
	}
	if constexpr (LANES >= 64u) {
		const uint32_t u = __builtin_bit_cast(uint32_t, x);
		const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
		x = sum(p[0], p[1]);
	}
	return x;
}

static inline uint32_t n2_dtype_bytes(uint32_t dtype) { return dtype == N2_DTYPE_F32 ? 4u : 2u; }

// Rows of a matrix that a call reads or writes, for the check that nothing is written over.  A vector is one row.
struct N2Rows {
	uintptr_t begin;
	uint64_t rows, width, stride;  // in bytes
};
static inline N2Rows n2_rows(const void* p, uint64_t rows, uint64_t width, uint64_t stride, uint64_t bytes) {
	if (p == nullptr || rows == 0 || width == 0) return {0, 0, 0, 0};
	return {reinterpret_cast<uintptr_t>(p), rows, width * bytes, rows == 1 ? width * bytes : stride * bytes};
}
static inline N2Rows n2_vector(const void* p, uint64_t n, uint64_t bytes) { return n2_rows(p, 1, n, n, bytes); }
static inline bool n2_rows_meet(const N2Rows& a, const N2Rows& b) {
	if (a.rows == 0 || b.rows == 0) return false;
	const uintptr_t a_end = a.begin + (a.rows - 1) * a.stride + a.width, b_end = b.begin + (b.rows - 1) * b.stride + b.width;
	if (a.begin >= b_end || b.begin >= a_end) return false;
	if (a.rows > 1 && b.rows > 1 && a.stride == b.stride) {  // columns side by side in one wider matrix
		const uint64_t d = b.begin >= a.begin ? (b.begin - a.begin) % a.stride : (a.stride - (a.begin - b.begin) % a.stride) % a.stride;
		if (d >= a.width && d + b.width <= a.stride) return false;
	}
	return true;
}
// one of `written` meets one of `read` or another one of `written`
template <int N, int M>
static inline bool n2_overlap(const N2Rows (&written)[N], const N2Rows (&read)[M]) {
	for (int i = 0; i < N; ++i) {
		for (int j = 0; j < i; ++j)
			if (n2_rows_meet(written[i], written[j])) return true;
		for (int j = 0; j < M; ++j)
			if (n2_rows_meet(written[i], read[j])) return true;
	}
	return false;
}
// the rows and the stride are addressable: the last byte lies below 2^63
static inline bool n2_rows_fit(uint64_t rows, uint64_t stride) { return rows == 0 || stride <= (1ull << 60) / rows; }
