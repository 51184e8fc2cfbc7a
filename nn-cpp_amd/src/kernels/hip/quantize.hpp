// quantize.hpp - a row's scale and its 8-bit codes (internal to libnnh).
//
// scale = max |x| / 127 rounded to 32 bits, code = the whole number nearest to x / scale, ties to even. The nearest is found by a
// product with the scale's reciprocal, which may be off by one in the last place, and put right by the rest x - code scale: a fused
// multiply-add gives it exactly where it decides, near half a scale (both have 24 bits, and the rest's bits lie above half the scale's
// last place). Rows of such a small scale that its reciprocal is not a number to work with divide in 64 bits.
#pragma once

#include <hip/hip_runtime.h>

#include "linear_int8.hpp"

namespace nnh {
namespace q8 {

template <typename T>
__device__ __forceinline__ float float_of(T x) { return (float)x; }

struct alignas(16) Word {
	unsigned x[4];
};

// Eight consecutive elements; those past D are zero.
template <typename T, bool VEC>
__device__ __forceinline__ void eight(float (&y)[8], const T* row, int at, int D) {
	if constexpr (VEC) {
		union {
			Word w[8 * sizeof(T) / 16];
			T e[8];
		} u;
#pragma unroll
		for (int i = 0; i < (int)(8 * sizeof(T) / 16); ++i) u.w[i] = ((const Word*)(row + at))[i];
#pragma unroll
		for (int i = 0; i < 8; ++i) y[i] = float_of(u.e[i]);
	} else {
#pragma unroll
		for (int i = 0; i < 8; ++i) y[i] = at + i < D ? float_of(row[at + i]) : 0.0f;
	}
}

// The largest |x|, infinity where one is not finite.
__device__ __forceinline__ float top_of(const float (&v)[8]) {
	float top = 0.0f;
	bool fine = true;
#pragma unroll
	for (int i = 0; i < 8; ++i) {
		top = fmaxf(top, fabsf(v[i]));  // (leaves NaN out)
		fine = fine && !(__float_as_uint(v[i]) << 1 >= 0xff000000u);
	}
	return fine ? top : __builtin_huge_valf();
}
// Of a thread's share of a row, eight elements at `at`, at + step, ...
template <typename T, bool VEC>
__device__ __forceinline__ float share_top(const T* x, int D, int at, int step) {
	float top = 0.0f, v[8];
	for (; at < D; at += step) {
		eight<T, VEC>(v, x, at, D);
		top = fmaxf(top, top_of(v));
	}
	return top;
}

struct Scale {
	float value, inv;
	bool none, small;
	__device__ __forceinline__ explicit Scale(float top) {
		const bool fine = top < __builtin_huge_valf();
		value = fine ? top / 127.0f : __builtin_nanf("");
		inv = 1.0f / value;
		none = !fine || value == 0.0f;
		small = value < 0x1p-100f;
	}
};

__device__ __forceinline__ int code_of(float x, float scale, float inv) {
	float n = rintf(x * inv);
	const float d = __builtin_fmaf(-n, scale, x), h = 0.5f * scale;
	const bool odd = ((int)n & 1) != 0;
	if (d > h || (d == h && odd)) n += 1.0f;
	if (d < -h || (d == -h && odd)) n -= 1.0f;
	return (int)n;
}

__device__ __forceinline__ uint64_t codes_of(const float (&v)[8], const Scale& s) {
	uint64_t w = 0;
	if (s.none) return w;
#pragma unroll
	for (int i = 0; i < 8; ++i) {
		// (a scale below the least normal number may be rounded down by more than its share: codes stay within 127)
		const int code = s.small ? (int)fmin(fmax(rint((double)v[i] / (double)s.value), -127.0), 127.0) : code_of(v[i], s.value, s.inv);
		w |= (uint64_t)(code & 255) << (8 * i);
	}
	return w;
}
// Eight codes from element `at` on, zeros past D.
template <typename T, bool VEC>
__device__ __forceinline__ uint64_t eight_codes(const T* x, int D, int at, const Scale& s) {
	if (at >= D) return 0;
	float v[8];
	eight<T, VEC>(v, x, at, D);
	return codes_of(v, s);
}

}  // namespace q8
}  // namespace nnh
