// quantize.hpp - a row's scale and its 8-bit codes (internal to libnnh).
//
// scale = max |x| / 127 rounded to 32 bits, code = the whole number nearest to x / scale, ties to even. The nearest is found by a
// product with the scale's reciprocal, which may be off by one in the last place, and put right by the rest x - code scale: a fused
// multiply-add gives it exactly where it decides, near half a scale (both have 24 bits, and the rest's bits lie above half the scale's
// last place); most elements are nowhere near, which is seen first. Rows of such a small scale that its reciprocal is not a number to work with divide in 64 bits.
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

// The bits of the largest |x|; those of infinity or NaN are above every number's.
__device__ __forceinline__ unsigned top_of(const float (&v)[8]) {
	unsigned top = 0;
#pragma unroll
	for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
	return top;
}
// Of a thread's share of a row, eight elements at `at`, at + step, ...
template <typename T, bool VEC>
__device__ __forceinline__ unsigned share_top(const T* x, int D, int at, int step) {
	unsigned top = 0;
	float v[8];
	for (; at < D; at += step) {
		eight<T, VEC>(v, x, at, D);
		top = max(top, top_of(v));
	}
	return top;
}

struct Scale {
	float value, inv;
	bool none, small;
	__device__ __forceinline__ explicit Scale(unsigned top) {
		const bool fine = top < 0x7f800000u;
		value = fine ? __uint_as_float(top) / 127.0f : __builtin_nanf("");
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
	if (!s.small) {
		// x inv is within 2^-16 of x / scale: where no element lies that near to the middle of two whole numbers, a sum with 1.5 2^23 rounds
		// to the right one and leaves the code in its lowest byte
		unsigned y[8];
		float far = 0.0f;
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			const float sum = __builtin_fmaf(v[i], s.inv, 0x1.8p23f);
			far = fmaxf(far, fabsf(__builtin_fmaf(v[i], s.inv, 0x1.8p23f - sum)));
			y[i] = __float_as_uint(sum);
		}
		if (far < 0.5f - 0x1p-15f) {
			const auto four = [](unsigned a, unsigned b, unsigned c, unsigned d) {
				return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
			};
			return (uint64_t)four(y[4], y[5], y[6], y[7]) << 32 | four(y[0], y[1], y[2], y[3]);
		}
	}
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
