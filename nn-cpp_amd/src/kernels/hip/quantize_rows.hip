// quantize_rows.hip - rows to 8-bit codes with a scale each (linear_int8.hpp).
//
// scale = max |x| / 127 rounded to 32 bits, code = the whole number nearest to x / scale, ties to even. The nearest is found by a
// product with the scale's reciprocal, which may be off by one in the last place, and put right by the rest x - code scale: a fused
// multiply-add gives it exactly where it decides, near half a scale (both have 24 bits, and the rest's bits lie above half the scale's
// last place). Rows of such a small scale that its reciprocal is not a number to work with divide in 64 bits.
//
// Bound by memory: a row is read once for its maximum and again, from the caches, for its codes.
#include <cmath>

#include "linear_int8.hpp"

namespace nnh {

namespace {

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

__device__ __forceinline__ int code_of(float x, float scale, float inv) {
	float n = rintf(x * inv);
	const float d = __builtin_fmaf(-n, scale, x), h = 0.5f * scale;
	const bool odd = ((int)n & 1) != 0;
	if (d > h || (d == h && odd)) n += 1.0f;
	if (d < -h || (d == -h && odd)) n -= 1.0f;
	return (int)n;
}

// TPR threads to a row: a wave for short rows, a workgroup for others.
template <typename T, bool VEC, int TPR>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
	constexpr int kRows = 256 / TPR;
	__shared__ float part[4];
	const int t = threadIdx.x % TPR;
	const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
	const bool on = row < a.rows;
	const T* const x = (const T*)a.x + (on ? row : 0) * a.ldx;
	float top = 0.0f;
	bool fine = true;
	float v[8];
	for (int at = t * 8; at < a.D; at += TPR * 8) {
		eight<T, VEC>(v, x, at, a.D);
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			top = fmaxf(top, fabsf(v[i]));  // (leaves NaN out)
			fine = fine && !(__float_as_uint(v[i]) << 1 >= 0xff000000u);
		}
	}
	if (!fine) top = __builtin_huge_valf();
#pragma unroll
	for (int s = 32; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
	if (TPR > 64) {
		if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
		__syncthreads();
		top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
	}
	if (!on) return;
	fine = top < __builtin_huge_valf();
	const float scale = fine ? top / 127.0f : __builtin_nanf("");
	if (t == 0) a.scale[row] = scale;
	int8_t* const c = a.codes + row * a.ldc;
	const bool none = !fine || scale == 0.0f, small = scale < 0x1p-100f;
	const float inv = 1.0f / scale;
	for (int at = t * 8; at < a.pad; at += TPR * 8) {
		int code[8];
		if (at < a.D) {
			eight<T, VEC>(v, x, at, a.D);
#pragma unroll
			for (int i = 0; i < 8; ++i) {
				// (a scale below the least normal number may be rounded down by more than its share: codes stay within 127)
				if (small && !none) code[i] = (int)fmin(fmax(rint((double)v[i] / (double)scale), -127.0), 127.0);
				else code[i] = none ? 0 : code_of(v[i], scale, inv);
			}
		} else {
#pragma unroll
			for (int i = 0; i < 8; ++i) code[i] = 0;
		}
		if constexpr (VEC) {
			uint64_t w = 0;
#pragma unroll
			for (int i = 0; i < 8; ++i) w |= (uint64_t)(code[i] & 255) << (8 * i);
			*(uint64_t*)(c + at) = w;
		} else {
#pragma unroll
			for (int i = 0; i < 8; ++i)
				if (at + i < a.pad) c[at + i] = (int8_t)code[i];
		}
	}
}

template <typename T, bool VEC>
hipError_t launch(const QuantizeArgs& a, hipStream_t s) {
	if (a.D <= 1024) quantize_rows_kernel<T, VEC, 64><<<(unsigned)((a.rows + 3) / 4), 256, 0, s>>>(a);
	else quantize_rows_kernel<T, VEC, 256><<<(unsigned)a.rows, 256, 0, s>>>(a);
	return hipGetLastError();
}

}  // namespace

hipError_t quantize_rows(const QuantizeArgs& a, int type, hipStream_t s) {
	if (a.rows == 0) return hipSuccess;
	const int64_t size = type == kF32 ? 4 : 2;
	const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx * size % 16 == 0 && a.D % 8 == 0 && reinterpret_cast<uintptr_t>(a.codes) % 8 == 0 &&
	                 a.ldc % 8 == 0 && a.pad % 8 == 0;
	if (type == kF32) return vec ? launch<float, true>(a, s) : launch<float, false>(a, s);
	return vec ? launch<__bf16, true>(a, s) : launch<__bf16, false>(a, s);
}

}  // namespace nnh
