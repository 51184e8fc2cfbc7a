// adamw.hip - AdamW's kernel (adamw.hpp).
//
// Bound by memory: every element is read and written once, four consecutive elements a thread (a 16-byte word of an fp32
// tensor), so that a block of 64 elements is a row of 16 lanes and its maximum takes four DPP steps. A launch takes the
// tensors by value in its arguments (no table in device memory to keep up to date, and a captured launch keeps its own), as
// many as fit; a workgroup finds its tensor by its number.
//
// 8-bit moments: m as an e4m3 code times a power of two per block of 64, sqrt(v) the same way. The power is the one that
// brings the block's largest value into [128, 256), which an exponent decides alone. The square root halves v's range of
// exponents: 2^-9 .. 256 hold 2^34 of v. A second moment that is not zero never becomes zero (its root rounds to the
// smallest code at least), or an element whose gradient is far below its block's largest would divide by eps alone. The
// moments before rounding are computed in 64 bits, so that a code is the nearest one to the formula's value and not a
// neighbour's that fp32 would round to; the update itself takes them before they are rounded to codes.
// An infinite or NaN moment becomes e4m3's NaN and leaves its block's scale to the others.
//
// Measured: 8-bit moments of 16-bit gradients and 32-bit parameters with a bf16 copy, 6.5 GB a step, 1548 us (4.2 TB/s; a
// large copy reaches 4.7). A step of 0.1 million parameters is one launch of 7 us, 11 us a step from Python.
#include "adamw.hpp"

#include <cmath>

namespace nnh {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

constexpr int kTensors = 52, kThreads = 256, kSteps = 4, kPerBlock = kThreads * 4 * kSteps;

struct Batch {
	AdamWArgs a;
	AdamWTensor t[kTensors];
	unsigned begin[kTensors + 1];  // each tensor's first workgroup
	uint64_t wide;                 // bit i: tensor i's pointers take words of four elements
	int n;
};
static_assert(sizeof(Batch) <= 4096, "kernel arguments");

template <typename T>
struct Four;
template <>
struct Four<float> {
	typedef f32x4 V;
};
template <>
struct Four<__bf16> {
	typedef bf16x4 V;
};

template <typename T>
__device__ __forceinline__ void load4(float* x, const T* p, int live, bool wide) {
	if (wide) {
		const typename Four<T>::V v = *(const typename Four<T>::V*)p;
#pragma unroll
		for (int i = 0; i < 4; ++i) x[i] = (float)v[i];
	} else {
#pragma unroll
		for (int i = 0; i < 4; ++i) x[i] = i < live ? (float)p[i] : 0.0f;
	}
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* x, int live, bool wide) {
	if (wide) {
		typename Four<T>::V v;
#pragma unroll
		for (int i = 0; i < 4; ++i) v[i] = (T)x[i];
		*(typename Four<T>::V*)p = v;
	} else {
#pragma unroll
		for (int i = 0; i < 4; ++i)
			if (i < live) p[i] = (T)x[i];
	}
}

__device__ __forceinline__ double two_to(int e) { return __hiloint2double((e + 1023) << 20, 0); }
// The biased exponent of |x|.
__device__ __forceinline__ int exponent_of(double x) { return (__double2hiint(x) & 0x7fffffff) >> 20; }

// The largest of a row of 16 lanes, in all of them.
__device__ __forceinline__ int row_max(int x) {
	x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false));
	x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false));
	x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false));
	return max(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false));
}

// x, below 257 in magnitude, to the nearest e4m3 value, ties to even: adding 1.5 2^52 of its steps leaves whole steps.
__device__ __forceinline__ float nearest_e4m3(double x) {
	const int e = max(exponent_of(x), 1023 - 6);
	const double c = __hiloint2double((e - 3 + 52) << 20 | 0x80000, 0);
	return (float)((x + c) - c);
}

// The stored exponent of a block whose largest value has biased exponent `top` (0: nothing but zeros).
__device__ __forceinline__ int scale_of(int top) { return top == 0 ? 0 : min(max(top - 1022 - 8 + 127, 0), 254); }

__device__ __forceinline__ uint32_t codes_of(const float* y) {
	int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
	return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}

template <typename P, typename G, int BITS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Batch b) {
	int at = 0;
	for (int step = 32; step; step /= 2)  // the last tensor that begins at or before this workgroup
		if (at + step < b.n && b.begin[at + step] <= blockIdx.x) at += step;
	const AdamWTensor t = b.t[at];
	const bool wide = b.wide >> at & 1;
	double first = b.a.first, second = b.a.second;
	if (b.a.step_device) {
		const double step = (double)*b.a.step_device;
		first = 1.0 - exp2(step * b.a.log1);
		second = 1.0 - exp2(step * b.a.log2);
	}
	const double lr = b.a.lr_device ? (double)*b.a.lr_device : b.a.lr;
	const float keep = (float)(1.0 - lr * b.a.decay), rate = (float)(lr / first), inv = (float)(1.0 / sqrt(second)), eps = (float)b.a.eps;
	const float scale = b.a.grad_scale ? *b.a.grad_scale : 1.0f;
	const int64_t base = (int64_t)(blockIdx.x - b.begin[at]) * kPerBlock + threadIdx.x * 4;
#pragma unroll
	for (int s = 0; s < kSteps; ++s) {
		const int64_t i = base + (int64_t)s * kThreads * 4;
		const int live = (int)min(t.count - i, (int64_t)4);  // a whole row of 16 lanes stays together for its maximum
		if (t.count - (i - (threadIdx.x & 15) * 4) <= 0) break;
		const bool w = wide && live == 4;
		float p[4] = {}, g[4] = {}, m[4], v[4];
		if (live > 0) {
			load4(p, (const P*)t.p + i, live, w);
			load4(g, (const G*)t.g + i, live, w);
		}
		if constexpr (BITS == 32) {
			if (live <= 0) continue;
			load4(m, (const float*)t.m + i, live, w);
			load4(v, (const float*)t.v + i, live, w);
			const float b1 = (float)b.a.beta1, b2 = (float)b.a.beta2, c1 = (float)(1.0 - b.a.beta1), c2 = (float)(1.0 - b.a.beta2);
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				g[j] *= scale;
				m[j] = __builtin_fmaf(b1, m[j], c1 * g[j]);
				v[j] = __builtin_fmaf(b2, v[j], c2 * (g[j] * g[j]));
			}
			store4((float*)t.m + i, m, live, w);
			store4((float*)t.v + i, v, live, w);
		} else {
			uint32_t cm = 0, cv = 0;
			int sm = 0, sv = 0;
			if (live > 0) {
				if (w) {
					cm = *(const uint32_t*)((const uint8_t*)t.m + i);
					cv = *(const uint32_t*)((const uint8_t*)t.v + i);
				} else {
					for (int j = 0; j < live; ++j) {
						cm |= (uint32_t)((const uint8_t*)t.m)[i + j] << 8 * j;
						cv |= (uint32_t)((const uint8_t*)t.v)[i + j] << 8 * j;
					}
				}
				sm = t.m_scale[i >> 6];
				sv = t.v_scale[i >> 6];
			}
			const f32x2 m01 = __builtin_amdgcn_cvt_pk_f32_fp8(cm, false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(cm, true);
			const f32x2 r01 = __builtin_amdgcn_cvt_pk_f32_fp8(cv, false), r23 = __builtin_amdgcn_cvt_pk_f32_fp8(cv, true);
			const float om[4] = {m01[0], m01[1], m23[0], m23[1]}, orr[4] = {r01[0], r01[1], r23[0], r23[1]};
			const double um = two_to(sm - 127), uv = two_to(sv - 127), c1 = 1.0 - b.a.beta1, c2 = 1.0 - b.a.beta2;
			double dm[4], dv[4];
			int tm = 0, tv = 0;
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const double gd = (double)g[j] * (double)scale, r = (double)orr[j] * uv;
				dm[j] = b.a.beta1 * ((double)om[j] * um) + c1 * gd;
				dv[j] = b.a.beta2 * (r * r) + c2 * (gd * gd);
				const int em = exponent_of(dm[j]), ev = exponent_of(dv[j]);
				tm = em < 2047 ? max(tm, em) : tm;
				tv = ev < 2047 ? max(tv, ev) : tv;
				m[j] = (float)dm[j];
				v[j] = (float)dv[j];
			}
			tm = row_max(tm);
			tv = row_max(tv);
			// v in [2^(k - 1), 2^k) has its root in [2^(h - 1), 2^h) with h = ceil(k / 2)
			const int hm = scale_of(tm), hv = tv == 0 ? 0 : scale_of(((tv - 1022 + 1) >> 1) + 1022);
			const double im = two_to(127 - hm), iv = two_to(127 - hv);
			float ym[4], yv[4];
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				ym[j] = nearest_e4m3(dm[j] * im);
				const double r = sqrt(dv[j]) * iv;
				yv[j] = nearest_e4m3(r);
				if (r > 0.0 && yv[j] == 0.0f) yv[j] = 0.001953125f;
				if (exponent_of(dm[j]) == 2047) ym[j] = __builtin_nanf("");
				if (exponent_of(dv[j]) == 2047) yv[j] = __builtin_nanf("");
			}
			if (live <= 0) continue;
			cm = codes_of(ym);
			cv = codes_of(yv);
			if (w) {
				*(uint32_t*)((uint8_t*)t.m + i) = cm;
				*(uint32_t*)((uint8_t*)t.v + i) = cv;
			} else {
				for (int j = 0; j < live; ++j) {
					((uint8_t*)t.m)[i + j] = (uint8_t)(cm >> 8 * j);
					((uint8_t*)t.v)[i + j] = (uint8_t)(cv >> 8 * j);
				}
			}
			if ((threadIdx.x & 15) == 0) {
				t.m_scale[i >> 6] = (uint8_t)hm;
				t.v_scale[i >> 6] = (uint8_t)hv;
			}
		}
#pragma unroll
		for (int j = 0; j < 4; ++j) p[j] = p[j] * keep - rate * (m[j] / (sqrtf(v[j]) * inv + eps));
		store4((P*)t.p + i, p, live, w);
		if (t.copy) store4((__bf16*)t.copy + i, p, live, w);
	}
}

template <typename P, typename G>
hipError_t launch(const Batch& b, unsigned blocks, int bits, hipStream_t s) {
	if (bits == 32) adamw_kernel<P, G, 32><<<blocks, kThreads, 0, s>>>(b);
	else adamw_kernel<P, G, 8><<<blocks, kThreads, 0, s>>>(b);
	return hipGetLastError();
}

}  // namespace

hipError_t adamw_step(const AdamWArgs& a, const AdamWTensor* tensors, size_t n, int p_type, int g_type, int bits, hipStream_t s) {
	constexpr uint64_t kMaxBlocks = (1u << 24) - 1;  // of 256 work-items, below 2^32 together
	Batch b{};
	b.a = a;
	uint64_t blocks = 0;
	auto flush = [&]() -> hipError_t {
		if (b.n == 0) return hipSuccess;
		b.begin[b.n] = (unsigned)blocks;
		const unsigned x = (unsigned)blocks;
		hipError_t e;
		if (p_type == 0) e = g_type == 0 ? launch<float, float>(b, x, bits, s) : launch<float, __bf16>(b, x, bits, s);
		else e = g_type == 0 ? launch<__bf16, float>(b, x, bits, s) : launch<__bf16, __bf16>(b, x, bits, s);
		b.n = 0;
		b.wide = 0;
		blocks = 0;
		return e;
	};
	for (size_t i = 0; i < n; ++i) {
		AdamWTensor t = tensors[i];
		const size_t ps = p_type == 0 ? 4 : 2, gs = g_type == 0 ? 4 : 2;
		while (t.count > 0) {
			const uint64_t room = kMaxBlocks - blocks;
			if (b.n == kTensors || room == 0) {
				const hipError_t e = flush();
				if (e != hipSuccess) return e;
				continue;
			}
			AdamWTensor part = t;
			part.count = (int64_t)(room * kPerBlock) < t.count ? (int64_t)(room * kPerBlock) : t.count;
			const auto on = [](const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; };
			const size_t ss = bits == 32 ? 16 : 4;
			if (on(t.p, 4 * ps) && on(t.g, 4 * gs) && on(t.m, ss) && on(t.v, ss) && on(t.copy, 8)) b.wide |= (uint64_t)1 << b.n;
			b.begin[b.n] = (unsigned)blocks;
			b.t[b.n++] = part;
			blocks += ((uint64_t)part.count + kPerBlock - 1) / kPerBlock;
			t.count -= part.count;
			t.p = (char*)t.p + part.count * ps;
			t.g = (const char*)t.g + part.count * gs;
			t.m = (char*)t.m + part.count * (bits == 32 ? 4 : 1);
			t.v = (char*)t.v + part.count * (bits == 32 ? 4 : 1);
			if (bits == 8) {
				t.m_scale += part.count / 64;
				t.v_scale += part.count / 64;
			}
			if (t.copy) t.copy = (char*)t.copy + part.count * 2;
		}
	}
	return flush();
}

}  // namespace nnh
