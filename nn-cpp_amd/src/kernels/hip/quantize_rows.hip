// quantize_rows.hip - rows to 8-bit codes with a scale each (quantize.hpp).
//
// Bound by memory: a row of up to 8192 elements is read once, into registers, a longer one once more, from the caches, for its codes.
// 8192 bf16 rows of 4096 take 24 us (100 MB, 4.3 TB/s); 32 of them 5 us, a launch and two trips to memory.
#include "quantize.hpp"

namespace nnh {

namespace {

// TPR threads to a row: a wave for short rows, a workgroup for others. A thread holds 8 HOLD elements (0: it reads them again).
template <typename T, bool VEC, int TPR, int HOLD>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantizeArgs a) {
	constexpr int kRows = 256 / TPR;
	__shared__ unsigned part[4];
	const int t = threadIdx.x % TPR;
	const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
	const bool on = row < a.rows;
	const T* const x = (const T*)a.x + (on ? row : 0) * a.ldx;
	float v[HOLD ? HOLD : 1][8];
	unsigned top = 0;
	if constexpr (HOLD > 0) {
#pragma unroll
		for (int k = 0; k < HOLD; ++k) {
			const int at = (k * TPR + t) * 8;
#pragma unroll
			for (int i = 0; i < 8; ++i) v[k][i] = 0.0f;
			if (at < a.D) q8::eight<T, VEC>(v[k], x, at, a.D);
		}
#pragma unroll
		for (int k = 0; k < HOLD; ++k) top = max(top, q8::top_of(v[k]));
	} else {
		top = q8::share_top<T, VEC>(x, a.D, t * 8, TPR * 8);
	}
#pragma unroll
	for (int s = 32; s; s >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, s));
	if (TPR > 64) {
		if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
		__syncthreads();
		top = max(max(part[0], part[1]), max(part[2], part[3]));
	}
	if (!on) return;
	const q8::Scale scale(top);
	if (t == 0) a.scale[row] = scale.value;
	int8_t* const c = a.codes + row * a.ldc;
	const auto store = [&](int at, uint64_t w) {
		if constexpr (VEC) {
			*(uint64_t*)(c + at) = w;
		} else {
#pragma unroll
			for (int i = 0; i < 8; ++i)
				if (at + i < a.pad) c[at + i] = (int8_t)(w >> (8 * i));
		}
	};
	if constexpr (HOLD > 0) {
#pragma unroll
		for (int k = 0; k < HOLD; ++k) {
			const int at = (k * TPR + t) * 8;
			if (at < a.pad) store(at, q8::codes_of(v[k], scale));
		}
	} else {
		for (int at = t * 8; at < a.pad; at += TPR * 8) store(at, q8::eight_codes<T, VEC>(x, a.D, at, scale));
	}
}

template <typename T, bool VEC>
hipError_t launch(const QuantizeArgs& a, hipStream_t s) {
	if (a.pad <= 1024) quantize_rows_kernel<T, VEC, 64, 2><<<(unsigned)((a.rows + 3) / 4), 256, 0, s>>>(a);
	else if (a.pad <= 8192) quantize_rows_kernel<T, VEC, 256, 4><<<(unsigned)a.rows, 256, 0, s>>>(a);
	else quantize_rows_kernel<T, VEC, 256, 0><<<(unsigned)a.rows, 256, 0, s>>>(a);
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
