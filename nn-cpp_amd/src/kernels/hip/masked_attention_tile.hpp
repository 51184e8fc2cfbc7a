// masked_attention_tile.hpp - the pieces that the masked attention kernels share: tiles in LDS, their matrix operands,
// and what a query sees.
//
// Products are 32 x 32 blocks of MFMA. The accumulator of a block has, in lane l, column l % 32 and rows
// 8 (i / 4) + 4 (l / 32) + i % 4 in register i; an operand of 16 depths has, in lane l, row (or column) l % 32 and the
// eight depths 8 (l / 32) + 0..7. A block's scores therefore go into the next product as they are, as the operand whose
// depth is the accumulator's row axis, when the other operand takes its depths in the same order: depth block t of lane
// half h is 16 t + 4 h + {0..3} and 16 t + 8 + 4 h + {0..3}. No probability moves between lanes.
//
// A tile is [row][RB bytes] in LDS, its 16-byte words permuted within a row so that both reads of it are free of bank
// conflicts: 16-byte words of 8 consecutive rows (an operand with the tile's rows as rows) and the transposed reads of 4
// rows by 64 bytes (an operand with the tile's rows as depth). Words move from memory into LDS without passing through
// registers, so the permutation is in what each lane loads.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "masked_attention.hpp"

namespace nnh {
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kInf = __builtin_huge_valf();

// 16 zero bytes that lanes without a word of their own load.
static __device__ const u32x4 kZeroWord = {0, 0, 0, 0};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__bf16 x) { return (float)x; }

// Eight consecutive depths of one operand row.
template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
	union {
		bf16x8 v;
		u32x4 w;
		s16x4 h[2];
		bf16x2 p[4];
		__bf16 e[8];
	};
};
template <>
struct Frag<float> {
	union {
		f32x4 h[2];
		u32x4 w2[2];
		float e[8];
	};
};

// acc += A B over 16 depths.
__device__ __forceinline__ void mma(f32x16& acc, const Frag<__bf16>& a, const Frag<__bf16>& b) {
	acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, acc, 0, 0, 0);
}
__device__ __forceinline__ void mma(f32x16& acc, const Frag<float>& a, const Frag<float>& b) {
#pragma unroll
	for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a.e[j], b.e[j], acc, 0, 0, 0);
}

// Registers 8 t .. 8 t + 7 of a block as an operand; in bf16 each value is rounded to the nearest once (the operand's
// type: its sum, and the statistics beside it, stay in fp32).
__device__ __forceinline__ void operand_of(Frag<__bf16>& f, const f32x16& x, int t) {
#pragma unroll
	for (int j = 0; j < 4; ++j) f.p[j] = __builtin_convertvector(f32x2{x[8 * t + 2 * j], x[8 * t + 2 * j + 1]}, bf16x2);
}
__device__ __forceinline__ void operand_of(Frag<float>& f, const f32x16& x, int t) {
#pragma unroll
	for (int j = 0; j < 8; ++j) f.e[j] = x[8 * t + j];
}

// Bytes of a tile's row: the power of two that holds DH elements.
template <typename T, int DH>
constexpr int row_bytes() {
	int b = 64;
	while (b < DH * (int)sizeof(T)) b *= 2;
	return b;
}

// Where the 16-byte word c of a row lives: c ^ swizzle(row).
template <int RB>
__device__ __forceinline__ int swizzle(int row) {
	if (RB == 64) return (row >> 2) & 3;
	if (RB == 128) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
	return (row & 3) << 2 | ((row >> 2) & 3);
}

// A lane's value that the compiler takes as new here: what follows from it is worked out again instead of being kept in
// registers over a whole loop, a dozen per constant added, until accumulators are spilled for them.
__device__ __forceinline__ int fresh(int x) {
	asm volatile("" : "+v"(x));
	return x;
}

// The lane's number, worked out anew for the same reason.
__device__ __forceinline__ int fresh_lane() {
	int x;
	asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(x));
	return x;
}

// Each lane's 16 (or 4) bytes at `src`, or at base + its offset, into LDS, 64 of them in a row from `to` (the wave's) on. Written
// out, since the compiler's own form makes it wait for every such load that is on its way before the next transposed read of
// any tile; the waits are the kernels' (wait_loads, and a barrier where waves share tiles). No vector
// register receives anything. m0 has the place in LDS and is named as overwritten: the compiler gives it to no value of its own
// (it is reserved, which the warning says), but its sequences that write m0 and read it again must not take one of these in between.
// `AT` bytes behind a place that the wave's loads have in common: one scalar register for all of them.
__device__ __forceinline__ unsigned lds_place(const char* to) {
	return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)to);
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int AT>
__device__ __forceinline__ void load_words(const void* src, unsigned to) {
	asm volatile("s_add_u32 m0, %0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(src), "i"(AT) : "m0", "scc");
}
template <int AT>
__device__ __forceinline__ void load_words(const void* base, unsigned offset, unsigned to) {
	// (a base that a vector instruction has just written, as one that reloads it does, may be read five wait states later)
	asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(offset), "s"(base), "i"(AT) : "m0", "scc");
}
__device__ __forceinline__ void load_numbers(const void* src, char* to) {
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_place(to)), "v"(src) : "m0");
}
#pragma clang diagnostic pop

// f(0) .. f(N - 1), the number a constant.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F f) {
	if constexpr (I < N) {
		f(std::integral_constant<int, I>{});
		each<N, I + 1>(f);
	}
}

// N products in groups of G, the operands of the next group on their way from LDS while one multiplies: read(i, f), product(i, f).
// Left to itself the compiler, short of registers elsewhere, reads each operand just before its product, which then waits for LDS
// every time.
template <typename F, int N, int G, typename Read, typename Product>
__device__ __forceinline__ void in_groups(Read read, Product product) {
	static_assert(N % G == 0, "whole groups");
	F f[2][G];
	each<G>([&](auto j) { read(decltype(j)::value, f[0][decltype(j)::value]); });
	each<N / G>([&](auto group) {
		constexpr int g = decltype(group)::value;
		if constexpr (g + 1 < N / G) each<G>([&](auto j) { read((g + 1) * G + decltype(j)::value, f[(g + 1) % 2][decltype(j)::value]); });
		each<G>([&](auto j) { product(g * G + decltype(j)::value, f[g % 2][decltype(j)::value]); });
		__builtin_amdgcn_sched_barrier(0);
	});
}
// Two operands of one product.
template <typename T>
struct FragPair {
	Frag<T> a, b;
};

// Loads a tile of R rows of `dh` elements from base + row * stride, NW waves sharing the work. Rows past the `live` (at least one)
// first ones, which nothing sees, are the last live one again, or zeros. VEC: every row is 16-byte aligned, dh a whole number
// of words and a tile's extent below 2^31 bytes (wide_row); then nothing passes through registers, and the caller waits
// for the loads (wait_loads). A load instruction fills 64 words, whole rows of them from a row that is a multiple of their number
// on: the permutation of a word is then the lane's own part XOR the wave's XOR the instruction's.
template <typename T, int DH, int R, int NW, bool VEC>
__device__ __forceinline__ void load_tile(char* tile, const T* base, int64_t stride, int live, int dh, int wave, int lane) {
	constexpr int RB = row_bytes<T, DH>(), W = RB / 16, E = 16 / (int)sizeof(T), kSteps = R * RB / 1024 / NW;
	static_assert(kSteps * NW * 1024 == R * RB, "a tile splits evenly over the waves");
	if constexpr (VEC) {
		lane = fresh_lane();
		constexpr int kRows = 64 / W;  // of a load; load j of a wave has rows (j * NW + wave) * kRows ..
		const int r = lane / W, w = (lane % W) ^ swizzle<RB>(r) ^ swizzle<RB>(wave * kRows);
		const unsigned pitch = (unsigned)(stride * (int64_t)sizeof(T)), at = r * pitch;
		const unsigned to = lds_place(tile + wave * 1024);
		const char* const from = (const char*)(base + (int64_t)(wave * kRows) * stride);
		if (live >= R && dh == DH) {
			each<kSteps>([&](auto step) {
				constexpr int j = decltype(step)::value;
				const int c = w ^ swizzle<RB>(j * NW * kRows);
				if (DH * (int)sizeof(T) == RB || c * E < DH) load_words<j * NW * 1024>(from + j * NW * kRows * (int64_t)pitch, at + c * 16, to);
			});
		} else {
			each<kSteps>([&](auto step) {
				constexpr int j = decltype(step)::value;
				const int c = w ^ swizzle<RB>(j * NW * kRows);
				const void* src = (const char*)base + (min((j * NW + wave) * kRows + r, live - 1) * pitch + c * 16);
				if (c * E >= dh) src = &kZeroWord;  // depths past dh multiply zeros: finite ones
				if (DH * (int)sizeof(T) == RB || c * E < DH) load_words<j * NW * 1024>(src, to);
			});
		}
	} else {
#pragma unroll
		for (int j = 0; j < kSteps; ++j) {
			const int first = (j * NW + wave) * 64, row = (first + lane) / W, c = ((first + lane) % W) ^ swizzle<RB>(row);
			union {
				T e[E];
				u32x4 w;
			} x;
#pragma unroll
			for (int i = 0; i < E; ++i) x.e[i] = row < live && c * E + i < dh ? base[row * stride + c * E + i] : (T)0.0f;
			*(u32x4*)(tile + (first + lane) * 16) = x.w;
		}
	}
}

// Every load into LDS that the wave has issued has arrived.
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }

// Values loaded before a loop are here before it begins. Where the first use of one is in the loop, the compiler's wait for it is
// there too, in every round, and waits for the tile that is on its way as well.
template <int N>
__device__ __forceinline__ void arrived(Frag<__bf16> (&f)[N]) {
#pragma unroll
	for (int t = 0; t < N; ++t) asm volatile("" : "+v"(f[t].w));
}
template <int N>
__device__ __forceinline__ void arrived(Frag<float> (&f)[N]) {
#pragma unroll
	for (int t = 0; t < N; ++t) asm volatile("" : "+v"(f[t].w2[0]), "+v"(f[t].w2[1]));
}
__device__ __forceinline__ void arrived() { __builtin_amdgcn_s_waitcnt(0x0070); }  // vmcnt(0) lgkmcnt(0), known to the compiler

// Whether any of the NW waves of a workgroup says so; flags: room for NW ints in the kernel's LDS.
template <int NW>
__device__ __forceinline__ bool any_wave(int* flags, int wave, int lane, bool x) {
	const int mine = __any(x);
	if (lane == 0) flags[wave] = mine;
	__syncthreads();
	int any = 0;
#pragma unroll
	for (int w = 0; w < NW; ++w) any |= flags[w];
	any = __builtin_amdgcn_readfirstlane(any);
	if (any) __syncthreads();  // the flags are written again
	return any != 0;
}

// Where a lane reads its operands in a tile of RB-byte rows. The permutation XORs a row's low bits onto its words' numbers, so
// with a lane's own part worked out once, every further step (depth, column block) is an XOR by a constant and every block of
// 16 or 32 rows a constant to add.
template <typename T, int RB>
struct Reader {
	int r, c;

	__device__ __forceinline__ explicit Reader(int lane) {
		const int col = lane & 31, half = lane >> 5, i = lane & 15;
		if constexpr (sizeof(T) == 2) {
			r = col * RB + ((half ^ swizzle<RB>(col)) * 16);
			const int row = 4 * half + (i >> 2);
			c = row * RB + (((2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ swizzle<RB>(row)) * 16) + (i & 1) * 8;
		} else {
			r = col * RB + (((2 * half) ^ swizzle<RB>(col)) * 16);
			c = 4 * half * RB + (((col >> 2) ^ half) * 16) + (col & 3) * 4;
		}
	}
	// Operand with the 32 rows from `at` on as rows: row lane % 32, depths 16 t + 8 half + 0..7.
	__device__ __forceinline__ void rows(Frag<T>& f, const char* at, int t) const {
		if constexpr (sizeof(T) == 2) {
			f.w = *(const u32x4*)(at + (r ^ (32 * t)));
		} else {
			f.w2[0] = *(const u32x4*)(at + (r ^ (64 * t)));
			f.w2[1] = *(const u32x4*)(at + (r ^ (64 * t) ^ 16));
		}
	}
	// Operand with the 16 rows from `at` on as depth, in the order of the accumulator's rows: 4 half + {0..3} and 8 + 4 half +
	// {0..3}, of column 32 block + lane % 32. In 16 bits one transposed read fetches, for each 16 lanes, 4 rows of 16 elements
	// (each lane naming 4 consecutive ones) and hands each lane a column of them.
	__device__ __forceinline__ void columns(Frag<T>& f, const char* at, int block) const {
		if constexpr (sizeof(T) == 2) {
			f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + (c ^ (64 * block))));
			f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * RB + (c ^ (64 * block) ^ 32)));
		} else {
#pragma unroll
			for (int j = 0; j < 8; ++j)
				f.e[j] = *(const float*)(at + (8 * (j >> 2) + (j & 3)) * RB + (c ^ (128 * block) ^ (64 * (j & 3)) ^ (32 * (j >> 2))));
		}
	}
};

// The same places kept in registers, one to a read, for kernels with room for them: a tile's own place is then part of the
// instruction, and no read costs an addition.
template <typename T, int DH>
struct Places {
	static constexpr int RB = row_bytes<T, DH>();
	int r[DH / 16], c[DH / 32][2];

	__device__ __forceinline__ explicit Places(int lane) {
		static_assert(sizeof(T) == 2, "16-bit types");
		const Reader<T, RB> at(lane);
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) r[t] = fresh(at.r ^ (32 * t));
#pragma unroll
		for (int b = 0; b < DH / 32; ++b) {
			c[b][0] = fresh(at.c ^ (64 * b));
			c[b][1] = fresh(at.c ^ (64 * b) ^ 32);
		}
	}
	__device__ __forceinline__ void rows(Frag<T>& f, const char* at, int t) const { f.w = *(const u32x4*)(at + r[t]); }
	__device__ __forceinline__ void columns(Frag<T>& f, const char* at, int block) const {
		f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + c[block][0]));
		f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * RB + c[block][1]));
	}
};

// One element of a tile.
template <typename T, int DH>
__device__ __forceinline__ float element_of(const char* tile, int row, int d) {
	constexpr int RB = row_bytes<T, DH>(), E = 16 / (int)sizeof(T);
	return to_float(*(const T*)(tile + row * RB + (((d / E) ^ swizzle<RB>(row)) * 16) + (d % E) * (int)sizeof(T)));
}

// Operand straight from memory: one row's depths 16 t + 8 half + 0..7, zeros past dh and where off.
template <typename T, bool VEC>
__device__ __forceinline__ void row_from(Frag<T>& f, const T* row, int dh, int half, int t, bool on) {
	const int d = 16 * t + 8 * half;
	if (VEC) {
		constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
		for (int x = 0; x < 8 / E; ++x) {
			u32x4 w = {0, 0, 0, 0};
			if (on && d + x * E < dh) w = *(const u32x4*)(row + d + x * E);
			if constexpr (sizeof(T) == 2) f.w = w;
			else f.w2[x] = w;
		}
	} else {
#pragma unroll
		for (int j = 0; j < 8; ++j) f.e[j] = on && d + j < dh ? row[d + j] : (T)0.0f;
	}
}

__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }
// Infinities and NaN out of an operand (the safe pass: see masked_attention_forward_kernel).
template <typename T>
__device__ __forceinline__ void only_finite(Frag<T>& f) {
#pragma unroll
	for (int j = 0; j < 8; ++j)
		if (not_finite(to_float(f.e[j]))) f.e[j] = (T)0.0f;
}

// x of the other half's lane with the same column, added to or maximised with the own.
__device__ __forceinline__ float max_halves(float x) {
	const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
	return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float x) {
	const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
	return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Rows of a block's column as they are stored in 16 bits: of the 16 elements 16 g .. 16 g + 15, of which a lane holds two runs of
// four (registers 8 g .. 8 g + 7 of a block), the lower half takes the first eight and the upper half the others.
__device__ __forceinline__ void eight_of(Frag<__bf16>& f) {
#pragma unroll
	for (int i = 0; i < 2; ++i) {
		const auto r = __builtin_amdgcn_permlane32_swap(f.w[i], f.w[2 + i], false, false);
		f.w[i] = r[0];
		f.w[2 + i] = r[1];
	}
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh(x). In 16 bits 1 - 2 / (1 + e^2x) with the hardware's reciprocal: off by about 1e-7 of 1, far below the operands'
// own rounding. In 32 bits the sum loses the small x's last bits, so below 0.55 the odd power series (to x^15, the rest is
// under 5e-8 of the value there), above it the quotient divided exactly.
template <typename T>
__device__ __forceinline__ float tanh_of(float x) {
	const float e = exp2_of(x * (2.0f * kLog2e));
	if constexpr (sizeof(T) == 2) {
		return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
	} else {
		const float y = x * x;
		float p = -929569.0f / 638512875.0f;
		p = __builtin_fmaf(p, y, 21844.0f / 6081075.0f);
		p = __builtin_fmaf(p, y, -1382.0f / 155925.0f);
		p = __builtin_fmaf(p, y, 62.0f / 2835.0f);
		p = __builtin_fmaf(p, y, -17.0f / 315.0f);
		p = __builtin_fmaf(p, y, 2.0f / 15.0f);
		p = __builtin_fmaf(p, y, -1.0f / 3.0f);
		return y < 0.3025f ? __builtin_fmaf(x * y, p, x) : 1.0f - 2.0f / (1.0f + e);
	}
}

// A block's range as scalars: read through the constant cache, so that no wait for a vector load waits for tiles on their way too
// (nothing writes the ranges while a kernel that reads them runs).
__device__ __forceinline__ DocRange range_at(const DocRange* ranges, int64_t i) {
	typedef const __attribute__((address_space(4))) int scalar_int;
	const scalar_int* p = (const scalar_int*)(uintptr_t)(ranges + i);
	return {p[0], p[1], p[2]};
}

// What one query sees of the keys: lo <= j < hi or j < pre, and its own document's. A query that is none (past the last
// row, or of no document) sees nothing.
struct Sight {
	int lo, hi, pre, doc;
	__device__ __forceinline__ bool sees(int j) const { return (j >= lo && j < hi) || j < pre; }
};

// The bounds of an int expression that may pass 2^31 (positions are at most 2^30 + 2^30).
__device__ __forceinline__ int clamped(int64_t x, int lo, int hi) { return (int)(x < lo ? lo : x > hi ? hi : x); }

__device__ __forceinline__ int live_keys(const MaskedAttentionArgs& a, int n) {
	return a.k_lens ? clamped(a.k_lens[n], 0, a.Tk) : a.Tk;
}
// The position of sample n's first query.
__device__ __forceinline__ int first_position(const MaskedAttentionArgs& a, int n) {
	return a.q_start ? clamped(a.q_start[n], -(1 << 30), 1 << 30) : 0;
}
__device__ __forceinline__ Sight sight_of(const MaskedAttentionArgs& a, int n, int i, int live, int pos0) {
	Sight s{0, 0, 0, 0};
	if (i >= a.Tq) return s;
	s.doc = a.q_docs ? a.q_docs[(int64_t)n * a.Tq + i] : 0;
	if (a.q_docs && s.doc < 0) return s;
	const int64_t pos = (int64_t)pos0 + i;
	s.hi = live;
	if (a.causal) s.hi = clamped(pos + 1, 0, live);
	if (a.window) {
		s.lo = clamped(pos - a.window + 1, 0, live);
		s.hi = min(s.hi, clamped(pos + a.window, 0, live));
	}
	if (a.prefix) s.pre = clamped(a.prefix[n], 0, live);
	return s;
}

}  // namespace attn
}  // namespace nnh
