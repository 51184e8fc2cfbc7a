// linear_int8_tile.hpp - products of 8-bit codes on the matrix cores (linear_int8.hpp).
//
// y[row][col] = sum over depth of W[col][depth] X[row][depth]. Both operands have their depth contiguous, and 32 of their codes are
// the 32 bytes that 16 depths of a bf16 product take: tiles, ring, loads and reads of LDS are gemm16.hpp's, in units of two codes, and
// an MFMA of 32 x 32 x 32 does twice the depth in the same time. The bounds are the same too, with twice the operations: 8192 rows,
// 4096 deep, 16384 columns take 490 to 520 us (2110 to 2240 TOP/s; the library's product of such codes 2126).
#pragma once

#include "gemm16.hpp"
#include "linear_int8.hpp"
#include "quantize.hpp"

namespace nnh {
namespace i8 {

typedef int i32x16 __attribute__((ext_vector_type(16)));
using attn::f32x2;
using attn::f32x4;
using attn::Frag;
using attn::i32x4;
using attn::u32x4;
using attn::bf16x2;

__device__ __forceinline__ void mma(i32x16& acc, const Frag<__bf16>& a, const Frag<__bf16>& b) {
	union {
		u32x4 w;
		i32x4 i;
	} x{a.w}, y{b.w};
	acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(x.i, y.i, acc, 0, 0, 0);
}

// What a sum becomes: one rounding to 32 bits (sums are whole numbers below 2^31), one for each scale, one for the bias.
__device__ __forceinline__ float scaled(int sum, float x_scale, float w_scale, float bias) { return (float)sum * x_scale * w_scale + bias; }

template <typename T>
__device__ __forceinline__ float bias_at(const LinearInt8Args& a, int col) { return a.bias ? attn::to_float(((const T*)a.bias)[col]) : 0.0f; }

template <class S, typename T>
__global__ __launch_bounds__(S::kThreads, 2) void linear_int8_tile_kernel(LinearInt8Args a) {
	constexpr int BM = S::BM, BN = S::BN, WM = S::WM, WN = S::WN, I = WM / 32, J = WN / 32, NW = S::kWaves, BK = g16::BK;
	__shared__ __attribute__((aligned(1024))) char lds[S::kLds];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5, wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
	int m0, n0, from = 0, depth = (a.D + 15) / 16 * 8;  // in units of two codes
	g16::tile_of((a.V + BM - 1) / BM, (a.rows + BN - 1) / BN, m0, n0);
	m0 *= BM;
	n0 *= BN;
	if (a.parts) {
		from = blockIdx.y * a.part_units;
		depth = min(depth - from, a.part_units);
	}
	g16::Loader<BM, NW, false> la;
	g16::Loader<BN, NW, false> lb;
	la.begin((const __bf16*)a.w + from, a.ldw / 2, m0, a.V, wave, lane);
	lb.begin((const __bf16*)a.x + from, a.ldx / 2, n0, a.rows, wave, lane);
	i32x16 acc[I][J];
#pragma unroll
	for (int i = 0; i < I; ++i)
#pragma unroll
		for (int j = 0; j < J; ++j)
#pragma unroll
			for (int x = 0; x < 16; ++x) acc[i][j][x] = 0;

	const g16::Reader<BM, false> ra(wm, lane);
	const g16::Reader<BN, false> rb(wn, lane);
	const int stages = (depth + BK - 1) / BK;
	Frag<__bf16> fa[2][I], fb[2][J];
	auto read = [&](int set, const char* x, const char* y, int t) {
#pragma unroll
		for (int i = 0; i < I; ++i) ra.read(fa[set][i], x, i, t);
#pragma unroll
		for (int j = 0; j < J; ++j) rb.read(fb[set][j], y, j, t);
	};
	auto multiply = [&](int set, auto load) {
		constexpr int kReads = I + J;
		attn::each<I * J>([&](auto at) {
			constexpr int x = decltype(at)::value, per = I * J / S::kLoads;
			mma(acc[x / J][x % J], fa[set][x / J], fb[set][x % J]);
			if constexpr (x % per == per - 1) load(std::integral_constant<int, x / per>{});
		});
#pragma unroll
		for (int x = 0; x < I * J; ++x) {
			__builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
			__builtin_amdgcn_sched_group_barrier(0x100, (kReads + I * J - 1) / (I * J), 0);
		}
		__builtin_amdgcn_sched_barrier(0);
	};
	// The ring of five half stages and the order of its loads and waits: as in gemm16_kernel.
	auto place = [&](int x) { return lds + x % 5 * S::kHalf; };
	auto load_a = [&](auto j, int x, int s) { la.template load<decltype(j)::value>(place(x), depth - s * BK, wave, lane); };
	auto load_b = [&](auto j, int x, int s) { lb.template load<decltype(j)::value>(place(x), depth - s * BK, wave, lane); };
	auto step = [&](int s, auto mod) {
		constexpr int M = decltype(mod)::value;
		read(1, place(2 * M), place(2 * M + 1), 1);
		multiply(0, [&](auto j) { load_a(j, 2 * M + 4, s + 2); });
#pragma unroll
		for (int t = 1; t < BK / 16 - 1; ++t) {
			read(~t & 1, place(2 * M), place(2 * M + 1), t + 1);
			multiply(t & 1, [](auto) {});
		}
		asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(S::kLoads) : "memory");
		__builtin_amdgcn_s_barrier();
		asm volatile("" ::: "memory");
		read(0, place(2 * M + 2), place(2 * M + 3), 0);
		multiply(1, [&](auto j) { load_b(j, 2 * M, s + 2); });
	};
#pragma unroll
	for (int s = 0; s < 2; ++s) {
		attn::each<S::kLoads>([&](auto j) { load_a(j, 2 * s, s); });
		attn::each<S::kLoads>([&](auto j) { load_b(j, 2 * s + 1, s); });
	}
	asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * S::kLoads) : "memory");
	__builtin_amdgcn_s_barrier();
	asm volatile("" ::: "memory");
	read(0, place(0), place(1), 0);
	for (int s = 0; s < stages; s += 5) {
		step(s, std::integral_constant<int, 0>{});
		if (s + 1 < stages) step(s + 1, std::integral_constant<int, 1>{});
		if (s + 2 < stages) step(s + 2, std::integral_constant<int, 2>{});
		if (s + 3 < stages) step(s + 3, std::integral_constant<int, 3>{});
		if (s + 4 < stages) step(s + 4, std::integral_constant<int, 4>{});
	}
	attn::wait_loads();
	__syncthreads();  // LDS is the output tile's from here on

	// register 4 g + x of block (i, j): column m0 + wm + 32 i + 8 g + 4 half + x, row n0 + wn + 32 j + col
	const int mw = m0 + wm + 4 * half;
	if (a.parts) {
#pragma unroll
		for (int j = 0; j < J; ++j) {
			const int n = n0 + wn + 32 * j + col;
			if (n >= a.rows) continue;
			int* const o = a.parts + ((int64_t)blockIdx.y * a.rows + n) * a.V;
#pragma unroll
			for (int i = 0; i < I; ++i)
#pragma unroll
				for (int x = 0; x < 16; ++x) {
					const int m = mw + 32 * i + 8 * (x / 4) + x % 4;
					if (m < a.V) o[m] = acc[i][j][x];
				}
		}
		return;
	}
	float xs[J];
#pragma unroll
	for (int j = 0; j < J; ++j) xs[j] = a.x_scale[min(n0 + wn + 32 * j + col, a.rows - 1)];
	constexpr int W = BM / 8;  // 16-byte words of 16-bit results to a row
	__bf16* const tile = (__bf16*)lds;
	const bool through = sizeof(T) == 2 && a.whole_words;
#pragma unroll
	for (int i = 0; i < I; ++i)
#pragma unroll
		for (int g = 0; g < 4; ++g) {
			const int m = mw + 32 * i + 8 * g;
			float ws[4], b[4];
#pragma unroll
			for (int x = 0; x < 4; ++x) {
				ws[x] = a.w_scale[min(m + x, a.V - 1)];
				b[x] = bias_at<T>(a, min(m + x, a.V - 1));
			}
#pragma unroll
			for (int j = 0; j < J; ++j) {
				float y[4];
#pragma unroll
				for (int x = 0; x < 4; ++x) y[x] = scaled(acc[i][j][4 * g + x], xs[j], ws[x], b[x]);
				const int n = n0 + wn + 32 * j + col;
				if constexpr (sizeof(T) == 2) {
					if (through) {  // through LDS, 16-byte words permuted by row, for stores of whole rows
						union {
							bf16x2 p[2];
							uint64_t w;
						} z;
						z.p[0] = __builtin_convertvector(f32x2{y[0], y[1]}, bf16x2);
						z.p[1] = __builtin_convertvector(f32x2{y[2], y[3]}, bf16x2);
						const int r = wn + 32 * j + col;
						*(uint64_t*)(tile + r * BM + ((((wm + 32 * i + 8 * g) / 8) ^ (r % W)) * 8) + 4 * half) = z.w;
						continue;
					}
				}
				if (n >= a.rows) continue;
				T* const o = (T*)a.y + (int64_t)n * a.ldy + m;
				if (sizeof(T) == 4 && a.whole_words) {
					if (m < a.V) *(f32x4*)o = f32x4{y[0], y[1], y[2], y[3]};
				} else {
#pragma unroll
					for (int x = 0; x < 4; ++x)
						if (m + x < a.V) o[x] = (T)y[x];
				}
			}
		}
	if (through) {
		__syncthreads();
		for (int w = threadIdx.x; w < BN * W; w += S::kThreads) {
			const int r = w / W, c = w % W;
			if (n0 + r < a.rows && m0 + c * 8 < a.V)
				*(u32x4*)((__bf16*)a.y + (int64_t)(n0 + r) * a.ldy + m0 + c * 8) = *(const u32x4*)(tile + r * BM + ((c ^ (r % W)) * 8));
		}
	}
}

// The runs' sums to results, a thread to an element.
template <typename T>
__global__ __launch_bounds__(256) void linear_int8_join_kernel(LinearInt8Args a, int parts) {
	const int64_t count = (int64_t)a.rows * a.V, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
	if (at >= count) return;
	int sum = 0;
	for (int p = 0; p < parts; ++p) sum += a.parts[p * count + at];
	const int row = (int)(at / a.V), col = (int)(at % a.V);
	((T*)a.y)[row * a.ldy + col] = (T)scaled(sum, a.x_scale[row], a.w_scale[col], bias_at<T>(a, col));
}

// Few rows (at most 32, 64 where the columns are few): bound by the weights' bytes. A workgroup takes 16 I columns, its NW waves the depth in NW runs, each weight
// code going from memory into the registers of the one MFMA (16 x 16 x 64) block that uses it, the loads of U steps on their way while
// U others are multiplied; whole numbers are added through LDS, so the order does not matter. The rows' codes come from L2, J blocks of
// 16. WHOLE: of fewer codes still (kWhole bytes), which every workgroup makes for itself in LDS: one launch in the place of two (1 row, 4096
// deep, 4096 columns: 7.9 us; by a launch of quantize_rows and this one 4.2 + 6.2, and one launch more on the host).
constexpr int kWhole = 16 * 1024;
__host__ __device__ inline int64_t whole_pitch(int64_t D) { return (D + 63) / 64 * 64 + 16; }  // (16 rows in 16 places of the banks)

template <int NW, typename T, bool VEC>
__device__ __forceinline__ void quantize_into(const LinearInt8Args& a, int8_t* codes, float* scales, unsigned* tops) {
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pitch = (int)whole_pitch(a.D);
	int team = NW;  // waves to a row
	while (team > 1 && NW / team < a.rows) team /= 2;
	const int t = wave % team * 64 + lane;
	for (int r0 = 0; r0 < a.rows; r0 += NW / team) {
		const int r = r0 + wave / team;
		const bool on = r < a.rows;
		const T* const x = (const T*)a.rows_in + (int64_t)(on ? r : 0) * a.ld_in;
		unsigned top = q8::share_top<T, VEC>(x, a.D, t * 8, team * 512);
#pragma unroll
		for (int d = 32; d; d >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
		__syncthreads();
		if (lane == 0) tops[wave] = top;
		__syncthreads();
		for (int w = 0; w < team; ++w) top = max(top, tops[wave / team * team + w]);
		const q8::Scale scale(top);
		if (!on) continue;
		if (t == 0) scales[r] = scale.value;
		for (int at = t * 8; at < pitch - 16; at += team * 512) *(uint64_t*)(codes + r * pitch + at) = q8::eight_codes<T, VEC>(x, a.D, at, scale);
	}
	__syncthreads();
}

template <int I, int J, int NW, typename T, bool WHOLE>
__global__ __launch_bounds__(64 * NW) void linear_int8_few_kernel(LinearInt8Args a) {
	constexpr int U = I * J > 4 ? 2 : 4;
	__shared__ int sums[NW][J * 16][I * 16 + 1];
	__shared__ __attribute__((aligned(16))) int8_t codes[WHOLE ? kWhole : 16];
	__shared__ float scales[16];
	__shared__ unsigned tops[NW];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int r = lane & 15, q = lane >> 4, m0 = blockIdx.x * 16 * I;
	const int steps = (a.D + 63) / 64, per = (steps + NW - 1) / NW, begin = min(wave * per, steps), end = min(begin + per, steps);
	const int limit = (a.D + 15) / 16 * 16;
	const int8_t* w[I];
	const int8_t* x[J];
#pragma unroll
	for (int i = 0; i < I; ++i) w[i] = a.w + (int64_t)min(m0 + 16 * i + r, a.V - 1) * a.ldw;
	i32x4 fa[2][U][I], fb[2][U][J], acc[I][J];
	const auto load_w = [&](int set, int s) {
#pragma unroll
		for (int u = 0; u < U; ++u) {
			// a step past the run's end multiplies the last one's weights with zeros; the rows' codes are zero past the limit
			const int k = min(s + u, end - 1) * 64 + 16 * q, at = k < limit ? k : 0;
#pragma unroll
			for (int i = 0; i < I; ++i) fa[set][u][i] = *(const i32x4*)(w[i] + at);
		}
	};
	const auto load_x = [&](int set, int s) {
#pragma unroll
		for (int u = 0; u < U; ++u) {
			const int k = min(s + u, end - 1) * 64 + 16 * q;
#pragma unroll
			for (int j = 0; j < J; ++j) fb[set][u][j] = s + u < end ? *(const i32x4*)(x[j] + k) : i32x4{0, 0, 0, 0};
		}
	};
	const auto multiply = [&](int set) {
#pragma unroll
		for (int u = 0; u < U; ++u)
#pragma unroll
			for (int i = 0; i < I; ++i)
#pragma unroll
				for (int j = 0; j < J; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fa[set][u][i], fb[set][u][j], acc[i][j], 0, 0, 0);
	};
#pragma unroll
	for (int i = 0; i < I; ++i)
#pragma unroll
		for (int j = 0; j < J; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
	if (begin < end) {  // (the first weights are on their way while the rows are quantised)
		load_w(0, begin);
		load_w(1, begin + U);
	}
	if constexpr (WHOLE) {
		if (a.wide_in) quantize_into<NW, T, true>(a, codes, scales, tops);
		else quantize_into<NW, T, false>(a, codes, scales, tops);
	}
#pragma unroll
	for (int j = 0; j < J; ++j) {
		const int row = min(16 * j + r, a.rows - 1);
		x[j] = WHOLE ? codes + row * (int)whole_pitch(a.D) : a.x + (int64_t)row * a.ldx;
	}
	if (begin < end) {
		load_x(0, begin);
		load_x(1, begin + U);
		for (int s = begin; s < end; s += 2 * U) {
			multiply(0);
			if (s + 2 * U < end) {
				load_w(0, s + 2 * U);
				load_x(0, s + 2 * U);
			}
			if (s + U < end) multiply(1);
			if (s + 3 * U < end) {
				load_w(1, s + 3 * U);
				load_x(1, s + 3 * U);
			}
		}
	}
	// register e of block (i, j): column 16 i + 4 q + e, row 16 j + r
#pragma unroll
	for (int i = 0; i < I; ++i)
#pragma unroll
		for (int j = 0; j < J; ++j)
#pragma unroll
			for (int e = 0; e < 4; ++e) sums[wave][16 * j + r][16 * i + 4 * q + e] = acc[i][j][e];
	__syncthreads();
	for (int at = threadIdx.x; at < 16 * J * 16 * I; at += 64 * NW) {
		const int row = at / (16 * I), c = at % (16 * I), col = m0 + c;
		if (row >= a.rows || col >= a.V) continue;
		int sum = 0;
#pragma unroll
		for (int n = 0; n < NW; ++n) sum += sums[n][row][c];
		((T*)a.y)[row * a.ldy + col] = (T)scaled(sum, WHOLE ? scales[row] : a.x_scale[row], a.w_scale[col], bias_at<T>(a, col));
	}
}

}  // namespace i8
}  // namespace nnh
