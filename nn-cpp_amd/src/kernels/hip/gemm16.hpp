// gemm16.hpp - bf16 products on the matrix cores for the linear head's cross entropy, with its epilogues (internal to libnnh).
//
// out[outer][inner] = sum over depth of A[inner][depth] B[outer][depth], fp32 accumulators. The product is computed
// transposed (A's rows are the MFMA's rows), so a lane holds, of one outer row, runs of four consecutive inner elements:
// a softmax over the inner axis is a reduction within the lane.
//
// What bounds it: the matrix cores, 32 cycles a 32 x 32 x 16 MFMA and SIMD. A workgroup's waves hold 128 x 64 (64 x 64) of the
// tile each, so a depth of 16 takes 6 KB (4 KB) of operands from LDS for 256 (128) cycles of MFMA: three quarters of (as
// much as) LDS delivers beside. Operands go from memory into LDS without passing through registers, in stages of 64 depths,
// one barrier a stage. A stage's two operands take LDS half of its MFMA time to fill (64 bytes a cycle and CU), so with two
// whole stages of LDS a stage would arrive just when it is needed; the ring has five halves instead, A's half is under way
// a stage longer, and only B's has to arrive between two barriers. An operand whose depth is not the contiguous axis is
// read by transposed LDS reads and needs no transposed copy.
//
// 8192 rows, 4096 wide, 128000 words: the scores 6.8 ms (1260 TFLOP/s), the gradient of the rows 6.4 (1340), of the weight 8.1 (1060: its
// operands are both read transposed, twice the LDS instructions), where a library product of 8192^3 reaches 1474. Power holds
// the clock near 1.9 GHz meanwhile.
#pragma once

#include <type_traits>

#include "linear_cross_entropy.hpp"
#include "masked_attention_tile.hpp"

namespace nnh {
namespace g16 {

using attn::bf16x2;
using attn::f32x16;
using attn::f32x2;
using attn::f32x4;
using attn::Frag;
using attn::kInf;
using attn::kLog2e;
using attn::lds_s16x4;
using attn::u32x4;

constexpr int BK = 64;

template <int BM_, int BN_, int WM_, int WN_>
struct Tile {
	static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
	static constexpr int kWaves = (BM / WM) * (BN / WN), kThreads = 64 * kWaves;
	static constexpr int kA = BM * BK * 2, kB = BN * BK * 2, kStage = kA + kB;  // bytes
	static constexpr int kHalf = kA, kLoads = kHalf / 1024 / kWaves;  // an operand's part of a stage, a wave's loads for it
	static constexpr int kLds = 5 * kHalf > BM * BN * 2 ? 5 * kHalf : BM * BN * 2;
	static_assert(kA == kB, "the ring's places are alike");
	static_assert(kA % (1024 * kWaves) == 0 && kB % (1024 * kWaves) == 0, "a stage splits evenly over the waves");
	static_assert(kLds <= 160 * 1024, "LDS");
};

// What a wave loads of one operand, R rows to the tile: kSteps words a lane and stage. TR: depth is not contiguous.
template <int R, int NW, bool TR>
struct Loader {
	static constexpr int kSteps = R * BK * 2 / 1024 / NW;
	const __bf16* p[kSteps];
	int64_t step;  // elements from one stage to the next

	__device__ __forceinline__ void begin(const __bf16* base, int64_t ld, int first_row, int rows, int wave, int lane) {
		step = TR ? BK * ld : BK;
#pragma unroll
		for (int j = 0; j < kSteps; ++j) {
			const int w = (j * NW + wave) * 64 + lane;
			if (TR) {
				const int k = w / (R / 8), c = (w % (R / 8)) ^ attn::swizzle<R * 2>(k);
				// words past the operand's rows come from its first ones: their outputs are not stored
				const int r = first_row + c * 8 < rows ? first_row + c * 8 : 0;
				p[j] = base + k * ld + r;
			} else {
				const int r = w / 8, c = (w % 8) ^ attn::swizzle<128>(r);
				p[j] = base + (int64_t)min(first_row + r, rows - 1) * ld + c * 8;
			}
		}
	}
	// The stage's load j, after which it moves on; live: depths left, none or less past the last stage (what is past them is zero).
	// on: with MASK, bit k of a word for each depth of the stage: whether it is to be loaded.
	template <int j, bool MASK = false>
	__device__ __forceinline__ void load(char* tile, int live, int wave, int lane, uint64_t on = 0) {
		const int w = (j * NW + wave) * 64 + lane;
		const int k = TR ? w / (R / 8) : ((w % 8) ^ attn::swizzle<128>(w / 8)) * 8;
		const bool take = MASK ? (on >> k & 1) != 0 : k < live;
		attn::load_words<j * NW * 1024>(take ? (const void*)p[j] : (const void*)&attn::kZeroWord, attn::lds_place(tile + wave * 1024));
		p[j] += step;
	}
};

// Where a lane reads its operands: operand rows row0 + lane % 32 (row0 a multiple of 32), depths 16 t + 8 (lane / 32) + 0..7.
// As in attn::Reader, further depths are an XOR or a constant away.
template <int R, bool TR>
struct Reader {
	int at;
	__device__ __forceinline__ Reader(int row0, int lane) {
		const int half = lane >> 5, i = lane & 15;
		if (TR) {
			const int k = 8 * half + (i >> 2);
			at = k * (R * 2) + (((row0 / 8 + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ attn::swizzle<R * 2>(k)) * 16) + (i & 1) * 8;
		} else {
			at = (row0 + (lane & 31)) * 128 + ((half ^ attn::swizzle<128>(lane & 31)) * 16);
		}
	}
	// Block i of 32 rows from row0 on.
	__device__ __forceinline__ void read(Frag<__bf16>& f, const char* tile, int i, int t) const {
		if (TR) {
			// four rows further the permutation's low bits differ by 1; 16 rows further it is the same
			f.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + 16 * t * (R * 2) + (at ^ (64 * i))));
			f.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + (16 * t + 4) * (R * 2) + (at ^ (64 * i) ^ 16)));
		} else {
			f.w = *(const u32x4*)(tile + i * 32 * 128 + (at ^ (32 * t)));
		}
	}
};

// Which tile of the grid a workgroup takes: a run of tiles to each XCD, eight outer tiles wide, so that the tiles in
// flight on one share their operands in its L2.
__device__ __forceinline__ void tile_of(int inner_tiles, int outer_tiles, int& inner, int& outer) {
	const unsigned total = (unsigned)inner_tiles * outer_tiles, q = total / 8, r = total % 8, x = blockIdx.x % 8;
	const unsigned id = x * q + min(x, r) + blockIdx.x / 8;
	const unsigned g = id / (8u * inner_tiles), in = id % (8u * inner_tiles), width = min(8u, outer_tiles - 8 * g);
	outer = 8 * g + in % width;
	inner = in / width;
}

template <class T, bool ATR, bool BTR, int EPI>
__global__ __launch_bounds__(T::kThreads, 2) void gemm16_kernel(Gemm16Args a) {
	constexpr int BM = T::BM, BN = T::BN, WM = T::WM, WN = T::WN, I = WM / 32, J = WN / 32, NW = T::kWaves;
	__shared__ __attribute__((aligned(1024))) char lds[T::kLds];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5, wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;
	int m0, n0, from = 0;
	tile_of((a.inner + BM - 1) / BM, (a.outer + BN - 1) / BN, m0, n0);
	m0 *= BM;
	n0 *= BN;
	Loader<BM, NW, ATR> la;
	Loader<BN, NW, BTR> lb;
	if (EPI == kGemm16Out && a.parts) {
		from = blockIdx.y * a.part_depth;
		a.depth = min(a.depth - from, a.part_depth);
	}
	la.begin((const __bf16*)a.a + from * (ATR ? a.lda : 1), a.lda, m0, a.inner, wave, lane);
	lb.begin((const __bf16*)a.b + from * (BTR ? a.ldb : 1), a.ldb, n0, a.outer, wave, lane);
	f32x16 acc[I][J];
#pragma unroll
	for (int i = 0; i < I; ++i)
#pragma unroll
		for (int j = 0; j < J; ++j)
#pragma unroll
			for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.0f;

	const Reader<BM, ATR> ra(wm, lane);
	const Reader<BN, BTR> rb(wn, lane);
	const int stages = (a.depth + BK - 1) / BK;
	Frag<__bf16> fa[2][I], fb[2][J];
	// Operands of depths 16 t .. of a stage whose halves are at `x` and `y`.
	auto read = [&](int set, const char* x, const char* y, int t) {
#pragma unroll
		for (int i = 0; i < I; ++i) ra.read(fa[set][i], x, i, t);
#pragma unroll
		for (int j = 0; j < J; ++j) rb.read(fb[set][j], y, j, t);
	};
	// The products of one operand set. A read of the next depths goes behind each, and of a half stage's loads (load(0) ..
	// load(kLoads - 1)) one behind every other: a wave whose loads wait for their turn multiplies nothing meanwhile.
	auto multiply = [&](int set, auto load) {
		constexpr int kReads = I * (ATR ? 2 : 1) + J * (BTR ? 2 : 1);
		attn::each<I * J>([&](auto at) {
			constexpr int x = decltype(at)::value, per = I * J / T::kLoads;
			attn::mma(acc[x / J][x % J], fa[set][x / J], fb[set][x % J]);
			if constexpr (x % per == per - 1) load(std::integral_constant<int, x / per>{});
		});
#pragma unroll
		for (int x = 0; x < I * J; ++x) {
			__builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
			__builtin_amdgcn_sched_group_barrier(0x100, (kReads + I * J - 1) / (I * J), 0);
		}
		__builtin_amdgcn_sched_barrier(0);
	};
	// Stage s has its halves in places 2 s and 2 s + 1 of the ring.
	auto place = [&](int x) { return lds + x % 5 * T::kHalf; };
	// A's half of stage s; of the rows that count alone where a.live names them (a weight's gradient, kMask): dz is zero for the
	// others, but x need not be finite there. Words past the last row's are zero, and the next stage's word is read a stage ahead.
	constexpr bool kMask = EPI == kGemm16Out && BTR;
	const uint64_t* const words = kMask ? a.live + from / BK : nullptr;
	uint64_t word = kMask && a.depth > 0 ? words[0] : 0;
	auto load_a = [&](auto j, int x, int s) {
		constexpr int J0 = decltype(j)::value;
		if constexpr (kMask) {
			la.template load<J0, true>(place(x), 0, wave, lane, word);
			if (J0 == T::kLoads - 1) word = s + 1 < stages ? words[s + 1] : 0;
		} else {
			la.template load<J0>(place(x), a.depth - s * BK, wave, lane);
		}
	};
	auto load_b = [&](auto j, int x, int s) { lb.template load<decltype(j)::value>(place(x), a.depth - s * BK, wave, lane); };
	// Stage s (s % 5 = S), whose first operands are in registers. Before its last depths are multiplied every wave has read
	// them, and the next stage has arrived: from there on B of stage s + 2 and then, a step later, A of stage s + 3 may take its
	// places, and the next one's first operands are read.
	auto step = [&](int s, auto mod) {
		constexpr int S = decltype(mod)::value;
		read(1, place(2 * S), place(2 * S + 1), 1);
		multiply(0, [&](auto j) { load_a(j, 2 * S + 4, s + 2); });
#pragma unroll
		for (int t = 1; t < BK / 16 - 1; ++t) {
			read(~t & 1, place(2 * S), place(2 * S + 1), t + 1);
			multiply(t & 1, [](auto) {});
		}
		asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(T::kLoads) : "memory");
		__builtin_amdgcn_s_barrier();
		asm volatile("" ::: "memory");
		read(0, place(2 * S + 2), place(2 * S + 3), 0);
		multiply(1, [&](auto j) { load_b(j, 2 * S, s + 2); });
	};
#pragma unroll
	for (int s = 0; s < 2; ++s) {
		attn::each<T::kLoads>([&](auto j) { load_a(j, 2 * s, s); });
		attn::each<T::kLoads>([&](auto j) { load_b(j, 2 * s + 1, s); });
	}
	asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * T::kLoads) : "memory");
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

	// register 4 g + x of block (i, j): inner m0 + wm + 32 i + 8 g + 4 half + x, outer n0 + wn + 32 j + col
	const int mw = m0 + wm + 4 * half;
	// The tile in 16 bits through LDS, 16-byte words permuted by row, for stores of whole rows.
	auto store_rows = [&]() {
		constexpr int W = BM / 8;  // words to a row
		__bf16* const tile = (__bf16*)lds;
#pragma unroll
		for (int j = 0; j < J; ++j) {
			const int r = wn + 32 * j + col;
#pragma unroll
			for (int i = 0; i < I; ++i)
#pragma unroll
				for (int g = 0; g < 4; ++g) {
					union {
						bf16x2 p[2];
						uint64_t w;
					} y;
					y.p[0] = __builtin_convertvector(f32x2{acc[i][j][4 * g], acc[i][j][4 * g + 1]}, bf16x2);
					y.p[1] = __builtin_convertvector(f32x2{acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]}, bf16x2);
					const int m = wm + 32 * i + 8 * g;
					*(uint64_t*)(tile + r * BM + (((m / 8) ^ (r % W)) * 8) + 4 * half) = y.w;
				}
		}
		__syncthreads();
		for (int w = threadIdx.x; w < BN * W; w += T::kThreads) {
			const int r = w / W, c = w % W;
			if (n0 + r < a.outer && m0 + c * 8 < a.ldo)
				*(u32x4*)((__bf16*)a.out + (int64_t)(n0 + r) * a.ldo + m0 + c * 8) = *(const u32x4*)(tile + r * BM + ((c ^ (r % W)) * 8));
		}
	};
	if constexpr (EPI == kGemm16Out) {
		const float scale = a.scale ? *a.scale * a.factor : a.factor;
		if (a.whole_words && !a.parts && !a.sum_in && !a.sum_out && a.first) {
#pragma unroll
			for (int i = 0; i < I; ++i)
#pragma unroll
				for (int j = 0; j < J; ++j)
#pragma unroll
					for (int x = 0; x < 16; ++x) acc[i][j][x] *= scale;
			store_rows();
			return;
		}
#pragma unroll
		for (int j = 0; j < J; ++j) {
			const int n = n0 + wn + 32 * j + col;
			if (n >= a.outer) continue;
			if (a.parts) {
				float* const o = a.parts + ((int64_t)blockIdx.y * a.outer + n) * a.inner;
#pragma unroll
				for (int i = 0; i < I; ++i)
#pragma unroll
					for (int x = 0; x < 16; ++x) {
						const int m = mw + 32 * i + 8 * (x / 4) + x % 4;
						if (m < a.inner) o[m] = acc[i][j][x];
					}
				continue;
			}
#pragma unroll
			for (int i = 0; i < I; ++i)
#pragma unroll
				for (int g = 0; g < 4; ++g) {
					const int m = mw + 32 * i + 8 * g;
#pragma unroll
					for (int x = 0; x < 4; ++x) {
						if (m + x >= a.inner) continue;
						float y = acc[i][j][4 * g + x] * scale;
						if (a.sum_in) y += a.sum[(int64_t)n * a.inner + m + x];
						if (a.sum_out) {
							a.sum[(int64_t)n * a.inner + m + x] = y;
						} else {
							__bf16* o = (__bf16*)a.out + (int64_t)n * a.ldo + m + x;
							if (!a.first) y += (float)*o;
							*o = (__bf16)y;
						}
					}
				}
		}
		return;
	} else {
		// a row's scores z = x w + b, in the lane: the whole softmax's statistics of this wave's WM columns, and what the
		// tile stores
		if (a.bias) {
#pragma unroll
			for (int i = 0; i < I; ++i)
#pragma unroll
				for (int x = 0; x < 16; ++x) {
					const int m = mw + 32 * i + 8 * (x / 4) + x % 4;
					const float b = m < a.inner ? (float)((const __bf16*)a.bias)[m] : 0.0f;
#pragma unroll
					for (int j = 0; j < J; ++j) acc[i][j][x] += b;
				}
		}
#pragma unroll
		for (int j = 0; j < J; ++j) {
			const int n = n0 + wn + 32 * j + col;
			const bool on = n < a.outer;
			const int target = on ? a.targets[n] - a.first_inner : -1;
			if constexpr (EPI == kGemm16Grad) {
				const float lse2 = on ? a.lse[n] * kLog2e : 0.0f, f = on ? a.weight[n] : 0.0f;
#pragma unroll
				for (int i = 0; i < I; ++i)
#pragma unroll
					for (int x = 0; x < 16; ++x) {
						const int m = mw + 32 * i + 8 * (x / 4) + x % 4;
						float y = attn::exp2_of(__builtin_fmaf(acc[i][j][x], kLog2e, -lse2));
						y = (m == target ? y - 1.0f : y) * f;
						acc[i][j][x] = m < a.inner && f != 0.0f ? y : 0.0f;
					}
			} else {
				float top = -kInf, sum = 0.0f;
				if (m0 + wm + WM > a.inner) {
#pragma unroll
					for (int i = 0; i < I; ++i)
#pragma unroll
						for (int x = 0; x < 16; ++x)
							if (mw + 32 * i + 8 * (x / 4) + x % 4 >= a.inner) acc[i][j][x] = -kInf;
				}
#pragma unroll
				for (int i = 0; i < I; ++i)
#pragma unroll
					for (int x = 0; x < 16; ++x) top = fmaxf(top, acc[i][j][x]);
				top = attn::max_halves(top);
				const int chunk = (m0 + wm) / WM;
				if (__any(target >= m0 + wm && target < m0 + wm + WM)) {
#pragma unroll
					for (int i = 0; i < I; ++i)
#pragma unroll
						for (int x = 0; x < 16; ++x)
							if (mw + 32 * i + 8 * (x / 4) + x % 4 == target && target < a.inner) a.hit[n] = acc[i][j][x];
				}
				const float base = top == -kInf ? 0.0f : top * kLog2e;
#pragma unroll
				for (int i = 0; i < I; ++i)
#pragma unroll
					for (int x = 0; x < 16; ++x) {
						acc[i][j][x] = attn::exp2_of(__builtin_fmaf(acc[i][j][x], kLog2e, -base));
						sum += acc[i][j][x];
					}
				sum = attn::add_halves(sum);
				if (on && half == 0 && m0 + wm < a.inner) ((f32x2*)a.stats)[(int64_t)n * a.chunks + chunk] = f32x2{top, sum};
			}
		}
		if constexpr (EPI != kGemm16Stats) store_rows();
	}
}

}  // namespace g16
}  // namespace nnh
