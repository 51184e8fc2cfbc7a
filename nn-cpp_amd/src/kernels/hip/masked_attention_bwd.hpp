// masked_attention_bwd.hpp - the backward kernels of masked attention (masked_attention.hpp), instantiated per element type
// by masked_attention_bwd_*.hip.
//
//   p = exp(z - lse),  dz = p (g.v - delta),  delta = g.out,  ds = dz (1 - (c / cap)^2)
//   dq = scale ds k,   dk = scale ds^T q,     dv = p^T g
//
// Two kernels, each recomputing the scores of its own products: dq by query rows (which also leaves delta and lse in units of log 2), then dk and dv
// by key rows, where the queries of all heads that share the key head are added in their order. No gradient is added by
// atomics, so the results repeat bit for bit; the price is seven products of a pair of rows where five would do.
//
// Causal, 8192 tokens, 16 heads of 128 on 8 key heads, bf16: dq 490-500 us, dk and dv 755 + 28 us to add their parts (690 TFLOP/s
// of the products made). As in the forward kernel the vector operations beside the products set the pace; dk and dv also read
// 40 KB of LDS for 32 products, a quarter more than the products' time, since a wave has no registers left for V.
#pragma once

#include <type_traits>

#include "masked_attention_tile.hpp"

namespace nnh {
namespace attn {

constexpr int kBwdWaves = 4, kBwdRows = 32 * kBwdWaves;

// Stores a column of a gradient, or adds it to what the row holds.
template <typename T, int DH, bool VEC>
__device__ __forceinline__ void store_gradient(T* o, const f32x16* x, float f, int dh, int half, bool first) {
	if constexpr (VEC && sizeof(T) == 2) {  // (dh is a multiple of 8)
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int g = 0; g < 2; ++g) {
				const int d = 32 * b + 16 * g + 8 * half;
				Frag<T> y, old;
				old.w = u32x4{0, 0, 0, 0};
				if (!first) {  // (the swap of two halves undoes itself)
					if (d < dh) old.w = *(const u32x4*)(o + d);
					eight_of(old);
				}
#pragma unroll
				for (int i = 0; i < 8; ++i) y.e[i] = (T)(first ? x[b][8 * g + i] * f : to_float(old.e[i]) + x[b][8 * g + i] * f);
				eight_of(y);
				if (d < dh) *(u32x4*)(o + d) = y.w;
			}
	} else {
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int g = 0; g < 4; ++g) {
				const int d = 32 * b + 8 * g + 4 * half;
				if constexpr (VEC) {
					if (d >= dh) continue;
					f32x4 y = f32x4{x[b][4 * g] * f, x[b][4 * g + 1] * f, x[b][4 * g + 2] * f, x[b][4 * g + 3] * f};
					if (!first) y = *(const f32x4*)(o + d) + y;
					*(f32x4*)(o + d) = y;
				} else {
#pragma unroll
					for (int i = 0; i < 4; ++i)
						if (d + i < dh) o[d + i] = (T)(first ? x[b][4 * g + i] * f : to_float(o[d + i]) + x[b][4 * g + i] * f);
				}
			}
	}
}

// Turns a block of raw scores into p (before masking) and, where scores are capped, leaves 1 - (c / cap)^2 in slope.
// far: the distance of register i's pair; lse2: its row's lse in units of log 2.
template <typename T, typename Far, typename Lse>
__device__ __forceinline__ void weights(f32x16& s, f32x16& slope, const MaskedAttentionArgs& a, float slope2, Far far, Lse lse2) {
	float c = a.scale * kLog2e;
	if (a.cap > 0.0f) {
		const float in = a.scale / a.cap;
		c = a.cap * kLog2e;
#pragma unroll
		for (int i = 0; i < 16; ++i) {
			s[i] = tanh_of<T>(s[i] * in);
			slope[i] = __builtin_fmaf(-s[i], s[i], 1.0f);
		}
	}
	if (a.slopes) {
#pragma unroll
		for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], c, -slope2 * far(i));
		c = 1.0f;
	}
#pragma unroll
	for (int i = 0; i < 16; ++i) s[i] = exp2_of(__builtin_fmaf(s[i], c, -lse2(i)));
}

// dq: a workgroup's 128 queries of one head against the keys they see, as in the forward kernel: transposed scores, a query
// a lane, dQ^T += K^T dS^T. The second pass is the forward's (values that are not finite in a partly seen tile).
//
// It starts from delta = g.out of the stored out and of what that lost in its rounding to 16 bits. Without the latter delta is
// off by out's rounding, and with it a row's gradient by that times the keys' weighted mean: as much again as the rounding of dS
// where scores are spread, three times that where a key or two have a row's weight. A row's p add up to 1, so its sum of
// p (g.v - delta) is what delta was off by: the delta that is left for the other kernel has it added either way.
template <typename T, int DH, bool VEC>
__global__ __launch_bounds__(256, (row_bytes<T, DH>() >= 512 ? 1 : 2)) void masked_attention_dq_kernel(MaskedAttentionArgs a) {
	constexpr int RB = row_bytes<T, DH>(), KT = RB >= 512 ? 32 : 64, kTile = KT * RB;
	__shared__ __attribute__((aligned(1024))) char lds[4 * kTile + 2 * 256 + kBwdWaves * 4];
	char* const docs_at = lds + 4 * kTile;  // the two tiles'
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;
	const int tiles = (a.Tq + kBwdRows - 1) / kBwdRows, pairs = a.N * a.Hkv;
	int tile, h, n;
	{
		const unsigned block = blockIdx.x;
		unsigned pair, rest;
		if (pairs % 8 == 0) {
			const unsigned per = pairs / 8, in = block / 8;
			pair = block % 8 * per + in % per;
			rest = in / per;
		} else {
			pair = block % pairs;
			rest = block / pairs;
		}
		n = pair / a.Hkv;
		h = pair % a.Hkv * a.G + rest % a.G;
		tile = tiles - 1 - (int)(rest / a.G);
	}
	const int q0 = tile * kBwdRows, i = q0 + wave * 32 + col, hk = h / a.G;
	const int live = live_keys(a, n), pos0 = first_position(a, n);
	const T* const kbase = (const T*)a.k + n * a.ks.sample + hk * a.ks.head;
	const T* const vbase = (const T*)a.v + n * a.vs.sample + hk * a.vs.head;
	const bool live_row = i < a.Tq;
	const int64_t row = ((int64_t)n * a.H + h) * a.Tq + min(i, a.Tq - 1);

	Frag<T> q[DH / 16], g[DH / 16];
	float delta = 0.0f;
	{
		const int64_t r = min(i, a.Tq - 1);
		const T* qr = (const T*)a.q + n * a.qs.sample + r * a.qs.row + h * a.qs.head;
		const T* gr = (const T*)a.g + n * a.gs.sample + r * a.gs.row + h * a.gs.head;
		const T* rest = a.rest ? (const T*)a.rest + n * a.rs.sample + r * a.rs.row + h * a.rs.head : nullptr;
		const T* orow = (const T*)a.out + n * a.os.sample + r * a.os.row + h * a.os.head;
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) {
			row_from<T, VEC>(q[t], qr, a.dh, half, t, live_row);
			row_from<T, VEC>(g[t], gr, a.dh, half, t, live_row);
			Frag<T> o;
			row_from<T, VEC>(o, orow, a.dh, half, t, live_row);
#pragma unroll
			for (int j = 0; j < 8; ++j) delta += to_float(g[t].e[j]) * to_float(o.e[j]);
		}
		if (sizeof(T) == 2 && rest) {
			float more = 0.0f;
#pragma unroll
			for (int t = 0; t < DH / 16; ++t) {
				Frag<T> o;
				row_from<T, VEC>(o, rest, a.dh, half, t, live_row);
#pragma unroll
				for (int j = 0; j < 8; ++j) more += to_float(g[t].e[j]) * to_float(o.e[j]);
			}
			delta += more;
		}
		delta = add_halves(delta);
	}
	const Sight see = sight_of(a, n, i, live, pos0);
	const int pos = pos0 + i;
	const float slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.0f, lse2 = a.lse[row] * kLog2e;
	int lo = 0, hi = live, pre = a.prefix ? clamped(a.prefix[n], 0, live) : 0;
	{
		const int64_t first = (int64_t)pos0 + q0, last = (int64_t)pos0 + min(q0 + kBwdRows, a.Tq) - 1;
		if (a.causal) hi = clamped(last + 1, 0, live);
		if (a.window) {
			lo = clamped(first - a.window + 1, 0, live);
			hi = min(hi, clamped(last + a.window, 0, live));
		}
	}
	const int kb = (a.Tk + 63) / 64;
	DocRange mine{0, 0, 0};
	if (a.q_docs) {
		const int nb = (a.Tq + 63) / 64, b0 = q0 / 64;
		mine = a.q_ranges[(int64_t)n * nb + b0];
		if (b0 + 1 < nb) {
			const DocRange o = a.q_ranges[(int64_t)n * nb + b0 + 1];
			mine.lo = min(mine.lo, o.lo);
			mine.hi = max(mine.hi, o.hi);
		}
	}
	const int nt = (max(hi, pre) + KT - 1) / KT;
	f32x16 d[DH / 32];
	float off;
	arrived(q);
	arrived(g);
	arrived();

	auto run = [&](auto safe) {
		off = 0.0f;
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int x = 0; x < 16; ++x) d[b][x] = 0.0f;
		int base = -64;
		uint64_t on = 0;
		auto next = [&]() -> int {
			while (on == 0) {
				base += 64;
				if (base >= nt) return -1;
				const int x = base + lane, k0 = x * KT;
				bool s = x < nt && ((k0 < hi && k0 + KT > lo) || k0 < pre);
				if (s && a.k_docs) {
					const DocRange r = a.k_ranges[(int64_t)n * kb + k0 / 64];
					s = r.lo <= mine.hi && r.hi >= mine.lo;
				}
				on = __ballot(s);
			}
			const int x = __builtin_ctzll(on);
			on &= on - 1;
			return base + x;
		};
		auto load = [&](int x, char* to, char* docs_to) {
			if (a.k_docs && wave == 0) load_numbers(a.k_docs + (int64_t)n * a.Tk + min(x * KT + lane, a.Tk - 1), docs_to);
			load_tile<T, DH, KT, kBwdWaves, VEC>(to, kbase + (int64_t)x * KT * a.ks.row, a.ks.row, live - x * KT, a.dh, wave, lane);
			load_tile<T, DH, KT, kBwdWaves, VEC>(to + kTile, vbase + (int64_t)x * KT * a.vs.row, a.vs.row, live - x * KT, a.dh, wave, lane);
		};
		auto take = [&](const char* kt, const char* vt, const int* docs, DocRange r, int k0) {
			bool some = (k0 < see.hi && k0 + KT > see.lo) || k0 < see.pre;
			bool all = (k0 >= see.lo && k0 + KT <= see.hi) || k0 + KT <= see.pre;
			if (a.k_docs) {
				some = some && see.doc >= r.lo && see.doc <= r.hi;
				all = all && see.doc == r.lo && see.doc == r.hi && !r.none;
			}
			if (!__any(some)) return;
			const bool partial = !__all(all);
#pragma clang loop unroll(disable)
			for (int x = 0; x < KT / 32; ++x) {
				const Reader<T, RB> at(fresh_lane());
				f32x16 s, dp, slope;
#pragma unroll
				for (int j = 0; j < 16; ++j) s[j] = dp[j] = 0.0f;
				in_groups<Frag<T>, DH / 8, sizeof(T) == 2 ? 4 : 1>([&](int i, Frag<T>& f) { at.rows(f, (i % 2 ? vt : kt) + 32 * x * RB, i / 2); },
				                                                  [&](int i, const Frag<T>& f) {
					                                                  if (i % 2) mma(dp, f, g[i / 2]);
					                                                  else mma(s, f, q[i / 2]);
				                                                  });
				const int j0 = fresh(k0 + 32 * x + 4 * half);
				weights<T>(s, slope, a, slope2, [&](int j) { const int y = pos - (j0 + 8 * (j / 4) + j % 4); return (float)(y < 0 ? -y : y); },
				           [&](int) { return lse2; });
#pragma unroll
				for (int j = 0; j < 16; ++j) s[j] *= dp[j] - delta;
				unsigned seen = 0xffff;
				if (partial) {
					seen = 0;
#pragma unroll
					for (int j = 0; j < 16; ++j) seen |= see.sees(j0 + 8 * (j / 4) + j % 4) ? 1u << j : 0u;
					if (a.k_docs) {
#pragma unroll
						for (int y = 0; y < 4; ++y) {
							const i32x4 e = *(const i32x4*)(docs + 32 * x + 8 * y + 4 * half);
#pragma unroll
							for (int j = 0; j < 4; ++j) seen &= e[j] == see.doc ? ~0u : ~(1u << (4 * y + j));
						}
					}
#pragma unroll
					for (int j = 0; j < 16; ++j) s[j] = seen >> j & 1 ? s[j] : 0.0f;
				}
				float part[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
				for (int j = 4; j < 16; ++j) part[j % 4] += s[j];
				off += (part[0] + part[1]) + (part[2] + part[3]);
				if (a.cap > 0.0f) {
#pragma unroll
					for (int j = 0; j < 16; ++j) s[j] *= slope[j];
				}
				const bool clean = decltype(safe)::value && partial;
				Frag<T> ds[2];
				operand_of(ds[0], s, 0);
				operand_of(ds[1], s, 1);
				constexpr int B = DH / 32;
				in_groups<Frag<T>, 2 * B, sizeof(T) == 2 ? 2 : 1>([&](int i, Frag<T>& f) { at.columns(f, kt + (32 * x + 16 * (i / B)) * RB, i % B); },
				                                                 [&](int i, Frag<T>& f) {
					                                                 if (clean) only_finite(f);
					                                                 mma(d[i % B], f, ds[i / B]);
				                                                 });
				if (clean) {  // a key that is not finite makes the queries that see it NaN
#pragma clang loop unroll(disable)
					for (int j = 0; j < 32; ++j) {
						const int bit = (j >> 3) * 4 + (j & 3), owner = col + 32 * ((j >> 2) & 1);
						const bool sees = (unsigned)__shfl((int)seen, owner) >> bit & 1;
#pragma unroll
						for (int b = 0; b < DH / 32; ++b)
#pragma unroll
							for (int y = 0; y < 16; ++y) {
								const float v = element_of<T, DH>(kt, 32 * x + j, 32 * b + 8 * (y / 4) + 4 * half + y % 4);
								d[b][y] += sees && not_finite(v) ? v - v : 0.0f;
							}
					}
				}
			}
		};
		int cur = next();
		auto step = [&](auto buf) {
			constexpr int B = decltype(buf)::value;
			char* const from = lds + B * 2 * kTile;
			wait_loads();
			__builtin_amdgcn_s_barrier();
			asm volatile("" ::: "memory");
			DocRange r{0, 0, 0};
			if (a.k_docs) r = range_at(a.k_ranges, (int64_t)n * kb + cur * KT / 64);
			const int then = next();
			if (then >= 0) load(then, lds + (1 - B) * 2 * kTile, docs_at + (1 - B) * 256);
			take(from, from + kTile, (const int*)(docs_at + B * 256), r, cur * KT);
			cur = then;
		};
		if (cur >= 0) load(cur, lds, docs_at);
		while (cur >= 0) {
			step(std::integral_constant<int, 0>{});
			if (cur >= 0) step(std::integral_constant<int, 1>{});
		}
		bool bad = false;
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int x = 0; x < 16; ++x) bad |= not_finite(d[b][x]);
		return any_wave<kBwdWaves>((int*)(docs_at + 2 * 256), wave, lane, bad);
	};
	if (run(std::false_type{})) run(std::true_type{});
	off = add_halves(off);
	if (live_row && half == 0) {
		a.delta[row] = delta + off;
		a.lse2[row] = lse2;
	}
	if (live_row && a.dq)
		store_gradient<T, DH, VEC>((T*)a.dq + n * a.dqs.sample + (int64_t)i * a.dqs.row + h * a.dqs.head, d, a.scale, a.dh, half,
		                           a.dq_first != 0);
}

// dk and dv: a workgroup's 128 keys of one key head against the queries, of all its heads in turn, that see them. Scores
// as they are (S = Q K^T), a key a lane: dV^T += G^T P, dK^T += Q^T dS. A wave's K stays in registers and the workgroup's V in
// LDS; the tiles of Q and G come through LDS with their rows' lse, delta and documents. A wave's step of 32 queries is a chain of
// products and exponentials that two waves a SIMD do not hide in full, and a causal mask gives the first keys a whole
// sequence of them: with too few workgroups to fill the GPU, a.parts of them share a key tile, each taking every
// a.parts-th tile of queries, and their sums are added afterwards in their order (masked_attention_dkv_join_kernel).
template <typename T, int DH, bool VEC>
__global__ __launch_bounds__(256, (row_bytes<T, DH>() >= 512 ? 1 : 2)) void masked_attention_dkv_kernel(MaskedAttentionArgs a) {
	constexpr int RB = row_bytes<T, DH>(), QT = 32, kTile = QT * RB;
	__shared__ __attribute__((aligned(1024))) char lds[kBwdRows * RB + 4 * kTile + 2 * 3 * 256 + kBwdWaves * 4];
	char* const vt = lds;
	char* const ring = lds + kBwdRows * RB;
	char* const rows = ring + 4 * kTile;  // per buffer 64 rows' lse, delta and documents
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;
	const int pairs = a.N * a.Hkv;
	int tile, pair, part;  // the first keys, which are seen most, come first
	{
		const unsigned block = blockIdx.x;
		unsigned rest;
		if (pairs % 8 == 0) {
			const unsigned per = pairs / 8, in = block / 8;
			pair = block % 8 * per + in % per;
			rest = in / per;
		} else {
			pair = block % pairs;
			rest = block / pairs;
		}
		part = rest % a.parts;
		tile = rest / a.parts;
	}
	const int n = pair / a.Hkv, hk = pair % a.Hkv, k0 = tile * kBwdRows, j = k0 + wave * 32 + col;
	const int live = live_keys(a, n), pos0 = first_position(a, n), pre = a.prefix ? clamped(a.prefix[n], 0, live) : 0;
	// The queries that see key j: lo <= i < hi (all of them for a key of the prefix).
	Sight see{0, 0, 0, 0};
	if (j < live) {
		see.doc = a.k_docs ? a.k_docs[(int64_t)n * a.Tk + j] : 0;
		if (see.doc >= 0) {
			see.hi = a.Tq;
			if (j >= pre) {
				const int64_t at = (int64_t)j - pos0;  // the query at key j's own position
				if (a.causal) see.lo = clamped(at, 0, a.Tq);
				if (a.window) {
					see.lo = max(see.lo, clamped(at - a.window + 1, 0, a.Tq));
					see.hi = clamped(at + a.window, 0, a.Tq);
				}
			}
		}
	}
	// and those that may see any of the workgroup's
	int lo = 0, hi = k0 < live ? a.Tq : 0;
	if (k0 >= pre) {
		const int64_t first = (int64_t)k0 - pos0, last = (int64_t)min(k0 + kBwdRows, live) - 1 - pos0;
		if (a.causal) lo = clamped(first, 0, a.Tq);
		if (a.window) {
			lo = max(lo, clamped(first - a.window + 1, 0, a.Tq));
			hi = min(hi, clamped(last + a.window, 0, a.Tq));
		}
	}
	const int qb = (a.Tq + 63) / 64;
	DocRange mine{0, 0, 0};
	if (a.k_docs && k0 < live) {
		const int nb = (a.Tk + 63) / 64, b0 = k0 / 64;
		mine = a.k_ranges[(int64_t)n * nb + b0];
		if (b0 + 1 < nb) {
			const DocRange o = a.k_ranges[(int64_t)n * nb + b0 + 1];
			mine.lo = min(mine.lo, o.lo);
			mine.hi = max(mine.hi, o.hi);
		}
	}
	const int nt = (hi + QT - 1) / QT;

	if (k0 < live)
		load_tile<T, DH, kBwdRows, kBwdWaves, VEC>(vt, (const T*)a.v + n * a.vs.sample + hk * a.vs.head + (int64_t)k0 * a.vs.row, a.vs.row, live - k0, a.dh, wave, lane);
	Frag<T> kf[DH / 16];
	{
		const T* kr = (const T*)a.k + n * a.ks.sample + (int64_t)min(j, a.Tk - 1) * a.ks.row + hk * a.ks.head;
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) row_from<T, VEC>(kf[t], kr, a.dh, half, t, j < live);
	}
	arrived(kf);
	arrived();
	f32x16 dk[DH / 32], dv[DH / 32];

	auto run = [&](auto safe) {
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int x = 0; x < 16; ++x) dk[b][x] = dv[b][x] = 0.0f;
		// The tiles of each head's queries in turn, the last ones first: those are seen by most keys under a causal mask, so the
		// workgroups of one key head read the same rows at about the same time.
		int head = -1, base = -64;
		uint64_t on = 0;
		auto next = [&]() -> int {
			while (on == 0) {
				base -= 64;
				if (base + 64 <= lo / QT || base < -63) {
					if (nt == 0 || ++head >= a.G) return -1;
					base = (nt - 1) / 64 * 64;
				}
				const int x = base + lane, q0 = x * QT;
				bool s = x < nt && q0 + QT > lo && x % a.parts == part;
				if (s && a.q_docs) {
					const DocRange r = a.q_ranges[(int64_t)n * qb + q0 / 64];
					s = r.lo <= mine.hi && r.hi >= mine.lo;
				}
				on = __ballot(s);
			}
			const int x = 63 - __builtin_clzll(on);
			on &= ~((uint64_t)1 << x);
			return base + x;
		};
		auto load = [&](int x, int buf) {
			const int h = hk * a.G + head, q0 = x * QT;
			load_tile<T, DH, QT, kBwdWaves, VEC>(ring + buf * 2 * kTile, (const T*)a.q + n * a.qs.sample + (int64_t)q0 * a.qs.row + h * a.qs.head, a.qs.row, a.Tq - q0, a.dh, wave, lane);
			load_tile<T, DH, QT, kBwdWaves, VEC>(ring + (buf * 2 + 1) * kTile, (const T*)a.g + n * a.gs.sample + (int64_t)q0 * a.gs.row + h * a.gs.head, a.gs.row, a.Tq - q0, a.dh, wave, lane);
			const int64_t r = min(q0 + lane, a.Tq - 1), row = ((int64_t)n * a.H + h) * a.Tq + r;
			if (wave == 0) load_numbers(a.lse2 + row, rows + buf * 768);
			if (wave == 1) load_numbers(a.delta + row, rows + buf * 768 + 256);
			if (wave == 2 && a.q_docs) load_numbers(a.q_docs + (int64_t)n * a.Tq + r, rows + buf * 768 + 512);
		};
		auto take = [&](const char* qt, const char* gt, const float* lse, const float* delta, const int* docs, DocRange r, int q0, int h) {
			bool some = q0 < see.hi && q0 + QT > see.lo, all = q0 >= see.lo && q0 + QT <= see.hi;
			if (a.q_docs) {
				some = some && see.doc >= r.lo && see.doc <= r.hi;
				all = all && see.doc == r.lo && see.doc == r.hi && !r.none;
			}
			if (!__any(some)) return;
			const bool partial = !__all(all);
			const Reader<T, RB> at(fresh_lane());
			// Each step's loads stay with it (sched_barrier): moved ahead they cost the registers that K is held in.
			f32x16 s, dp, slope;
#pragma unroll
			for (int y = 0; y < 16; ++y) s[y] = dp[y] = 0.0f;
			in_groups<Frag<T>, DH / 16, sizeof(T) == 2 ? 2 : 1>([&](int t, Frag<T>& f) { at.rows(f, qt, t); },
			                                                   [&](int t, const Frag<T>& f) { mma(s, f, kf[t]); });
			__builtin_amdgcn_sched_barrier(0);
			const int i0 = fresh(4 * half);  // the tile's row of register y: i0 + 8 (y / 4) + y % 4
			weights<T>(s, slope, a, a.slopes ? a.slopes[h] * kLog2e : 0.0f,
			           [&](int y) { const int z = pos0 + q0 + i0 + 8 * (y / 4) + y % 4 - j; return (float)(z < 0 ? -z : z); },
			           [&](int y) { return lse[i0 + 8 * (y / 4) + y % 4]; });
			unsigned seen = 0xffff;
			if (partial) {
				seen = 0;
#pragma unroll
				for (int y = 0; y < 16; ++y) seen |= see.sees(q0 + i0 + 8 * (y / 4) + y % 4) ? 1u << y : 0u;
				if (a.q_docs) {
#pragma unroll
					for (int z = 0; z < 4; ++z) {
						const i32x4 o = *(const i32x4*)(docs + i0 + 8 * z);
#pragma unroll
						for (int y = 0; y < 4; ++y) seen &= o[y] == see.doc ? ~0u : ~(1u << (4 * z + y));
					}
				}
#pragma unroll
				for (int y = 0; y < 16; ++y) s[y] = seen >> y & 1 ? s[y] : 0.0f;
			}
			Frag<T> p[2];
			operand_of(p[0], s, 0);
			operand_of(p[1], s, 1);
			if (a.cap > 0.0f) {
#pragma unroll
				for (int y = 0; y < 16; ++y) s[y] *= slope[y];
			}
			__builtin_amdgcn_sched_barrier(0);
			in_groups<FragPair<T>, DH / 16, 1>([&](int t, FragPair<T>& f) {
				at.rows(f.a, gt, t);
				at.rows(f.b, vt + wave * 32 * RB, t);
			}, [&](int, const FragPair<T>& f) { mma(dp, f.a, f.b); });
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int y = 0; y < 16; ++y) dp[y] = s[y] * (dp[y] - delta[i0 + 8 * (y / 4) + y % 4]);
			if (partial) {
#pragma unroll
				for (int y = 0; y < 16; ++y) dp[y] = seen >> y & 1 ? dp[y] : 0.0f;
			}
			const bool clean = decltype(safe)::value && partial;
			Frag<T> ds[2];
			operand_of(ds[0], dp, 0);
			operand_of(ds[1], dp, 1);
			constexpr int kEach = DH / 16;  // products of 16 of the rows: dv and dk in turn
			in_groups<Frag<T>, 2 * kEach, sizeof(T) == 2 ? 2 : 1>([&](int i, Frag<T>& f) { at.columns(f, (i % 2 ? qt : gt) + 16 * (i / kEach) * RB, i % kEach / 2); },
			                                                     [&](int i, Frag<T>& f) {
				                                                     if (clean) only_finite(f);
				                                                     if (i % 2) mma(dk[i % kEach / 2], f, ds[i / kEach]);
				                                                     else mma(dv[i % kEach / 2], f, p[i / kEach]);
			                                                     });
			if (clean) {  // rows that are not finite, to the keys that they see
#pragma clang loop unroll(disable)
				for (int i = 0; i < 32; ++i) {
					const int bit = (i >> 3) * 4 + (i & 3), owner = col + 32 * ((i >> 2) & 1);
					const bool sees = (unsigned)__shfl((int)seen, owner) >> bit & 1;
#pragma unroll
					for (int b = 0; b < DH / 32; ++b)
#pragma unroll
						for (int y = 0; y < 16; ++y) {
							const int d = 32 * b + 8 * (y / 4) + 4 * half + y % 4;
							const float gv = element_of<T, DH>(gt, i, d), qv = element_of<T, DH>(qt, i, d);
							dv[b][y] += sees && not_finite(gv) ? gv : 0.0f;
							dk[b][y] += sees && not_finite(qv) ? qv - qv : 0.0f;
						}
				}
			}
		};
		int cur = next();
		auto step = [&](auto buf) {
			constexpr int B = decltype(buf)::value;
			wait_loads();
			__builtin_amdgcn_s_barrier();
			asm volatile("" ::: "memory");
			DocRange r{0, 0, 0};
			if (a.q_docs) r = range_at(a.q_ranges, (int64_t)n * qb + cur * QT / 64);
			const int h = hk * a.G + head, then = next();
			if (then >= 0) load(then, 1 - B);
			take(ring + B * 2 * kTile, ring + (B * 2 + 1) * kTile, (const float*)(rows + B * 768), (const float*)(rows + B * 768 + 256), (const int*)(rows + B * 768 + 512), r, cur * QT, h);
			cur = then;
		};
		if (cur >= 0) load(cur, 0);
		while (cur >= 0) {
			step(std::integral_constant<int, 0>{});
			if (cur >= 0) step(std::integral_constant<int, 1>{});
		}
		bool bad = false;
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int x = 0; x < 16; ++x) bad |= not_finite(dk[b][x]) || not_finite(dv[b][x]);
		return any_wave<kBwdWaves>((int*)(rows + 2 * 768), wave, lane, bad);
	};
	if (run(std::false_type{})) run(std::true_type{});
	if (j >= a.Tk) return;
	if (a.parts > 1) {
		const int64_t rows = (int64_t)pairs * a.Tk, row = (int64_t)pair * a.Tk + j;
		const int width = (a.dh + 3) & ~3;
		store_gradient<float, DH, true>(a.partial + (2 * part * rows + row) * width, dk, a.scale, width, half, true);
		store_gradient<float, DH, true>(a.partial + ((2 * part + 1) * rows + row) * width, dv, 1.0f, width, half, true);
	} else {
		if (a.dk)
			store_gradient<T, DH, VEC>((T*)a.dk + n * a.dks.sample + (int64_t)j * a.dks.row + hk * a.dks.head, dk, a.scale, a.dh, half,
			                           a.dk_first != 0);
		if (a.dv)
			store_gradient<T, DH, VEC>((T*)a.dv + n * a.dvs.sample + (int64_t)j * a.dvs.row + hk * a.dvs.head, dv, 1.0f, a.dh, half,
			                           a.dv_first != 0);
	}
}

// Adds the parts' sums of dk and dv, a thread to four elements.
template <typename T>
__global__ __launch_bounds__(256) void masked_attention_dkv_join_kernel(MaskedAttentionArgs a) {
	const int fours = (a.dh + 3) / 4, width = 4 * fours;
	const int64_t rows = (int64_t)a.N * a.Hkv * a.Tk, at = (int64_t)blockIdx.x * 256 + threadIdx.x, row = at / fours;
	const int d = (int)(at % fours) * 4;
	if (row >= rows) return;
	const int j = (int)(row % a.Tk), hk = (int)(row / a.Tk % a.Hkv), n = (int)(row / a.Tk / a.Hkv);
#pragma unroll
	for (int x = 0; x < 2; ++x) {
		T* const o = x ? (T*)a.dv : (T*)a.dk;
		if (!o) continue;
		const HeadStrides s = x ? a.dvs : a.dks;
		const bool first = x ? a.dv_first != 0 : a.dk_first != 0;
		f32x4 y = *(const f32x4*)(a.partial + (x * rows + row) * width + d);
		for (int p = 1; p < a.parts; ++p) y += *(const f32x4*)(a.partial + ((2 * p + x) * rows + row) * width + d);
		T* const to = o + n * s.sample + (int64_t)j * s.row + hk * s.head + d;
#pragma unroll
		for (int i = 0; i < 4; ++i)
			if (d + i < a.dh) to[i] = (T)(first ? y[i] : to_float(to[i]) + y[i]);
	}
}

template <typename T, int DH, bool VEC>
hipError_t launch_backward(const MaskedAttentionArgs& a, hipStream_t s) {
	if (a.Tq > 0) {
		const int64_t blocks = (int64_t)a.N * a.H * ((a.Tq + kBwdRows - 1) / kBwdRows);
		masked_attention_dq_kernel<T, DH, VEC><<<(unsigned)blocks, 256, 0, s>>>(a);
		const hipError_t e = hipGetLastError();
		if (e != hipSuccess) return e;
	}
	if (!(a.dk || a.dv) || a.Tk == 0) return hipSuccess;
	const int64_t blocks = (int64_t)a.N * a.Hkv * ((a.Tk + kBwdRows - 1) / kBwdRows) * a.parts;
	masked_attention_dkv_kernel<T, DH, VEC><<<(unsigned)blocks, 256, 0, s>>>(a);
	const hipError_t e = hipGetLastError();
	if (e != hipSuccess || a.parts == 1) return e;
	const int64_t fours = (int64_t)a.N * a.Hkv * a.Tk * ((a.dh + 3) / 4);
	masked_attention_dkv_join_kernel<T><<<(unsigned)((fours + 255) / 256), 256, 0, s>>>(a);
	return hipGetLastError();
}

template <typename T>
hipError_t backward_of(const MaskedAttentionArgs& a, bool vec, hipStream_t s) {
	if (!vec) return launch_backward<T, 128, false>(a, s);
	if (a.dh <= 64) return launch_backward<T, 64, true>(a, s);
	if (a.dh <= 96) return launch_backward<T, 96, true>(a, s);
	return launch_backward<T, 128, true>(a, s);
}

}  // namespace attn
}  // namespace nnh
