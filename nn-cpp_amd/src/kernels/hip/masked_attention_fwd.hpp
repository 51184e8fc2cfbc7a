// masked_attention_fwd.hpp - the forward kernels of masked attention (masked_attention.hpp), instantiated per element type
// by masked_attention_fwd_*.hip.
//
// One pass over the keys with the running maximum and sum of the softmax. Scores are computed transposed, S^T = K Q^T, so a
// lane holds one query's column: its maximum, sum and rescaling are one number a lane, and P^T goes into O^T += V^T P^T from
// the registers it was computed in (masked_attention_tile.hpp).
//
// Causal, 8192 tokens, 16 heads of 128 on 8 key heads, bf16: 330-360 us, 770-830 TFLOP/s of the pairs seen. The matrix units are
// busy for 37% of that and the vector units (scale, exponential, maximum, sum, rounding: ten operations a score) for 57%; the
// two overlap little, with two waves a SIMD. A wave of 64 queries would halve the reads of LDS, which take about as long as the
// products, but leaves one wave a SIMD. Raising the priority of either phase's waves cost 10%.
// Split form, 32 samples of up to 8192 keys, 8 key heads: 152-159 us for 624 MB, 4.0 TB/s, against 4.7 for a large copy.
#pragma once

#include <type_traits>

#include "masked_attention_tile.hpp"

namespace nnh {
namespace attn {

// A wave's 32 query columns.
template <typename T, int DH>
struct Rows {
	Frag<T> q[DH / 16];
	f32x16 o[DH / 32];
	float m, l;  // maximum in units of log 2, and this half's part of the sum
	Sight s;
	int pos;
	float slope2;

	__device__ __forceinline__ void clear() {
		m = -kInf;
		l = 0.0f;
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
	}
	__device__ __forceinline__ bool bad() const {
		bool r = false;
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int i = 0; i < 16; ++i) r |= not_finite(o[b][i]);
		return r;
	}
};

// Takes the KT keys from k0 on, whose rows are in kt and vt and documents in docs and d, into the wave's columns.
template <typename T, int DH, int KT, bool SAFE, typename At>
__device__ __forceinline__ void take_keys(Rows<T, DH>& r, const MaskedAttentionArgs& a, At at, const char* kt, const char* vt, const int* docs, DocRange d, int k0, int lane) {
	constexpr int RB = row_bytes<T, DH>();
	const int col = lane & 31, half = lane >> 5;
	// whether some of the wave's queries see some of the tile, and whether all of them all of it
	bool some = (k0 < r.s.hi && k0 + KT > r.s.lo) || k0 < r.s.pre;
	bool all = (k0 >= r.s.lo && k0 + KT <= r.s.hi) || k0 + KT <= r.s.pre;
	if (a.k_docs) {
		some = some && r.s.doc >= d.lo && r.s.doc <= d.hi;
		all = all && r.s.doc == d.lo && r.s.doc == d.hi && !d.none;
	}
	if (!__any(some)) return;
	const bool partial = !__all(all);
	const int j0 = fresh(k0 + 4 * half);  // the key of block x's register i: j0 + 32 x + 8 (i / 4) + i % 4

	f32x16 s[KT / 32];
#pragma unroll
	for (int x = 0; x < KT / 32; ++x)
#pragma unroll
		for (int i = 0; i < 16; ++i) s[x][i] = 0.0f;
	constexpr int X = KT / 32, kGroup = sizeof(T) == 2 ? 2 * X : 1;
	in_groups<Frag<T>, DH / 16 * X, kGroup>([&](int i, Frag<T>& k) { at.rows(k, kt + 32 * (i % X) * RB, i / X); },
	                                        [&](int i, const Frag<T>& k) { mma(s[i % X], k, r.q[i / X]); });

	float c = a.scale * kLog2e;  // of the scores as they are, in units of log 2: multiplied in the exponential's own step
	if (a.cap > 0.0f) {
		const float in = a.scale / a.cap;
		c = a.cap * kLog2e;
#pragma unroll
		for (int x = 0; x < KT / 32; ++x)
#pragma unroll
			for (int i = 0; i < 16; ++i) s[x][i] = tanh_of<T>(s[x][i] * in);
	}
	if (a.slopes) {
#pragma unroll
		for (int x = 0; x < KT / 32; ++x)
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				const int d = r.pos - (j0 + 32 * x + 8 * (i / 4) + i % 4);
				s[x][i] = __builtin_fmaf(s[x][i], c, -r.slope2 * (float)(d < 0 ? -d : d));
			}
		c = 1.0f;
	}
	unsigned seen[KT / 32];  // bit i: the lane's query sees the key of register i
	if (partial) {
#pragma unroll
		for (int x = 0; x < KT / 32; ++x) {
			seen[x] = 0;
#pragma unroll
			for (int i = 0; i < 16; ++i) seen[x] |= r.s.sees(j0 + 32 * x + 8 * (i / 4) + i % 4) ? 1u << i : 0u;
			if (a.k_docs) {
#pragma unroll
				for (int g = 0; g < 4; ++g) {
					const i32x4 e = *(const i32x4*)(docs + 32 * x + 8 * g + 4 * half);
#pragma unroll
					for (int i = 0; i < 4; ++i) seen[x] &= e[i] == r.s.doc ? ~0u : ~(1u << (4 * g + i));
				}
			}
#pragma unroll
			for (int i = 0; i < 16; ++i) s[x][i] = seen[x] >> i & 1 ? s[x][i] : -kInf;
		}
	}

	float top = -kInf;
#pragma unroll
	for (int x = 0; x < KT / 32; ++x)
#pragma unroll
		for (int i = 0; i < 16; ++i) top = fmaxf(top, s[x][i]);
	top = max_halves(top) * c;
	// The base follows every new maximum (some of 32 rows have one in four tiles of ten): with one left behind by up to 2^8 no sum
	// would lose precision, but a row's largest weight would no longer be 1, which 16 bits hold exactly, and where a key or two
	// have a row's weight its rounding would be the result's (0.0021 for 0.0017 of the norm over a cache of 8192).
	if (__any(top > r.m)) {
		const float m = fmaxf(r.m, top), f = m == -kInf ? 1.0f : exp2_of(r.m - m);
		r.m = m;
		r.l *= f;
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int i = 0; i < 16; ++i) r.o[b][i] *= f;
	}
	const float base = r.m == -kInf ? 0.0f : r.m;
#pragma unroll
	for (int x = 0; x < KT / 32; ++x)
#pragma unroll
		for (int i = 0; i < 16; ++i) {
			s[x][i] = exp2_of(__builtin_fmaf(s[x][i], c, -base));
			r.l += s[x][i];
		}

	const bool clean = SAFE && partial;
#pragma unroll
	for (int x = 0; x < KT / 32; ++x)
#pragma unroll
		for (int t = 0; t < 2; ++t) {
			Frag<T> p;
			operand_of(p, s[x], t);
#pragma unroll
			for (int b = 0; b < DH / 32; ++b) {
				Frag<T> v;
				at.columns(v, vt + (32 * x + 16 * t) * RB, b);
				if (clean) only_finite(v);
				mma(r.o[b], v, p);
			}
		}
	if (clean) {  // what the product left out, to the queries that see it
#pragma clang loop unroll(disable)
		for (int j = 0; j < KT; ++j) {
			const unsigned word = j < 32 ? seen[0] : seen[KT / 32 - 1];
			const int i = ((j & 31) >> 3) * 4 + (j & 3), owner = col + 32 * ((j >> 2) & 1);
			const bool on = (unsigned)__shfl((int)word, owner) >> i & 1;
#pragma unroll
			for (int b = 0; b < DH / 32; ++b)
#pragma unroll
				for (int x = 0; x < 16; ++x) {
					const float v = element_of<T, DH>(vt, j, 32 * b + 8 * (x / 4) + 4 * half + x % 4);
					r.o[b][x] += on && not_finite(v) ? v : 0.0f;
				}
		}
	}
}

// What a result loses in being rounded to T: out's rounding is half a step of 16 bits, but the backward pass needs g.out to more
// than that (its difference from each g.v is what the gradients are made of where one key has most of a row's weight).
template <typename T>
__device__ __forceinline__ T rest_of(float x, T rounded) {
	const float y = to_float(rounded);
	return not_finite(y) ? (T)0.0f : (T)(x - y);
}

// Stores a column: head row `o` takes the dh sums times f, `rest` (16 bits only, or null) what they lose in their rounding.
template <typename T, int DH, bool VEC>
__device__ __forceinline__ void store_column(T* o, T* rest, const f32x16* x, float f, int dh, int half) {
	if constexpr (VEC && sizeof(T) == 2) {  // (dh is a multiple of 8)
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int g = 0; g < 2; ++g) {
				const int d = 32 * b + 16 * g + 8 * half;
				Frag<T> y, z;
#pragma unroll
				for (int i = 0; i < 8; ++i) {
					y.e[i] = (T)(x[b][8 * g + i] * f);
					z.e[i] = rest_of(x[b][8 * g + i] * f, y.e[i]);
				}
				eight_of(y);
				eight_of(z);
				if (d < dh) *(u32x4*)(o + d) = y.w;
				if (rest && d < dh) *(u32x4*)(rest + d) = z.w;
			}
	} else {
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int g = 0; g < 4; ++g) {
				const int d = 32 * b + 8 * g + 4 * half;
				if constexpr (VEC) {
					if (d < dh) *(f32x4*)(o + d) = f32x4{x[b][4 * g] * f, x[b][4 * g + 1] * f, x[b][4 * g + 2] * f, x[b][4 * g + 3] * f};
				} else {
#pragma unroll
					for (int i = 0; i < 4; ++i)
						if (d + i < dh) {
							const T y = (T)(x[b][4 * g + i] * f);
							o[d + i] = y;
							if (sizeof(T) == 2 && rest) rest[d + i] = rest_of(x[b][4 * g + i] * f, y);
						}
				}
			}
	}
}

constexpr int kWaves = 4, kQueries = 32 * kWaves;

// Keys to a tile: what two buffers of K and V leave two workgroups a CU for (one where a row is 512 bytes or more).
template <typename T, int DH>
constexpr int keys_per_tile() {
	return row_bytes<T, DH>() >= 512 ? 32 : 64;
}

// A workgroup's 128 queries of one head against all keys they see, the tiles read by all four waves.
//
// A masked score is taken out before the maximum, so a masked key's weight is exactly zero; the product with V still
// multiplies it, and zero times an infinity or NaN would reach queries that do not see the key. That shows in the result,
// so where a workgroup ends with one it starts over with such values out of the partly seen tiles' V, adding them to the
// queries that do see them.
template <typename T, int DH, bool VEC>
__global__ __launch_bounds__(256, (row_bytes<T, DH>() >= 512 ? 1 : 2)) void masked_attention_forward_kernel(MaskedAttentionArgs a) {
	constexpr int KT = keys_per_tile<T, DH>(), RB = row_bytes<T, DH>(), kTile = KT * RB;
	__shared__ __attribute__((aligned(1024))) char lds[4 * kTile + 2 * 256 + kWaves * 4];
	char* const docs = lds + 4 * kTile;  // the two tiles'
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;
	// Heads of one key head stay on one XCD where the pairs divide evenly (its L2 then holds their keys); the queries that
	// see most come first.
	const int tiles = (a.Tq + kQueries - 1) / kQueries, pairs = a.N * a.Hkv;
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
	const int q0 = tile * kQueries, i = q0 + wave * 32 + col, hk = h / a.G;
	const int live = live_keys(a, n), pos0 = first_position(a, n);
	const T* const kbase = (const T*)a.k + n * a.ks.sample + hk * a.ks.head;
	const T* const vbase = (const T*)a.v + n * a.vs.sample + hk * a.vs.head;

	Rows<T, DH> r;
	r.s = sight_of(a, n, i, live, pos0);
	r.pos = pos0 + i;
	r.slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
	{
		const T* row = (const T*)a.q + n * a.qs.sample + (int64_t)min(i, a.Tq - 1) * a.qs.row + h * a.qs.head;
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) row_from<T, VEC>(r.q[t], row, a.dh, half, t, i < a.Tq);
	}
	// what the workgroup's queries can see at most (positions, then documents)
	int lo = 0, hi = live, pre = a.prefix ? clamped(a.prefix[n], 0, live) : 0;
	{
		const int64_t first = (int64_t)pos0 + q0, last = (int64_t)pos0 + min(q0 + kQueries, a.Tq) - 1;
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
	arrived(r.q);
	arrived();

	constexpr bool kPlaces = sizeof(T) == 2 && VEC;
	const std::conditional_t<kPlaces, Places<T, DH>, int> places(lane);
	auto at = [&] {
		if constexpr (kPlaces) return places;
		else return Reader<T, RB>(fresh_lane());
	};
	auto run = [&](auto safe) {
		r.clear();
		// the tiles that some query may see, 64 at a time
		int base = -64;
		uint64_t on = 0;
		auto next = [&]() -> int {
			while (on == 0) {
				base += 64;
				if (base >= nt) return -1;
				const int x = base + lane, k0 = x * KT;
				bool see = x < nt && ((k0 < hi && k0 + KT > lo) || k0 < pre);
				if (see && a.k_docs) {
					const DocRange d = a.k_ranges[(int64_t)n * kb + k0 / 64];
					see = d.lo <= mine.hi && d.hi >= mine.lo;
				}
				on = __ballot(see);
			}
			const int x = __builtin_ctzll(on);
			on &= on - 1;
			return base + x;
		};
		auto load = [&](int x, char* to, char* docs_to) {
			if (a.k_docs && wave == 0) load_numbers(a.k_docs + (int64_t)n * a.Tk + min(x * KT + lane, a.Tk - 1), docs_to);
			load_tile<T, DH, KT, kWaves, VEC>(to, kbase + (int64_t)x * KT * a.ks.row, a.ks.row, live - x * KT, a.dh, wave, lane);
			load_tile<T, DH, KT, kWaves, VEC>(to + kTile, vbase + (int64_t)x * KT * a.vs.row, a.vs.row, live - x * KT, a.dh, wave, lane);
		};
		int cur = next();
		// one tile from `from`, the next one on its way to `to`
		auto step = [&](auto buf) {
			constexpr int B = decltype(buf)::value;
			char* const from = lds + B * 2 * kTile;
			wait_loads();
			__builtin_amdgcn_s_barrier();  // this tile has arrived for all waves, and all are done with the last one
			asm volatile("" ::: "memory");
			DocRange d{0, 0, 0};
			if (a.k_docs) d = range_at(a.k_ranges, (int64_t)n * kb + cur * KT / 64);
			const int then = next();
			if (then >= 0) load(then, lds + (1 - B) * 2 * kTile, docs + (1 - B) * 256);
			take_keys<T, DH, KT, decltype(safe)::value>(r, a, at(), from, from + kTile, (const int*)(docs + B * 256), d, cur * KT, lane);
			cur = then;
		};
		if (cur >= 0) load(cur, lds, docs);
		while (cur >= 0) {
			step(std::integral_constant<int, 0>{});
			if (cur >= 0) step(std::integral_constant<int, 1>{});
		}
		return any_wave<kWaves>((int*)(docs + 2 * 256), wave, lane, r.bad());
	};
	if (run(std::false_type{})) run(std::true_type{});

	const float l = add_halves(r.l);
	if (i < a.Tq) {
		T* o = (T*)a.out + n * a.os.sample + (int64_t)i * a.os.row + h * a.os.head;
		T* rest = a.rest ? (T*)a.rest + n * a.rs.sample + (int64_t)i * a.rs.row + h * a.rs.head : nullptr;
		store_column<T, DH, VEC>(o, rest, r.o, l == 0.0f ? 0.0f : 1.0f / l, a.dh, half);
		if (half == 0) a.lse[((int64_t)n * a.H + h) * a.Tq + i] = l == 0.0f ? -kInf : r.m * kLn2 + logf(l);
	}
}

// The split form, for few query rows: the G heads of a key head and the Tq queries together are the columns (32 to a
// workgroup), and the keys are divided over the grid and over a workgroup's waves, each with a ring of tiles of its own: of four
// where LDS holds them, two for rows of 256 bytes, and one, with no load ahead of its use, for fp32 heads of more than 64.
template <typename T, int DH>
struct SplitShape {
	static constexpr int KT = 32, RB = row_bytes<T, DH>(), kTile = KT * RB, kStage = 2 * kTile;
	static constexpr int NW = 4;
	static constexpr int ST = kStage * NW * 4 <= 128 * 1024 ? 4 : kStage * NW * 2 <= 128 * 1024 ? 2 : 1;
	static constexpr int kLoads = 2 * kTile / 1024;  // a wave's load instructions for a stage
	static constexpr int kMerge = NW * 32 * (DH + 4) * 4;
	static constexpr int kLds = NW * ST * kStage > kMerge ? NW * ST * kStage : kMerge;
	static_assert(kLds + NW * ST * 256 + NW * 4 <= 160 * 1024 && (ST - 1) * kLoads <= 63, "LDS, and loads that a wave may have outstanding");
};

template <typename T, int DH, bool VEC>
__global__ __launch_bounds__((64 * SplitShape<T, DH>::NW), 1) void masked_attention_split_kernel(MaskedAttentionArgs a) {
	using S = SplitShape<T, DH>;
	constexpr int KT = S::KT, NW = S::NW, ST = S::ST;
	__shared__ __attribute__((aligned(1024))) char lds[S::kLds + NW * ST * 256 + NW * 4];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;
	const int columns = a.Tq * a.G, pairs = a.N * a.Hkv;
	const int split = blockIdx.x % a.splits, pair = blockIdx.x / a.splits % pairs, group = blockIdx.x / a.splits / pairs;
	const int n = pair / a.Hkv, hk = pair % a.Hkv, c = group * 32 + col;
	const bool on_col = c < columns;
	const int i = on_col ? c / a.G : a.Tq, h = hk * a.G + (on_col ? c % a.G : 0);
	const int live = live_keys(a, n), pos0 = first_position(a, n);
	const T* const kbase = (const T*)a.k + n * a.ks.sample + hk * a.ks.head;
	const T* const vbase = (const T*)a.v + n * a.vs.sample + hk * a.vs.head;

	Rows<T, DH> r;
	r.s = sight_of(a, n, i, live, pos0);
	r.pos = pos0 + i;
	r.slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
	{
		const T* row = (const T*)a.q + n * a.qs.sample + (int64_t)min(i, a.Tq - 1) * a.qs.row + h * a.qs.head;
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) row_from<T, VEC>(r.q[t], row, a.dh, half, t, on_col);
	}
	// the keys that some query of the sample may see, divided into splits * NW runs of whole tiles
	int lo = 0, hi = live;
	const int pre = a.prefix ? clamped(a.prefix[n], 0, live) : 0;
	{
		const int64_t last = (int64_t)pos0 + a.Tq - 1;
		if (a.causal) hi = clamped(last + 1, 0, live);
		if (a.window) {
			lo = clamped((int64_t)pos0 - a.window + 1, 0, live);
			hi = min(hi, clamped(last + a.window, 0, live));
		}
		if (pre) lo = 0;
		hi = max(hi, pre);
	}
	const int t0 = lo / KT, t1 = (hi + KT - 1) / KT, per = (max(t1 - t0, 0) + a.splits * NW - 1) / (a.splits * NW);
	const int begin = min(t0 + (split * NW + wave) * per, t1), end = min(begin + per, t1);
	char* const ring = lds + wave * ST * S::kStage;
	char* const docs = lds + S::kLds + wave * ST * 256;
	arrived(r.q);
	arrived();

	auto run = [&](auto safe) {
		r.clear();
		auto load = [&](int x, int stage) {
			char* to = ring + stage * S::kStage;
			if (a.k_docs) load_numbers(a.k_docs + (int64_t)n * a.Tk + min(x * KT + lane, a.Tk - 1), docs + stage * 256);
			load_tile<T, DH, KT, 1, VEC>(to, kbase + (int64_t)x * KT * a.ks.row, a.ks.row, live - x * KT, a.dh, 0, lane);
			load_tile<T, DH, KT, 1, VEC>(to + S::kTile, vbase + (int64_t)x * KT * a.vs.row, a.vs.row, live - x * KT, a.dh, 0, lane);
		};
#pragma unroll
		for (int x = 0; x < ST - 1; ++x)
			if (begin + x < end) load(begin + x, x);
		int stage = 0;
		for (int x = begin; x < end; ++x) {
			if (ST > 1) {
				if (x + ST - 1 < end) {
					load(x + ST - 1, (stage + ST - 1) % ST);
					asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((ST - 1) * S::kLoads) : "memory");
				} else {
					wait_loads();
				}
			} else {
				load(x, 0);
				wait_loads();
			}
			const char* from = ring + stage * S::kStage;
			DocRange d{0, 0, 0};
			if (a.k_docs) d = range_at(a.k_ranges, (int64_t)n * ((a.Tk + 63) / 64) + x * KT / 64);
			take_keys<T, DH, KT, decltype(safe)::value>(r, a, Reader<T, S::RB>(fresh_lane()), from, from + S::kTile, (const int*)(docs + stage * 256), d, x * KT, lane);
			// the stage is loaded over next: its reads are done
			asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
			stage = (stage + 1) % ST;
		}
		return any_wave<NW>((int*)(lds + S::kLds + NW * ST * 256), wave, lane, r.bad());
	};
	if (run(std::false_type{})) run(std::true_type{});

	// the waves' parts, merged in their order
	float* const part = (float*)lds;  // {NW, 32, DH + 4}
	r.l = add_halves(r.l);
	{
		float* at = part + (wave * 32 + col) * (DH + 4);
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int g = 0; g < 4; ++g)
				*(f32x4*)(at + 32 * b + 8 * g + 4 * half) = f32x4{r.o[b][4 * g], r.o[b][4 * g + 1], r.o[b][4 * g + 2], r.o[b][4 * g + 3]};
		if (half == 0) {
			at[DH] = r.m;
			at[DH + 1] = r.l;
		}
	}
	__syncthreads();
	for (int x = wave; x < 32 && group * 32 + x < columns; x += NW) {
		const int cc = group * 32 + x, ii = cc / a.G, hh = hk * a.G + cc % a.G;
		float m = -kInf, l = 0.0f, f[NW];
#pragma unroll
		for (int w = 0; w < NW; ++w) m = fmaxf(m, part[(w * 32 + x) * (DH + 4) + DH]);
		const float base = m == -kInf ? 0.0f : m;
#pragma unroll
		for (int w = 0; w < NW; ++w) {
			f[w] = exp2_of(part[(w * 32 + x) * (DH + 4) + DH] - base);
			l += f[w] * part[(w * 32 + x) * (DH + 4) + DH + 1];
		}
		const int64_t row = ((int64_t)n * a.H + hh) * a.Tq + ii;
		float* const to = a.partial + ((int64_t)split * a.N * a.H * a.Tq + row) * (a.dh + 2);
		T* const o = (T*)a.out + n * a.os.sample + (int64_t)ii * a.os.row + hh * a.os.head;
		const float inv = l == 0.0f ? 0.0f : 1.0f / l;
		for (int d = lane; d < a.dh; d += 64) {
			float y = 0.0f;
#pragma unroll
			for (int w = 0; w < NW; ++w) y += f[w] * part[(w * 32 + x) * (DH + 4) + d];
			if (a.splits == 1) {
				o[d] = (T)(y * inv);
				if (sizeof(T) == 2 && a.rest) ((T*)a.rest)[n * a.rs.sample + (int64_t)ii * a.rs.row + hh * a.rs.head + d] = rest_of(y * inv, (T)(y * inv));
			} else {
				to[2 + d] = y;
			}
		}
		if (lane == 0) {
			if (a.splits == 1) {
				a.lse[row] = l == 0.0f ? -kInf : m * kLn2 + logf(l);
			} else {
				to[0] = m;
				to[1] = l;
			}
		}
	}
}

// Joins the split form's parts, one wave to a row, in their order.
template <typename T>
__global__ __launch_bounds__(256) void masked_attention_join_kernel(MaskedAttentionArgs a) {
	const int lane = threadIdx.x & 63;
	const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (int64_t)a.N * a.H * a.Tq;
	if (row >= rows) return;
	const int i = (int)(row % a.Tq), h = (int)(row / a.Tq % a.H), n = (int)(row / a.Tq / a.H);
	const int64_t step = rows * (a.dh + 2);
	const float* const from = a.partial + row * (a.dh + 2);
	float m = -kInf;
	for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, from[s * step]);
	for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
	const float base = m == -kInf ? 0.0f : m;
	float l = 0.0f, y[2] = {0.0f, 0.0f};
	for (int s = 0; s < a.splits; ++s) {
		const float* p = from + s * step;
		const float f = exp2_of(p[0] - base);
		l += f * p[1];
#pragma unroll
		for (int x = 0; x < 2; ++x)
			if (lane + 64 * x < a.dh) y[x] += f * p[2 + lane + 64 * x];
	}
	T* const o = (T*)a.out + n * a.os.sample + (int64_t)i * a.os.row + h * a.os.head;
	const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
	for (int x = 0; x < 2; ++x)
		if (lane + 64 * x < a.dh) {
			o[lane + 64 * x] = (T)(y[x] * inv);
			if (sizeof(T) == 2 && a.rest) ((T*)a.rest)[n * a.rs.sample + (int64_t)i * a.rs.row + h * a.rs.head + lane + 64 * x] = rest_of(y[x] * inv, (T)(y[x] * inv));
		}
	if (lane == 0) a.lse[row] = l == 0.0f ? -kInf : m * kLn2 + logf(l);
}

template <typename T, int DH, bool VEC>
hipError_t launch_forward(const MaskedAttentionArgs& a, hipStream_t s) {
	const int64_t blocks = (int64_t)a.N * a.H * ((a.Tq + kQueries - 1) / kQueries);
	masked_attention_forward_kernel<T, DH, VEC><<<(unsigned)blocks, 256, 0, s>>>(a);
	return hipGetLastError();
}

template <typename T, int DH, bool VEC>
hipError_t launch_split(const MaskedAttentionArgs& a, hipStream_t s) {
	const int64_t groups = ((int64_t)a.Tq * a.G + 31) / 32, blocks = groups * a.N * a.Hkv * a.splits;
	masked_attention_split_kernel<T, DH, VEC><<<(unsigned)blocks, 64 * SplitShape<T, DH>::NW, 0, s>>>(a);
	hipError_t e = hipGetLastError();
	if (e != hipSuccess || a.splits == 1) return e;
	const int64_t rows = (int64_t)a.N * a.H * a.Tq;
	masked_attention_join_kernel<T><<<(unsigned)((rows + 3) / 4), 256, 0, s>>>(a);
	return hipGetLastError();
}

// The head width that a kernel is built for; rows that are not 16-byte aligned take the widest.
template <typename T>
hipError_t forward_of(const MaskedAttentionArgs& a, bool vec, bool split, hipStream_t s) {
#define NNH_ATTN(DH, VEC) (split ? launch_split<T, DH, VEC>(a, s) : launch_forward<T, DH, VEC>(a, s))
	if (!vec) return NNH_ATTN(128, false);
	if (a.dh <= 64) return NNH_ATTN(64, true);
	if (a.dh <= 96) return NNH_ATTN(96, true);
	return NNH_ATTN(128, true);
#undef NNH_ATTN
}

}  // namespace attn
}  // namespace nnh
