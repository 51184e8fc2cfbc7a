// paged_attention_fwd.hpp - the kernels of attention over pages, instantiated per element type by paged_attention_*.hip.
//
// The products and the softmax are masked attention's (take_keys in masked_attention_fwd.hpp): scores transposed, a lane holds
// one column's statistics, probabilities enter the second product from the registers they were made in. What differs is where
// columns and tiles come from. The columns are a sequence's rows times the query heads of one key head, head by head within a
// row, so that all heads of a key head read its tiles once and a causal workgroup of 128 columns spans few positions. A tile's
// rows lie in pages: lane l holds the place of the tile's row l, worked out from the page numbers of that tile, which were
// loaded into LDS a tile (split form: a ring of tiles) earlier, so that no load waits for another one's address. Pages may end
// anywhere in a tile.
#pragma once

#include "masked_attention_fwd.hpp"
#include "paged_attention.hpp"

namespace nnh {
namespace attn {

// A sequence's rows and tokens.
struct Sequence {
	int first, count;  // rows
	int pos0;          // position of the first row
	int live;          // tokens that have a place in the table
};

__device__ __forceinline__ Sequence sequence_of(const PackedRows& s, const PageTable& t, int n) {
	Sequence q;
	q.first = clamped(s.starts[n], 0, s.rows);
	q.count = clamped(s.starts[n + 1], q.first, s.rows) - q.first;
	const int len = clamped(s.lens[n], 0, 1 << 30);
	q.pos0 = len - q.count;
	q.live = t.pages > 0 ? (int)min((int64_t)len, (int64_t)t.width * t.size.d) : 0;
	return q;
}

// Keys that the rows of a sequence from position `first` to `last` may see: tiles of KT keys, numbered in one go over those of the
// prefix and those of the causal or window range.
template <int KT>
struct Tiles {
	int lo, hi, pre;    // keys lo .. hi - 1 and those below pre
	int prefix, skip, count;  // tiles of the prefix; tiles left out behind them; tiles in all
	__device__ __forceinline__ Tiles(const MaskedAttentionArgs& a, int n, int64_t first, int64_t last, int live) {
		lo = 0;
		hi = live;
		pre = a.prefix ? clamped(a.prefix[n], 0, live) : 0;
		if (a.causal) hi = clamped(last + 1, 0, live);
		if (a.window) {
			lo = clamped(first - a.window + 1, 0, live);
			hi = min(hi, clamped(last + a.window, 0, live));
		}
		prefix = (pre + KT - 1) / KT;
		const int from = max(lo / KT, prefix), to = max((hi + KT - 1) / KT, from);
		skip = from - prefix;
		count = prefix + to - from;
	}
	__device__ __forceinline__ int at(int t) const { return t < prefix ? t : t + skip; }
};

// A tile's rows: lane l's is row l % KT.
struct Places64 {
	int64_t at;  // of the lane's row, in elements from the head's first
	bool bad;    // the row has no page
};

// Loads the page numbers of tile x's rows, one to a lane.
template <int KT>
__device__ __forceinline__ void load_pages(const PageTable& t, int n, int x, int live, int lane, char* to) {
	const unsigned j = (unsigned)min(x * KT + (lane & (KT - 1)), live - 1);
	load_numbers(t.table + (int64_t)n * t.width + fdiv(j, t.size), to);
}

template <int KT>
__device__ __forceinline__ Places64 places_of(const PageTable& t, int x, int live, int lane, const char* pages) {
	const unsigned j = (unsigned)min(x * KT + (lane & (KT - 1)), live - 1);
	const int page = ((const int*)pages)[lane];
	Places64 p;
	p.bad = (unsigned)page >= (unsigned)t.pages;
	p.at = (p.bad ? 0 : page) * t.page + (int64_t)(j - fdiv(j, t.size) * t.size.d) * t.slot;
	return p;
}

__device__ __forceinline__ int64_t from_lane(int64_t x, int lane) {
	const unsigned lo = __shfl((int)(unsigned)x, lane), hi = __shfl((int)(unsigned)((uint64_t)x >> 32), lane);
	return (int64_t)((uint64_t)hi << 32 | lo);
}

// Tiles of K and V of R rows that lie at `at` (a lane each) from kb and vb, NW waves sharing the work (load_tile's, with a row's
// place in the place of a stride).
template <typename T, int DH, int R, int NW, bool VEC>
__device__ __forceinline__ void load_rows(char* kt, char* vt, const T* kb, const T* vb, int64_t at, int dh, int wave, int lane) {
	constexpr int RB = row_bytes<T, DH>(), W = RB / 16, E = 16 / (int)sizeof(T), kSteps = R * RB / 1024 / NW, kRows = 64 / W;
	static_assert(kSteps * NW * 1024 == R * RB, "a tile splits evenly over the waves");
	if constexpr (VEC) {
		const unsigned kto = lds_place(kt + wave * 1024), vto = lds_place(vt + wave * 1024);
		each<kSteps>([&](auto step) {
			constexpr int j = decltype(step)::value;
			const int row = (j * NW + wave) * kRows + lane / W, c = (lane % W) ^ swizzle<RB>(row);
			const int64_t o = from_lane(at, row) + c * E;
			const void* k = kb + o;
			const void* v = vb + o;
			if (c * E >= dh) k = v = &kZeroWord;  // depths past dh multiply zeros: finite ones
			if (DH * (int)sizeof(T) == RB || c * E < DH) {
				load_words<j * NW * 1024>(k, kto);
				load_words<j * NW * 1024>(v, vto);
			}
		});
	} else {
#pragma unroll 1
		for (int j = 0; j < kSteps; ++j) {
			const int first = (j * NW + wave) * 64, row = (first + lane) / W, c = ((first + lane) % W) ^ swizzle<RB>(row);
			const int64_t o = from_lane(at, row) + c * E;
			union {
				T e[E];
				u32x4 w;
			} x, y;
#pragma unroll
			for (int i = 0; i < E; ++i) {
				x.e[i] = c * E + i < dh ? kb[o + i] : (T)0.0f;
				y.e[i] = c * E + i < dh ? vb[o + i] : (T)0.0f;
			}
			*(u32x4*)(kt + (first + lane) * 16) = x.w;
			*(u32x4*)(vt + (first + lane) * 16) = y.w;
		}
	}
}

// What take_keys needs to know of a tile with rows that have no page: those are of no document, the others of document 0.
template <int KT>
__device__ __forceinline__ bool mark_bad(const Places64& p, int* marks, int lane) {
	const bool any = __any(p.bad);
	if (any) marks[lane & (KT - 1)] = p.bad ? -1 : 0;
	return any;
}

template <typename T, int DH>
__device__ __forceinline__ void begin_column(Rows<T, DH>& r, const PagedAttentionArgs& p, const MaskedAttentionArgs& a, const Sequence& s, int n, int i, int h) {
	r.s = sight_of(a, n, i, s.live, s.pos0);
	r.pos = s.pos0 + i;
	r.slope2 = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
}

// A workgroup's 128 columns of one sequence and key head against the keys they see, or one part of `wide_splits` of these; the
// tiles are read by all four waves. Values that are not finite in masked places: as in masked_attention_forward_kernel.
template <typename T, int DH, bool VEC>
__global__ __launch_bounds__(256, (row_bytes<T, DH>() >= 512 ? 1 : 2)) void paged_attention_kernel(PagedAttentionArgs p) {
	constexpr int KT = keys_per_tile<T, DH>(), RB = row_bytes<T, DH>(), kTile = KT * RB;
	__shared__ __attribute__((aligned(1024))) char lds[4 * kTile + 2 * 256 + 2 * kWaves * 256 + kWaves * 4];
	char* const pages = lds + 4 * kTile;  // page numbers of two tiles
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	int* const marks = (int*)(pages + 2 * 256 + wave * 2 * 256);  // the wave's own, of two tiles
	const int col = lane & 31, half = lane >> 5;
	// Tiles of one key head stay on one XCD where the pairs divide evenly (its L2 then holds the keys); those that see most come first.
	const int pairs = p.s.N * p.a.Hkv, splits = p.wide_splits;
	int tile, part, hk, n;
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
		n = pair / p.a.Hkv;
		hk = pair % p.a.Hkv;
		part = rest % splits;
		tile = rest / splits;
	}
	const Sequence s = sequence_of(p.s, p.t, n);
	MaskedAttentionArgs a = p.a;
	a.Tq = min(s.count, p.most);
	const int columns = a.Tq * a.G, tiles = (columns + kQueries - 1) / kQueries;
	if (columns <= p.few || tile >= tiles) return;
	tile = tiles - 1 - tile;
	const int c0 = tile * kQueries, c = c0 + wave * 32 + col;
	const int i = c < columns ? c / a.G : a.Tq, h = hk * a.G + c % a.G;
	const T* const kbase = (const T*)a.k + hk * p.t.head;
	const T* const vbase = (const T*)a.v + hk * p.t.head;

	Rows<T, DH> r;
	begin_column(r, p, a, s, n, i, h);
	{
		const T* row = (const T*)a.q + (int64_t)(s.first + min(i, a.Tq - 1)) * a.qs.row + h * a.qs.head;
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) row_from<T, VEC>(r.q[t], row, a.dh, half, t, i < a.Tq);
	}
	const Tiles<KT> seen(a, n, (int64_t)s.pos0 + c0 / a.G, (int64_t)s.pos0 + (min(c0 + kQueries, columns) - 1) / a.G, s.live);
	const int begin = (int)((int64_t)seen.count * part / splits), end = (int)((int64_t)seen.count * (part + 1) / splits);
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
		bool bad[2] = {false, false};
		// Tile t of the part into buffer B, its page numbers having arrived.
		auto load = [&](int t, auto buf) {
			constexpr int B = decltype(buf)::value;
			const Places64 x = places_of<KT>(p.t, seen.at(t), s.live, lane, pages + B * 256);
			bad[B] = mark_bad<KT>(x, marks + B * 64, lane);
			load_rows<T, DH, KT, kWaves, VEC>(lds + B * 2 * kTile, lds + B * 2 * kTile + kTile, kbase, vbase, x.at, a.dh, wave, lane);
		};
		auto step = [&](int t, auto buf) {
			constexpr int B = decltype(buf)::value;
			char* const from = lds + B * 2 * kTile;
			wait_loads();
			__builtin_amdgcn_s_barrier();  // this tile and the next one's page numbers have arrived for all waves, which are done with the last tile
			asm volatile("" ::: "memory");
			if (t + 1 < end) {
				load(t + 1, std::integral_constant<int, 1 - B>{});
				// (all waves have read the numbers that these replace before the barrier)
				if (wave == 0 && t + 2 < end) load_pages<KT>(p.t, n, seen.at(t + 2), s.live, lane, pages + B * 256);
			}
			a.k_docs = bad[B] ? p.t.table : nullptr;
			take_keys<T, DH, KT, decltype(safe)::value>(r, a, at(), from, from + kTile, marks + B * 64, DocRange{0, 0, 1}, seen.at(t) * KT, lane);
		};
		if (begin < end) {
			if (wave == 0) {
				load_pages<KT>(p.t, n, seen.at(begin), s.live, lane, pages);
				if (begin + 1 < end) load_pages<KT>(p.t, n, seen.at(begin + 1), s.live, lane, pages + 256);
			}
			wait_loads();
			__syncthreads();
			load(begin, std::integral_constant<int, 0>{});
		}
		for (int t = begin; t < end; t += 2) {
			step(t, std::integral_constant<int, 0>{});
			if (t + 1 < end) step(t + 1, std::integral_constant<int, 1>{});
		}
		return any_wave<kWaves>((int*)(pages + 2 * 256 + 2 * kWaves * 256), wave, lane, r.bad());
	};
	if (run(std::false_type{})) run(std::true_type{});

	const float l = add_halves(r.l);
	if (i >= a.Tq) return;
	const int64_t row = s.first + i;
	if (splits == 1) {
		T* o = (T*)a.out + row * a.os.row + h * a.os.head;
		store_column<T, DH, VEC>(o, (T*)nullptr, r.o, l == 0.0f ? 0.0f : 1.0f / l, a.dh, half);
		if (half == 0) p.lse[row * a.H + h] = l == 0.0f ? -kInf : r.m * kLn2 + logf(l);
	} else {
		float* const to = p.partial + (((int64_t)part * p.s.rows + row) * a.H + h) * (a.dh + 2);
#pragma unroll
		for (int b = 0; b < DH / 32; ++b)
#pragma unroll
			for (int x = 0; x < 16; ++x) {
				const int d = 32 * b + 8 * (x / 4) + 4 * half + x % 4;
				if (d < a.dh) to[2 + d] = r.o[b][x];
			}
		if (half == 0) {
			to[0] = r.m;
			to[1] = l;
		}
	}
}

// The split form, for sequences of few columns: 32 to a workgroup, the keys divided over the grid and over a workgroup's waves,
// each with a ring of tiles and of page numbers of its own.
template <typename T, int DH>
struct PagedSplitShape : SplitShape<T, DH> {
	using S = SplitShape<T, DH>;
	static constexpr int kPages = 2 * S::ST * 256, kMarks = S::ST * 128;  // of a wave
	static constexpr int kAll = S::kLds + S::NW * (kPages + kMarks) + S::NW * 4;
	static_assert(kAll <= 160 * 1024 && (S::ST - 1) * (S::kLoads + 1) <= 63, "LDS, and loads that a wave may have outstanding");
};

template <typename T, int DH, bool VEC>
__global__ __launch_bounds__((64 * SplitShape<T, DH>::NW), 1) void paged_attention_split_kernel(PagedAttentionArgs p) {
	using S = PagedSplitShape<T, DH>;
	constexpr int KT = S::KT, NW = S::NW, ST = S::ST;
	__shared__ __attribute__((aligned(1024))) char lds[S::kAll];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;
	const int pairs = p.s.N * p.a.Hkv;
	const int split = blockIdx.x % p.splits, pair = blockIdx.x / p.splits % pairs, group = blockIdx.x / p.splits / pairs;
	const int n = pair / p.a.Hkv, hk = pair % p.a.Hkv;
	const Sequence s = sequence_of(p.s, p.t, n);
	MaskedAttentionArgs a = p.a;
	a.Tq = min(s.count, p.most);
	const int columns = a.Tq * a.G, c = group * 32 + col;
	if (columns > p.few || group * 32 >= columns) return;
	const bool on_col = c < columns;
	const int i = on_col ? c / a.G : a.Tq, h = hk * a.G + (on_col ? c % a.G : 0);
	const T* const kbase = (const T*)a.k + hk * p.t.head;
	const T* const vbase = (const T*)a.v + hk * p.t.head;

	Rows<T, DH> r;
	begin_column(r, p, a, s, n, i, h);
	{
		const T* row = (const T*)a.q + (int64_t)(s.first + min(i, a.Tq - 1)) * a.qs.row + h * a.qs.head;
#pragma unroll
		for (int t = 0; t < DH / 16; ++t) row_from<T, VEC>(r.q[t], row, a.dh, half, t, on_col);
	}
	// the keys that some row of the sequence may see, divided into splits * NW runs of whole tiles
	const Tiles<KT> seen(a, n, s.pos0, (int64_t)s.pos0 + a.Tq - 1, s.live);
	const int per = (seen.count + p.splits * NW - 1) / (p.splits * NW);
	const int begin = min((split * NW + wave) * per, seen.count), end = min(begin + per, seen.count);
	char* const ring = lds + wave * ST * S::kStage;
	char* const pages = lds + S::kLds + wave * S::kPages;
	int* const marks = (int*)(lds + S::kLds + NW * S::kPages + wave * S::kMarks);
	arrived(r.q);
	arrived();

	auto run = [&](auto safe) {
		r.clear();
		unsigned bad = 0;  // bit: the stage's tile has rows without a page
		// (numbers past the run's end are some tile's of the sequence: loaded for the count of loads alone)
		auto numbers = [&](int t) { load_pages<KT>(p.t, n, seen.at(min(t, seen.count - 1)), s.live, lane, pages + t % (2 * ST) * 256); };
		auto load = [&](int t, int stage) {
			const Places64 x = places_of<KT>(p.t, seen.at(t), s.live, lane, pages + t % (2 * ST) * 256);
			bad = (bad & ~(1u << stage)) | (mark_bad<KT>(x, marks + stage * KT, lane) ? 1u << stage : 0u);
			char* to = ring + stage * S::kStage;
			load_rows<T, DH, KT, 1, VEC>(to, to + S::kTile, kbase, vbase, x.at, a.dh, 0, lane);
		};
		if (begin < end) {
			for (int x = 0; x < ST; ++x) numbers(begin + x);
			wait_loads();
		}
#pragma unroll
		for (int x = 0; x < ST - 1; ++x)
			if (begin + x < end) {
				numbers(begin + ST + x);
				load(begin + x, x);
			}
		int stage = 0;
		for (int t = begin; t < end; ++t) {
			// Before a tile's loads go the numbers of one ST tiles further: when a tile has arrived, so have the numbers that the
			// loads of the next round need.
			if (t + ST - 1 < end) {
				numbers(t + 2 * ST - 1);
				load(t + ST - 1, (stage + ST - 1) % ST);
				asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((ST - 1) * (S::kLoads + 1)) : "memory");
			} else {
				wait_loads();
			}
			const char* from = ring + stage * S::kStage;
			a.k_docs = bad >> stage & 1 ? p.t.table : nullptr;
			take_keys<T, DH, KT, decltype(safe)::value>(r, a, Reader<T, S::RB>(fresh_lane()), from, from + S::kTile, marks + stage * KT, DocRange{0, 0, 1}, seen.at(t) * KT, lane);
			// the stage is loaded over next: its reads are done
			asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
			stage = (stage + 1) % ST;
		}
		return any_wave<NW>((int*)(lds + S::kLds + NW * (S::kPages + S::kMarks)), wave, lane, r.bad());
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
		const int64_t row = s.first + ii;
		float* const to = p.partial + (((int64_t)split * p.s.rows + row) * a.H + hh) * (a.dh + 2);
		T* const o = (T*)a.out + row * a.os.row + hh * a.os.head;
		const float inv = l == 0.0f ? 0.0f : 1.0f / l;
		for (int d = lane; d < a.dh; d += 64) {
			float y = 0.0f;
#pragma unroll
			for (int w = 0; w < NW; ++w) y += f[w] * part[(w * 32 + x) * (DH + 4) + d];
			if (p.splits == 1) o[d] = (T)(y * inv);
			else to[2 + d] = y;
		}
		if (lane == 0) {
			if (p.splits == 1) {
				p.lse[row * a.H + hh] = l == 0.0f ? -kInf : m * kLn2 + logf(l);
			} else {
				to[0] = m;
				to[1] = l;
			}
		}
	}
}

// Joins the parts, one wave to a row and head, in their order.
template <typename T>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(PagedAttentionArgs p) {
	const int lane = threadIdx.x & 63;
	const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
	if (at >= (int64_t)p.s.rows * p.a.H) return;
	const int row = (int)(at / p.a.H), h = (int)(at % p.a.H);
	// the sequence that has the row, by its bounds in order
	int lo = 0, hi = p.s.N;
	while (lo < hi) {
		const int mid = (lo + hi) / 2;
		if (p.s.starts[mid + 1] <= row) lo = mid + 1;
		else hi = mid;
	}
	if (lo == p.s.N) return;
	const Sequence s = sequence_of(p.s, p.t, lo);
	const int count = min(s.count, p.most);
	if (row < s.first || row >= s.first + count) return;
	const int splits = count * p.a.G <= p.few ? p.splits : p.wide_splits;
	if (splits == 1) return;
	const int64_t step = (int64_t)p.s.rows * p.a.H * (p.a.dh + 2);
	const float* const from = p.partial + at * (p.a.dh + 2);
	float m = -kInf;
	for (int x = lane; x < splits; x += 64) m = fmaxf(m, from[x * step]);
	for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
	const float base = m == -kInf ? 0.0f : m;
	float l = 0.0f, y[2] = {0.0f, 0.0f};
	for (int x = 0; x < splits; ++x) {
		const float* q = from + x * step;
		const float f = exp2_of(q[0] - base);
		l += f * q[1];
#pragma unroll
		for (int d = 0; d < 2; ++d)
			if (lane + 64 * d < p.a.dh) y[d] += f * q[2 + lane + 64 * d];
	}
	T* const o = (T*)p.a.out + row * p.a.os.row + h * p.a.os.head;
	const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
	for (int d = 0; d < 2; ++d)
		if (lane + 64 * d < p.a.dh) o[lane + 64 * d] = (T)(y[d] * inv);
	if (lane == 0) p.lse[at] = l == 0.0f ? -kInf : m * kLn2 + logf(l);
}

template <typename T, int DH, bool VEC>
hipError_t launch_paged(const PagedAttentionArgs& p, hipStream_t s) {
	const int64_t pairs = (int64_t)p.s.N * p.a.Hkv, most = (int64_t)p.most * p.a.G;  // (checked to be an int)
	hipError_t e = hipSuccess;
	if (p.wide_splits) {
		paged_attention_kernel<T, DH, VEC><<<(unsigned)(pairs * ((most + kQueries - 1) / kQueries) * p.wide_splits), 256, 0, s>>>(p);
		e = hipGetLastError();
	}
	if (e == hipSuccess && p.splits) {
		const int64_t groups = ((most < p.few ? most : p.few) + 31) / 32;
		paged_attention_split_kernel<T, DH, VEC><<<(unsigned)(pairs * groups * p.splits), 64 * SplitShape<T, DH>::NW, 0, s>>>(p);
		e = hipGetLastError();
	}
	if (e == hipSuccess && (p.wide_splits > 1 || p.splits > 1)) {
		paged_attention_join_kernel<T><<<(unsigned)(((int64_t)p.s.rows * p.a.H + 3) / 4), 256, 0, s>>>(p);
		e = hipGetLastError();
	}
	return e;
}

template <typename T>
hipError_t paged_of(const PagedAttentionArgs& p, bool vec, hipStream_t s) {
	if (!vec) return launch_paged<T, 128, false>(p, s);
	if (p.a.dh <= 64) return launch_paged<T, 64, true>(p, s);
	if (p.a.dh <= 96) return launch_paged<T, 96, true>(p, s);
	return launch_paged<T, 128, true>(p, s);
}

}  // namespace attn
}  // namespace nnh
