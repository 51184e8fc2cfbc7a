// paged_attention_fwd.hpp - the kernels of attention over pages, instantiated per element type by paged_attention_*.hip.
//
// The products and the softmax are masked attention's (take_keys in masked_attention_fwd.hpp): scores transposed, a lane holds
// one column's statistics, probabilities enter the second product from the registers they were made in. What differs is where
// columns and tiles come from. The columns are a sequence's rows times the query heads of one key head, head by head within a
// row, so that all heads of a key head read its tiles once and a causal workgroup of 128 columns spans few positions. A tile's
// rows lie in pages: lane l holds the place of the tile's row l, worked out from the page numbers of that tile, which were
// loaded into LDS a tile (split form: a ring of tiles) earlier, so that no load waits for another one's address. Pages may end
// anywhere in a tile. In bf16 a probability is rounded once, to the operand of its product with v (the matrix units take both in one type; sums
// and statistics stay in fp32): a result over 4096 keys alike is off by 0.0023 of its norm, 0.0017 of which is its own rounding.
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

// Keys that the rows of a sequence from position `first` to `last` may see: tiles of 2^shift keys, numbered in one go over those of
// the prefix and those of the causal or window range.
struct Tiles {
	int prefix, skip, count;  // tiles of the prefix; tiles left out behind them; tiles in all
	__device__ __forceinline__ Tiles(const MaskedAttentionArgs& a, int n, int64_t first, int64_t last, int live, int shift) {
		int lo = 0, hi = live;
		const int pre = a.prefix ? clamped(a.prefix[n], 0, live) : 0, up = (1 << shift) - 1;
		if (a.causal) hi = clamped(last + 1, 0, live);
		if (a.window) {
			lo = clamped(first - a.window + 1, 0, live);
			hi = min(hi, clamped(last + a.window, 0, live));
		}
		prefix = (pre + up) >> shift;
		const int from = max(lo >> shift, prefix), to = max((hi + up) >> shift, from);
		skip = from - prefix;
		count = prefix + to - from;
	}
	__device__ __forceinline__ int at(int t) const { return t < prefix ? t : t + skip; }
};

// How the sequences that a form takes are divided: a sequence's columns in groups (of 2^width), the keys that its rows see in parts of
// `chunk` tiles, as many as bring about `target` pairs of the two together over all sequences, whatever their lengths. A grid of
// a few more workgroups than there are pairs has them in order; a workgroup finds its own, a wave looking at 64 sequences at a time.
struct Share {
	int groups, tiles;
	Sequence s;
};
__device__ __forceinline__ Share share_of(const PagedAttentionArgs& p, const Form& f, int n) {
	const Sequence s = sequence_of(p.s, p.t, n);
	const int count = min(s.count, p.most), columns = count * p.a.G;
	if (columns == 0 || (columns > p.few) != f.wide) return {0, 0, s};
	return {(columns + (1 << f.width) - 1) >> f.width, Tiles(p.a, n, s.pos0, (int64_t)s.pos0 + count - 1, s.live, f.shift).count, s};
}
__device__ __forceinline__ int parts_of(const Share& x, int chunk) { return max(1, (int)(((int64_t)x.tiles + chunk / 2) / chunk)); }
__device__ __forceinline__ int chunk_of(const PagedAttentionArgs& p, const Form& f) {
	if (f.target == 0) return 1 << 30;
	int64_t work = 0;
	for (int n = threadIdx.x & 63; n < p.s.N; n += 64) {
		const Share x = share_of(p, f, n);
		work += (int64_t)x.groups * x.tiles;
	}
#pragma unroll
	for (int d = 32; d; d >>= 1) work += __shfl_xor(work, d);
	const int64_t target = f.target * (int64_t)rounds_of(work, f.target);
	return max(kLeastKeys >> f.shift, (int)((work + target - 1) / target));
}
// Pair `index` of a group and a part, or sequence `of`'s first one; n < 0: there are not so many.
struct Turn {
	int n, group, part, parts;
	int64_t first;
	Sequence s;
};
__device__ __forceinline__ Turn turn_of(const PagedAttentionArgs& p, const Form& f, int index, int of) {
	const int lane = threadIdx.x & 63, chunk = chunk_of(p, f);
	int64_t ahead = 0;
	for (int n0 = 0; n0 < p.s.N; n0 += 64) {
		const int n = n0 + lane;
		const Share x = n < p.s.N ? share_of(p, f, n) : Share{0, 0, {0, 0, 0, 0}};
		const int parts = parts_of(x, chunk);
		const int64_t own = (int64_t)x.groups * parts;
		int64_t up = own;
#pragma unroll
		for (int d = 1; d < 64; d *= 2) {
			const int64_t o = __shfl_up(up, d);
			if (lane >= d) up += o;
		}
		const int64_t first = ahead + up - own;
		const uint64_t hit = __ballot(of >= 0 ? n == of : index >= first && index < first + own);
		if (hit) {
			const int at = __builtin_ctzll(hit);
			Turn t;
			t.n = n0 + at;
			t.first = __shfl(first, at);
			t.parts = __builtin_amdgcn_readfirstlane(__shfl(parts, at));
			const int in = __builtin_amdgcn_readfirstlane((int)(index - t.first));  // (sequence `of`'s: not used)
			t.group = in / t.parts;
			t.part = in % t.parts;
			const auto own_of = [&](int v) { return __builtin_amdgcn_readfirstlane(__shfl(v, at)); };
			t.s = {own_of(x.s.first), own_of(x.s.count), own_of(x.s.pos0), own_of(x.s.live)};
			return t;
		}
		ahead += __shfl(up, 63);
	}
	return {-1, 0, 0, 1, 0, {0, 0, 0, 0}};
}
// Where a column of a pair leaves its maximum, sum and dh sums.
__device__ __forceinline__ float* partial_of(const PagedAttentionArgs& p, const Form& f, int hk, int index, int column) {
	return f.partial + (((int64_t)hk * f.pairs + index) * f.room + column) * (p.a.dh + 2);
}

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

// A workgroup's 128 columns of one sequence and key head against a part of the keys they see (mostly all); the tiles are read by all
// four waves. Values that are not finite in masked places: as in masked_attention_forward_kernel.
// Bound by the vector operations beside the products: 4096 tokens over 16384, 32 on 8 heads of 128, in bf16: 1040 us, 925 TFLOP/s.
template <typename T, int DH, bool VEC>
__global__ __launch_bounds__(256, (row_bytes<T, DH>() >= 512 ? 1 : 2)) void paged_attention_kernel(PagedAttentionArgs p) {
	constexpr int KT = keys_per_tile<T, DH>(), RB = row_bytes<T, DH>(), kTile = KT * RB;
	__shared__ __attribute__((aligned(1024))) char lds[4 * kTile + 2 * 256 + 2 * kWaves * 256 + kWaves * 4];
	char* const pages = lds + 4 * kTile;  // page numbers of two tiles
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	int* const marks = (int*)(pages + 2 * 256 + wave * 2 * 256);  // the wave's own, of two tiles
	const int col = lane & 31, half = lane >> 5;
	// (workgroups of one key head side by side on one XCD, where the heads are eight or divide by it: its L2 then holds the keys)
	const int hk = blockIdx.x % p.a.Hkv, index = blockIdx.x / p.a.Hkv;
	const Turn turn = turn_of(p, p.wide, index, -1);
	const int n = turn.n;
	if (n < 0) return;
	const Sequence s = turn.s;
	MaskedAttentionArgs a = p.a;
	a.Tq = min(s.count, p.most);
	// the columns that see most come first
	const int columns = a.Tq * a.G, c0 = ((columns - 1) / kQueries - turn.group) * kQueries, c = c0 + wave * 32 + col;
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
	const Tiles seen(a, n, (int64_t)s.pos0 + c0 / a.G, (int64_t)s.pos0 + (min(c0 + kQueries, columns) - 1) / a.G, s.live, KT == 64 ? 6 : 5);
	const int begin = (int)((int64_t)seen.count * turn.part / turn.parts), end = (int)((int64_t)seen.count * (turn.part + 1) / turn.parts);
	// the page numbers of the first two tiles, on their way beside q
	const auto first_numbers = [&] {
		if (wave != 0 || begin >= end) return;
		load_pages<KT>(p.t, n, seen.at(begin), s.live, lane, pages);
		if (begin + 1 < end) load_pages<KT>(p.t, n, seen.at(begin + 1), s.live, lane, pages + 256);
	};
	first_numbers();
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
			if (decltype(safe)::value) first_numbers();
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
	if (turn.parts == 1) {
		T* o = (T*)a.out + row * a.os.row + h * a.os.head;
		store_column<T, DH, VEC>(o, (T*)nullptr, r.o, l == 0.0f ? 0.0f : 1.0f / l, a.dh, half);
		if (half == 0) p.lse[row * a.H + h] = l == 0.0f ? -kInf : r.m * kLn2 + logf(l);
	} else {
		float* const to = partial_of(p, p.wide, hk, index, c - c0);
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
// Two waves and few tiles on their way, so that four workgroups share a CU (two where a row is 512 bytes or more) and some stream while
// others begin or end: a workgroup's bounds, page numbers and first tiles are trips to memory one after another, 6 us of its time.
// Four waves where all pairs run at once and are short, eight where a CU has one alone (one token over 500 keys, 8 key heads of 128 in bf16:
// 13 us, four 16; of 300 keys 12.6 and 13.4).
// Bound by memory: a token of each of 64 sequences of up to 8192, 32 on 8 heads of 128, in bf16: 268 us, 4.9 TB/s.
template <typename T, int DH, int NW_>
struct PagedSplitShape {
	static constexpr int KT = 32, RB = row_bytes<T, DH>(), kTile = KT * RB, kStage = 2 * kTile;
	static constexpr int NW = NW_;
	static constexpr int ST = RB <= 128 ? 2 : 1;
	static constexpr int kLoads = 2 * kTile / 1024;  // a wave's load instructions for a stage
	static constexpr int kMerge = NW * 32 * (DH + 4) * 4;
	static constexpr int kLds = NW * ST * kStage > kMerge ? NW * ST * kStage : kMerge;
	static constexpr int kPages = 2 * ST * 256, kMarks = ST * 128;  // of a wave
	static constexpr int kAll = kLds + NW * (kPages + kMarks) + NW * 4;
	static_assert(kAll <= (RB >= 512 ? 40 : 20) * NW * 1024 && (ST - 1) * (kLoads + 1) <= 63, "LDS of two workgroups a CU, and loads that a wave may have outstanding");
};

template <typename T, int DH, bool VEC, int NW>
__global__ __launch_bounds__(64 * NW, (row_bytes<T, DH>() >= 512 ? 1 : 2)) void paged_attention_split_kernel(PagedAttentionArgs p) {
	using S = PagedSplitShape<T, DH, NW>;
	constexpr int KT = S::KT, ST = S::ST;
	__shared__ __attribute__((aligned(1024))) char lds[S::kAll];
	const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int col = lane & 31, half = lane >> 5;
	const int hk = blockIdx.x % p.a.Hkv, index = blockIdx.x / p.a.Hkv;
	const Turn turn = turn_of(p, p.split, index, -1);
	const int n = turn.n;
	if (n < 0) return;
	const Sequence s = turn.s;
	MaskedAttentionArgs a = p.a;
	a.Tq = min(s.count, p.most);
	const int columns = a.Tq * a.G, c = turn.group * 32 + col;
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
	// the part's keys, divided over the waves in whole tiles
	const Tiles seen(a, n, s.pos0, (int64_t)s.pos0 + a.Tq - 1, s.live, 5);
	const int begin = (int)((int64_t)seen.count * (turn.part * NW + wave) / (turn.parts * NW)), end = (int)((int64_t)seen.count * (turn.part * NW + wave + 1) / (turn.parts * NW));
	char* const ring = lds + wave * ST * S::kStage;
	char* const pages = lds + S::kLds + wave * S::kPages;
	int* const marks = (int*)(lds + S::kLds + NW * S::kPages + wave * S::kMarks);
	// (numbers past the run's end are some tile's of the sequence: loaded for the count of loads alone)
	const auto numbers = [&](int t) { load_pages<KT>(p.t, n, seen.at(min(t, seen.count - 1)), s.live, lane, pages + t % (2 * ST) * 256); };
	// those of the first tiles, on their way beside q
	const auto first_numbers = [&] {
		if (begin < end)
			for (int x = 0; x < ST; ++x) numbers(begin + x);
	};
	first_numbers();
	arrived(r.q);
	arrived();

	auto run = [&](auto safe) {
		r.clear();
		unsigned bad = 0;  // bit: the stage's tile has rows without a page
		auto load = [&](int t, int stage) {
			const Places64 x = places_of<KT>(p.t, seen.at(t), s.live, lane, pages + t % (2 * ST) * 256);
			bad = (bad & ~(1u << stage)) | (mark_bad<KT>(x, marks + stage * KT, lane) ? 1u << stage : 0u);
			char* to = ring + stage * S::kStage;
			load_rows<T, DH, KT, 1, VEC>(to, to + S::kTile, kbase, vbase, x.at, a.dh, 0, lane);
		};
		if (decltype(safe)::value) first_numbers();
		wait_loads();
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
	for (int x = wave; x < 32 && turn.group * 32 + x < columns; x += NW) {
		const int cc = turn.group * 32 + x, ii = cc / a.G, hh = hk * a.G + cc % a.G;
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
		float* const to = partial_of(p, p.split, hk, index, x);
		T* const o = (T*)a.out + row * a.os.row + hh * a.os.head;
		const float inv = l == 0.0f ? 0.0f : 1.0f / l;
		for (int d = lane; d < a.dh; d += 64) {
			float y = 0.0f;
#pragma unroll
			for (int w = 0; w < NW; ++w) y += f[w] * part[(w * 32 + x) * (DH + 4) + d];
			if (turn.parts == 1) o[d] = (T)(y * inv);
			else to[2 + d] = y;
		}
		if (lane == 0) {
			if (turn.parts == 1) {
				p.lse[row * a.H + hh] = l == 0.0f ? -kInf : m * kLn2 + logf(l);
			} else {
				to[0] = m;
				to[1] = l;
			}
		}
	}
}

// Joins the parts in their order, a wave to `per` heads of a row. Bound by latency: bounds, shares, maxima and sums one after another
// (64 rows of 32 heads 8 us, 1052 of 12 13).
template <typename T>
__global__ __launch_bounds__(256) void paged_attention_join_kernel(PagedAttentionArgs p, int per) {
	const int lane = threadIdx.x & 63;
	const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
	const int shares = (p.a.H + per - 1) / per, row = (int)(at / shares), h0 = (int)(at % shares) * per;
	if (row >= p.s.rows) return;
	const int lo = sequence_with(p.s, row, lane);
	if (lo == p.s.N) return;
	const Sequence s = sequence_of(p.s, p.t, lo);
	const int count = min(s.count, p.most);
	if (row < s.first || row >= s.first + count) return;
	const Form& form = count * p.a.G > p.few ? p.wide : p.split;
	const Turn turn = turn_of(p, form, 0, lo);
	const int splits = turn.parts;
	if (splits == 1) return;
	const int groups = (count * p.a.G + (1 << form.width) - 1) >> form.width;
	for (int h = h0; h < min(h0 + per, p.a.H); ++h) {
		const int hk = h / p.a.G, column = (row - s.first) * p.a.G + h % p.a.G;
		const int group = form.wide ? groups - 1 - (column >> form.width) : column >> form.width;
		if (turn.first + (int64_t)groups * splits > form.pairs) continue;  // (bounds of rows that overlap: more pairs than there is room for)
		const int64_t step = (int64_t)(p.a.dh + 2) * form.room;
		const float* const from = partial_of(p, form, hk, (int)turn.first + group * splits, column & ((1 << form.width) - 1));
		float m = -kInf;
		for (int x = lane; x < splits; x += 64) m = fmaxf(m, from[x * step]);
		for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
		const float base = m == -kInf ? 0.0f : m;
		// each lane a part's factor, then all parts' sums in their order, several loads on their way
		float l = 0.0f, y[2] = {0.0f, 0.0f};
		for (int x0 = 0; x0 < splits; x0 += 64) {
			const bool on = x0 + lane < splits;
			const float mine = on ? exp2_of(from[(x0 + lane) * step] - base) : 0.0f, own = on ? mine * from[(x0 + lane) * step + 1] : 0.0f;
			const int some = min(64, splits - x0);
			const auto add = [&](int x, float a, float b) {
				const float f = __shfl(mine, x);
				l += __shfl(own, x);
				y[0] += f * a;
				y[1] += f * b;
			};
			const float* const at = from + x0 * step + 2;
			const int d0 = min(lane, p.a.dh - 1), d1 = min(lane + 64, p.a.dh - 1);
			for (int x = 0; x < some; x += 8) {
				float a[8], b[8];
#pragma unroll
				for (int i = 0; i < 8; ++i) {  // (past the last part: that one's again, not added)
					a[i] = at[min(x + i, some - 1) * step + d0];
					b[i] = at[min(x + i, some - 1) * step + d1];
				}
#pragma unroll
				for (int i = 0; i < 8; ++i)
					if (x + i < some) add(x + i, a[i], b[i]);
			}
		}
		T* const o = (T*)p.a.out + row * p.a.os.row + h * p.a.os.head;
		const float inv = l == 0.0f ? 0.0f : 1.0f / l;
	#pragma unroll
		for (int d = 0; d < 2; ++d)
			if (lane + 64 * d < p.a.dh) o[lane + 64 * d] = (T)(y[d] * inv);
		if (lane == 0) p.lse[(int64_t)row * p.a.H + h] = l == 0.0f ? -kInf : m * kLn2 + logf(l);
	}
}

template <typename T, int DH, bool VEC>
hipError_t launch_paged(const PagedAttentionArgs& given, hipStream_t s) {
	PagedAttentionArgs p = given;
	p.wide.shift = keys_per_tile<T, DH>() == 64 ? 6 : 5;
	hipError_t e = hipSuccess;
	if (p.wide.pairs) {
		paged_attention_kernel<T, DH, VEC><<<(unsigned)((int64_t)p.wide.pairs * p.a.Hkv), 256, 0, s>>>(p);
		e = hipGetLastError();
	}
	if (e == hipSuccess && p.split.pairs) {
		const int64_t blocks = (int64_t)p.split.pairs * p.a.Hkv;
		constexpr int kMost = row_bytes<T, DH>() <= 256 ? 8 : 4;  // waves that fit a CU's LDS
		if (!p.split.target && blocks <= 256) paged_attention_split_kernel<T, DH, VEC, kMost><<<(unsigned)blocks, 64 * kMost, 0, s>>>(p);
		else if (!p.split.target && blocks <= 1024) paged_attention_split_kernel<T, DH, VEC, 4><<<(unsigned)blocks, 256, 0, s>>>(p);
		else paged_attention_split_kernel<T, DH, VEC, 2><<<(unsigned)blocks, 128, 0, s>>>(p);
		e = hipGetLastError();
	}
	if (e == hipSuccess && (p.wide.target || p.split.target)) {
		// what the heads of a row share takes a wave as long as a head does: several heads to a wave where that still makes 4096 of them
		const int per = (int)std::max<int64_t>(1, std::min<int64_t>(p.a.H, (int64_t)p.s.rows * p.a.H / 4096));
		const int64_t waves = (int64_t)p.s.rows * ((p.a.H + per - 1) / per);
		paged_attention_join_kernel<T><<<(unsigned)((waves + 3) / 4), 256, 0, s>>>(p, per);
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
