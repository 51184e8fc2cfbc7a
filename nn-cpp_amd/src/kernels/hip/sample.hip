// sample.hip - the choice of a token from a row of logits under temperature, min-p, top-k and top-p (sample.hpp).
//
// With the row's logits in descending order (equal ones by their index), w = exp((z - max) / temperature) and prefix sums W of w, each
// filter keeps a prefix: min-p those with w >= min_p; top-k the first k; top-p the shortest whose sum reaches top_p of what the other
// two left. The token is the first of the kept prefix whose sum passes u of the prefix's. So every step asks one question: which
// element has before < X <= before + own, with `before` the sum (or the number) of the elements ahead of it; nothing is sorted.
//
// Weights are whole numbers: w 2^bits rounded to the nearest, bits 45 for a vocabulary of 128000. Their sums are exact, so they do
// not depend on an order, and the products with u and top_p are taken exactly too (128 bits): what is off is each w alone, by half of
// 2^-bits and the exponential's 2^-49 beside the largest weight of 1, and a choice differs from that of exact weights only where a sum is nearer
// to its border than these add up to.
//
// One pass over a row finds the maximum, one sums weights (with top-k: counts) by bins of a share of a factor of two, in the order wanted:
// a window of 32 factors of two, in which the element nearly always is, the rest in registers. Then the element asked for is in a known
// bin, whose elements go into a list in LDS and are ordered by comparing each with each. With top-k the list takes all elements up to
// the k-th where they are few, and the later questions are answered there. A bin with more than the list holds is divided further by the
// order's own key (32 bits of the logit, then the index).
//
// A vocabulary of up to 8192 is a workgroup's alone, in one launch. Of larger ones a workgroup would read 10 bytes a cycle, so the two passes
// have launches of their own, several workgroups to a row (Slices), which also note the elements within 10 factors of two of the largest: a
// third launch, a workgroup to a row, answers from the bins and the notes, and reads the row again where the element lies deeper or the notes
// are more than it holds (13 us a question, 256 rows of 128000 in bf16; without notes every question cost that).
// The exponential: 2^-d = 2^-n 2^-(k/1024) 2^-r from a table of 1024 and the power series to r^3 (|r| ln 2 <= 3.4e-4: off by 2^-50.7 of it).
// With the roundings of the table (2^-52), the series and the product (2^-53 each) and of d (four of 2^-53, as much of d e^-d, 0.37 at most)
// it is off by 2^-49.6 of the largest weight: more than half of 2^-bits for vocabularies of up to 8192.
//
// The second pass is bound by vector instructions (fp32: about 25 an element, most of them in 64 bits, at the rate of 32; 16-bit values are
// counted instead, and weighed once each), the third launch by latency (13 to 17 us: loads, scan, list and order one after another).
// Measured: 1 x 50257 3 + 6 + 13 us, 64 x 32000 5.5 + 12 + 14.5, 256 x 128000 in bf16 (with top-p and min-p) 13.5 + 34 + 46.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "sample.hpp"

namespace nnh {

namespace {

typedef unsigned long long u64;

constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.6931471805599453094;
constexpr int kFine = 1 << 10;       // steps to a factor of two, entries of the table
// Steps that the bins cover. (256 rows of 128000 in bf16, logits of standard deviation 3 drawn from whole: 83 us, with half of it 142, as one
// row of a hundred goes past it; deviation 0.75: 123 and 93, as a bin is then more than the list holds.)
constexpr int kWindow = 32 * kFine;
// (large vocabularies: see Slices)
constexpr int kSliceThreads = 512, kSliceBins = 2048, kSliceWaves = kSliceThreads / 64;
constexpr int64_t kSliceRows = 512;  // rows at a time
constexpr int kList = 512;           // elements whose order is found by comparing them
constexpr int kNear = 10 * kFine;    // steps from the largest weight within which the first pass notes where elements are
constexpr int kNearRow = 4096, kNearWave = 512;  // as many of a row, of a wave's share of it

typedef unsigned Word __attribute__((ext_vector_type(4)));
template <typename X>
using Global = __attribute__((address_space(1))) X*;
__device__ const Word kNothing = {0, 0, 0, 0};
// Pointers into LDS as such, for functions that are called: the passes over a row are, so that each has the registers to itself (a
// kernel of all of them kept a hundred scalars in vector registers and fetched them back for every word).
template <typename X>
using Lds = __attribute__((address_space(3))) X*;
template <typename X>
__device__ __forceinline__ Lds<X> lds_of(X* p) {
	return (Lds<X>)p;
}
template <typename X>
__device__ __forceinline__ X add_to(Lds<X> p, X x) {
	return __hip_atomic_fetch_add(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

struct alignas(16) Item {
	u64 key, mass;
};

struct Found {
	u64 key, before, mass;  // of the element: its place in the order, the sum ahead of it, its own
};

template <int NT, int BINS, int NEAR>
struct Shared {
	u64 near[NEAR];      // keys of the elements within kNear steps
	u64 sum[BINS + 1];   // what is ahead of each bin (weights or numbers); the last entry: all
	u64 part[BINS + 1];  // the same of a bin that is divided further
	Item list[kList];
	u64 before[kList];
	unsigned rank[kList];
	double table[kFine];
	u64 wave_sum[NT / 64];
	float wave_top[NT / 64];
	u64 low, high, tail;
	unsigned listed;
	int bin;
	Found found;
};

// Descending order as ascending whole numbers (both zeros are one logit).
__device__ __forceinline__ unsigned order_of(float z) {
	const unsigned b = __float_as_uint(z + 0.0f);
	return b >> 31 ? b : 0x7fffffffu - b;
}
__device__ __forceinline__ float logit_of(unsigned o) { return __uint_as_float(o >> 31 ? o : 0x7fffffffu - o); }
__device__ __forceinline__ u64 key_of(float z, int i) { return (u64)order_of(z) << 32 | (unsigned)i; }

// floor(f x) or ceil(f x) for f < 1 (0 below 0).
__device__ __forceinline__ u64 part_of(float f, u64 x, bool up) {
	if (!(f > 0.0f)) return 0;
	const unsigned b = __float_as_uint(f), e = b >> 23;
	const unsigned m = e ? (b & 0x7fffffu) | 0x800000u : b & 0x7fffffu;
	const int shift = 150 - (int)(e ? e : 1);  // f = m 2^-shift, shift at least 24
	const unsigned __int128 y = (unsigned __int128)m * x;  // below 2^87
	if (shift >= 100) return up && y != 0 ? 1 : 0;
	const u64 q = (u64)(y >> shift);
	return q + (up && (y & (((unsigned __int128)1 << shift) - 1)) != 0 ? 1 : 0);
}

// Words first .. last - 1 (of 16 bytes, at multiples of that in memory) of a row, taken by the workgroup's threads in turn. The row's
// first and last word may be shared with others: these two are loaded by their own elements.
template <typename T, int NT>
struct Row {
	static constexpr int E = 16 / (int)sizeof(T);
	typedef std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t> Raw;  // an element's bits
	Global<const Raw> z;  // element 0 of word 0, which may lie before the row
	Global<const Word> whole;  // word 0, where the row has words of its own (`own` .. `behind` - 1); else a word of zeros
	int begin, end;       // the row's elements
	int own, behind;
	int first, last;

	__device__ __forceinline__ Row(const T* row, int V) {
		begin = (int)(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
		end = begin + V;
		z = (Global<const Raw>)(row - begin);
		own = begin ? 1 : 0;
		behind = end / E;
		whole = own < behind ? (Global<const Word>)z : (Global<const Word>)&kNothing;
		first = 0;
		last = (end + E - 1) / E;
	}
	__device__ __forceinline__ static float element(const Word& u, int i) {
		if constexpr (sizeof(T) == 2) return __uint_as_float(i & 1 ? u[i / 2] & 0xffff0000u : u[i / 2] << 16);
		else return __uint_as_float(u[i]);
	}
	// Element i, a lane's own choice.
	__device__ __forceinline__ static float pick(const Word& u, int i) {
		const int j = sizeof(T) == 2 ? i >> 1 : i;
		const unsigned low = j & 1 ? u[1] : u[0], high = j & 1 ? u[3] : u[2], x = j & 2 ? high : low;
		if constexpr (sizeof(T) == 2) return __uint_as_float(i & 1 ? x & 0xffff0000u : x << 16);
		else return __uint_as_float(x);
	}
	// A word by its elements; those beside the row are -infinity.
	__device__ __forceinline__ Word pieces(int w) const {
		Word u = {0, 0, 0, 0};
#pragma unroll
		for (int i = 0; i < E; ++i) {
			const int at = w * E + i;
			const unsigned raw = z[min(max(at, begin), end - 1)];
			const unsigned x = at >= begin && at < end ? raw : sizeof(T) == 2 ? 0xff80u : 0xff800000u;
			if constexpr (sizeof(T) == 2) u[i / 2] |= x << 16 * (i & 1);
			else u[i] = x;
		}
		return u;
	}
	// f(word, index of its first element), a thread's next P words on their way meanwhile.
	template <int P, typename F>
	__device__ __forceinline__ void words(F f) const {
		const int mine = first + (int)threadIdx.x;
		if (mine >= last) return;
		const int most = max(behind - 1, 0);
		Word head, tail, next[P];
		if (mine < own) head = pieces(0);
		if (behind < last) tail = pieces(last - 1);
		const auto load = [&](int w) -> Word { return whole[min(max(w, own), most)]; };
#pragma unroll
		for (int x = 0; x < P; ++x) next[x] = load(mine + x * NT);
#pragma clang loop unroll(disable)
		for (int w0 = mine; w0 < last; w0 += P * NT) {
#pragma unroll
			for (int x = 0; x < P; ++x) {
				const int w = w0 + x * NT;
				Word u = next[x];
				next[x] = load(w + P * NT);
				if (w >= last) break;
				if (w < own) u = head;
				else if (w >= behind) u = tail;
				f(u, w * E - begin);
			}
		}
	}
	__device__ __forceinline__ static float largest(const Word& u) {
		float m = element(u, 0);
#pragma unroll
		for (int i = 1; i < E; ++i) m = fmaxf(m, element(u, i));
		return m;
	}
	// Whether no element lies in low .. high; now and then it says no wrongly. Numbers above zero are in the order of their bits.
	__device__ __forceinline__ static bool none(const Word& u, float low, float high) {
		if (!(low > 0.0f)) return !(largest(u) >= low);
		const unsigned lo = __float_as_uint(low), hi = __float_as_uint(high);
		if constexpr (sizeof(T) == 2) {
			typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
			const u16x2 from = {(unsigned short)(lo >> 16), (unsigned short)(lo >> 16)};
			u16x2 m[4];
#pragma unroll
			for (int i = 0; i < 4; ++i) m[i] = __builtin_bit_cast(u16x2, (unsigned)u[i]) - from;
			const u16x2 near = __builtin_elementwise_min(__builtin_elementwise_min(m[0], m[1]), __builtin_elementwise_min(m[2], m[3]));
			return min((unsigned)near[0], (unsigned)near[1]) > (hi >> 16) - (lo >> 16);
		} else {
			return min(min(u[0] - lo, u[1] - lo), min(u[2] - lo, u[3] - lo)) > hi - lo;
		}
	}
	// f(z, index) of every element with low <= z <= high, infinities as the largest number; a lane's own, one after another.
	template <typename F>
	__device__ __forceinline__ void each(float low, float high, F f) const {
		words<4>([&](const Word& u, int at) {
			if (none(u, low, high)) return;
			unsigned on = 0;
#pragma unroll
			for (int i = 0; i < E; ++i) on |= element(u, i) >= low && element(u, i) <= high ? 1u << i : 0u;
			while (on) {
				const int i = __builtin_ctz(on);
				on &= on - 1;
				f(fminf(pick(u, i), FLT_MAX), at + i);
			}
		});
	}
};

// The same of the elements that the first pass has noted, by their keys in LDS.
template <int NT>
struct Noted {
	Lds<const u64> keys;
	int count;
	template <typename F>
	__device__ __forceinline__ void each(float low, float high, F f) const {
#pragma clang loop unroll(disable)
		for (int i = threadIdx.x; i < count; i += NT) {
			const u64 key = keys[i];
			const float z = logit_of((unsigned)(key >> 32));
			if (z >= low && z <= high) f(z, (int)(unsigned)key);
		}
	}
};

// A row's weights by the distance from the largest logit, in steps of 1 / kFine of a factor of two; a distance's whole part is found
// beside 3 2^51, where the sum's last place is 1 and its low word the number.
struct Weights {
	double top, c;
	double least;  // weights that are smaller are not kept (beside 2^52, as `beside` gives them)
	float bottom;  // and logits that are smaller have none
	Lds<const double> table;  // 2^(bits + i / kFine)
	__device__ __forceinline__ double steps(float z) const { return fmin((top - (double)z) * c, 64.0 * kFine); }
	// -round(steps) beside 3 2^51, and as a number.
	__device__ __forceinline__ static double whole(double steps) { return 0x1.8p52 - steps; }
	__device__ __forceinline__ static int back(double whole) { return (int)(unsigned)__double_as_longlong(whole); }
	// The weight 2^bits 2^(-steps / kFine), rounded to a whole number, beside 2^52: the sum's last place is 1, and its low bits the number.
	__device__ __forceinline__ double beside(double steps, double whole) const {
		constexpr double c = -kLn2 / kFine;
		const int k = back(whole);
		const double r = (whole - 0x1.8p52) + steps;
		double p = __builtin_fma(r, c * c * c / 6.0, c * c / 2.0);
		p = __builtin_fma(r, p, c);
		p = __builtin_fma(r, p, 1.0);
		return __builtin_ldexp(p * table[k & (kFine - 1)], k >> 10) + 0x1p52;
	}
	__device__ __forceinline__ static u64 number(double beside) { return (u64)__double_as_longlong(beside) & 0xfffffffffffffull; }
	// A logit that lies so far from the largest, moved by more than any rounding here.
	__device__ __forceinline__ float at(double steps, double way) const {
		const double z = top - steps / c, room = fabs(z) * 0x1p-22 + fabs(top) * 0x1p-22 + 0x1p-140;
		return (float)fmin(fmax(z + way * room, -(double)FLT_MAX), (double)FLT_MAX);
	}
};

// What is ahead of each bin, in place.
template <int NT, int BINS, int NEAR>
__device__ void scan_bins(Shared<NT, BINS, NEAR>& s, u64* sum) {
	constexpr int per = BINS / NT, NW = NT / 64;
	static_assert(per >= 1 && per * NT == BINS, "bins to a thread");
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	u64 m[per], all = 0;
#pragma unroll
	for (int i = 0; i < per; ++i) {
		m[i] = sum[threadIdx.x * per + i];
		all += m[i];
	}
	u64 up = all;
#pragma unroll
	for (int d = 1; d < 64; d *= 2) {
		const u64 o = __shfl_up(up, d);
		if (lane >= d) up += o;
	}
	if (lane == 63) s.wave_sum[wave] = up;
	__syncthreads();
	u64 ahead = lane < NW ? s.wave_sum[lane] : 0;
#pragma unroll
	for (int d = 1; d < NW; d *= 2) {
		const u64 o = __shfl_up(ahead, d);
		if (lane >= d) ahead += o;
	}
	ahead = __shfl(ahead, wave > 0 ? wave - 1 : 0);
	up = up - all + (wave > 0 ? ahead : 0);
#pragma unroll
	for (int i = 0; i < per; ++i) {
		sum[threadIdx.x * per + i] = up;
		up += m[i];
	}
	if (threadIdx.x == NT - 1) sum[BINS] = up;
	__syncthreads();
}

// The bin with ahead < x <= ahead + own.
template <int NT, int BINS, int NEAR>
__device__ int find_bin(Shared<NT, BINS, NEAR>& s, const u64* sum, u64 x) {
	for (int b = threadIdx.x; b < BINS; b += NT)
		if (sum[b] < x && x <= sum[b + 1]) s.bin = b;
	__syncthreads();
	const int b = s.bin;
	__syncthreads();
	return b;
}

// What the list's elements have ahead of them, which starts from the sum and number given.
template <int NT, int BINS, int NEAR>
__device__ void order_list(Shared<NT, BINS, NEAR>& s, u64 mass, unsigned count) {
	const int n = s.listed;
	for (int i = threadIdx.x; i < n; i += NT) {
		s.before[i] = mass;
		s.rank[i] = count;
	}
	__syncthreads();
	// element i by NT / width threads, each with its share of the others
	int width = 64;
	while (width < n) width *= 2;
	const int shares = NT > width ? NT / width : 1, share = threadIdx.x / width % shares, per = (n + shares - 1) / shares;
	for (int i = threadIdx.x % width; i < n; i += min(width, NT)) {
		const u64 key = s.list[i].key;
		u64 m = 0;
		unsigned c = 0;
#pragma unroll 4
		for (int j = share * per; j < min(n, (share + 1) * per); ++j) {
			const Item o = s.list[j];
			m += o.key < key ? o.mass : 0;
			c += o.key < key ? 1 : 0;
		}
		if (m) atomicAdd(&s.before[i], m);
		if (c) atomicAdd(&s.rank[i], c);
	}
	__syncthreads();
}

// What a row is asked for.
struct Asked {
	float temperature;
	int top_k;
	float top_p, min_p, u;
	__device__ __forceinline__ Asked(const SampleArgs& a, int64_t n)
	    : temperature(a.temperature ? a.temperature[n] : 1.0f), top_k(a.top_k ? a.top_k[n] : 0), top_p(a.top_p ? a.top_p[n] : 1.0f), min_p(a.min_p ? a.min_p[n] : 0.0f), u(a.u[n]) {
		if (top_k < 0 || top_k >= a.V) top_k = 0;
	}
	__device__ __forceinline__ bool cut() const { return min_p > 0.0f; }
};

__device__ __forceinline__ Weights weights_of(const SampleArgs& a, const Asked& q, float best, Lds<const double> table) {
	Weights w;
	w.top = fmin((double)best, (double)FLT_MAX);
	w.c = kFine * kLog2e / (double)q.temperature;
	w.table = table;
	const double p = q.cut() ? (double)fminf(q.min_p, 1.0f) : 0.0;
	w.least = 0x1p52 + (q.cut() ? fmax(1.0, ceil(__builtin_ldexp(p, a.bits))) : 1.0);
	// Smaller logits have no weight, or less than min_p's. Beside an infinity, nothing else has one.
	w.bottom = best > FLT_MAX ? best : w.at(kFine * fmin((double)a.bits + 1.0, q.cut() ? 0.001 - log2(p) : 64.0), -1.0);
	return w;
}

template <int NT>
__device__ __forceinline__ void fill_table(double* table, int bits) {
	for (int i = threadIdx.x; i < kFine; i += NT) table[i] = __builtin_ldexp(exp2((double)i * (1.0 / kFine)), bits);
}

// The largest of a thread's elements.
template <class R>
__device__ __forceinline__ float thread_top(const R& row) {
	float best = -__builtin_huge_valf();
	row.template words<4>([&](const Word& u, int) { best = fmaxf(best, R::largest(u)); });
	return best;
}

template <int NT>
__device__ __forceinline__ float all_top(float best, float* wave_top) {
#pragma unroll
	for (int d = 32; d; d >>= 1) best = fmaxf(best, __shfl_xor(best, d));
	if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = best;
	__syncthreads();
#pragma unroll
	for (int w = 0; w < NT / 64; ++w) best = fmaxf(best, wave_top[w]);
	return best;
}

// The first pass, over all there is: a word's elements side by side, each step of the one filling the waits of the others. What is no
// number is further away than any weight (the least of the two is the number), as are those below the least weight.
struct Notes {
	Lds<u64> at;  // the wave's own: keys of its elements within kNear steps
	int count;         // may pass kNearWave; lane 0's, which is the last to leave, counts
	__device__ __forceinline__ void add(bool near, float z, int index) {
		const uint64_t on = __ballot(near);
		if (!on) return;
		const int to = count + __builtin_amdgcn_mbcnt_hi((unsigned)(on >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)on, 0));
		if (near && to < kNearWave) at[to] = key_of(z, index);
		count += __builtin_popcountll(on);
	}
};
template <int kBin, bool NUMBER, bool CUT, bool NOTE, class R>
__device__ __forceinline__ double add_first(const R& row, const Weights& w, Lds<u64> sum, Notes& notes) {
	double tail = 0.0;
	row.template words<2>([&](const Word& u, int at) {
		int k[R::E];
		double y[R::E];
#pragma unroll
		for (int i = 0; i < R::E; ++i) {
			const double d = w.steps(R::element(u, i)), whole = Weights::whole(d);
			k[i] = -Weights::back(whole);
			if (!NUMBER || CUT) y[i] = w.beside(d, whole);
			if (CUT && y[i] < w.least) {
				k[i] = kWindow;
				y[i] = 0x1p52;
			}
		}
#pragma unroll
		for (int i = 0; i < R::E; ++i) {
			if (k[i] < kWindow) add_to(sum + (unsigned)k[i] / kBin, NUMBER ? (u64)1 : Weights::number(y[i]));
			else if (!NUMBER) tail += y[i] - 0x1p52;
			if constexpr (NOTE) notes.add(k[i] < kNear, R::element(u, i), at + i);
		}
	});
	return tail;
}
template <int kBin, bool NOTE, class R>
__device__ __forceinline__ double add_first(const R& row, const Weights& w, bool cut, bool number, Lds<u64> sum, Notes& notes) {
	if (number) return cut ? add_first<kBin, true, true, NOTE>(row, w, sum, notes) : add_first<kBin, true, false, NOTE>(row, w, sum, notes);
	return cut ? add_first<kBin, false, true, NOTE>(row, w, sum, notes) : add_first<kBin, false, false, NOTE>(row, w, sum, notes);
}

// The same over 16-bit logits, where a vocabulary's thousands share some hundreds of values: each value is counted (one addition in LDS an
// element, in the place of its weight's two dozen instructions), and weighed once at the end. Counted are magnitudes of 2^-8 to 2^8, others,
// which are rare, are weighed where they are. Notes may have a few elements more than are within kNear steps.
constexpr int kValues = 2 * 16 * 128, kLeastValue = (127 - 8) << 7;
template <int kBin, class R>
__device__ __forceinline__ double count_first(const R& row, const Weights& w, bool cut, bool number, Lds<u64> sum, Lds<unsigned> counts, Notes& notes) {
	double tail = 0.0;
	const float near = w.at(kNear + 1.0, -1.0);
	const auto weigh = [&](float z, u64 count) {
		const double d = w.steps(z), whole = Weights::whole(d), y = w.beside(d, whole);
		const int k = -Weights::back(whole);
		if (cut && y < w.least) return;
		if (k < kWindow) add_to(sum + (unsigned)k / kBin, number ? count : Weights::number(y) * count);
		else if (!number) tail += (y - 0x1p52) * (double)count;
	};
	row.template words<4>([&](const Word& u, int at) {
#pragma unroll
		for (int i = 0; i < R::E; ++i) {
			const unsigned raw = i & 1 ? u[i / 2] >> 16 : u[i / 2] & 0xffffu, place = (raw & 0x7fffu) - kLeastValue;
			const float z = R::element(u, i);
			if (place < kValues / 2) add_to(counts + (place | (raw >> 15) * (kValues / 2)), 1u);
			else if (z >= w.bottom) weigh(z, 1);
			notes.add(z >= near, z, at + i);
		}
	});
	__syncthreads();
	for (int i = threadIdx.x; i < kValues; i += kSliceThreads)
		if (counts[i]) weigh(__uint_as_float((unsigned)(i % (kValues / 2) + kLeastValue) << 16 | (unsigned)(i / (kValues / 2)) << 31), counts[i]);
	return tail;
}

// Adds a window's weights (or ones: numbers of elements) of elements up to the key `last` to bins of kBin steps, and returns the sum of
// the first window's weights behind it (of this thread: a whole number below 2^53).
template <int kBin, class R>
__device__ __forceinline__ double add_window(R row, Weights w, bool cut, bool number, int window, u64 last, float lowest, Lds<u64> sum) {
	const int from = window * kWindow;
	double tail = 0.0;
	const float high = window == 0 ? __builtin_huge_valf() : w.at(from - 1.0, 1.0);
	const float low = number || window > 0 ? fmaxf(lowest, w.at(from + kWindow + 1.0, -1.0)) : lowest;
	row.each(low, high, [&](float z, int i) {
		const double d = w.steps(z), whole = Weights::whole(d);
		const int k = -Weights::back(whole) - from;
		if (k < 0) return;
		if (last != ~0ull && key_of(z, i) > last) return;
		double y = 0.0;
		if (!number || cut) {
			y = w.beside(d, whole);
			if (cut && y < w.least) return;
		}
		if (k < kWindow) add_to(sum + (unsigned)k / kBin, number ? (u64)1 : Weights::number(y));
		else if (!number) tail += y - 0x1p52;
	});
	return tail;
}

// What a pass looks for: elements of steps begin .. end - 1 and logits low .. high with a key in from .. to.
struct Range {
	int begin, end;
	float low, high;
	u64 from, to;
};
struct List {
	Lds<Item> items;
	Lds<unsigned> count;  // may pass kList
	Lds<u64> low, high;   // the least and the largest key
};

template <class R>
__device__ __forceinline__ void gather(R row, Weights w, bool cut, Range r, List list) {
	u64 least = ~0ull, most = 0;
	row.each(r.low, r.high, [&](float z, int i) {
		const double d = w.steps(z), whole = Weights::whole(d);
		const int step = -Weights::back(whole);
		const u64 key = key_of(z, i);
		if (step < r.begin || step >= r.end || key < r.from || key > r.to) return;
		const double y = w.beside(d, whole);
		if (cut && y < w.least) return;
		const unsigned at = add_to(list.count, 1u);
		if (at < kList) {
			list.items[at].key = key;
			list.items[at].mass = Weights::number(y);
		}
		least = min(least, key);
		most = max(most, key);
	});
	if (least <= most) {
		__hip_atomic_fetch_min(list.low, least, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
		__hip_atomic_fetch_max(list.high, most, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
	}
}

// Weights (or numbers) of the elements with a key in r.from .. r.to by equal parts of that range.
template <class R>
__device__ __forceinline__ void divide(R row, Weights w, bool cut, bool number, Range r, int shift, Lds<u64> part) {
	row.each(r.low, r.high, [&](float z, int i) {
		const u64 key = key_of(z, i);
		if (key < r.from || key > r.to) return;
		const double d = w.steps(z), y = w.beside(d, Weights::whole(d));
		if (cut && y < w.least) return;
		add_to(part + ((key - r.from) >> shift), number ? (u64)1 : Weights::number(y));
	});
}

__device__ __forceinline__ void add_tail(double tail, u64* to) {
#pragma unroll
	for (int d = 32; d; d >>= 1) tail += __shfl_xor(tail, d);
	if ((threadIdx.x & 63) == 0 && tail > 0.0) atomicAdd(to, (u64)tail);
}

// Large vocabularies: the two passes that see all of a row, the maximum and the first window's bins, are taken by workgroups of their
// own, several to a row where there are few. Whole numbers are added up in memory, and the elements near the largest are noted,
// so that the workgroup that then answers the questions for the row seldom reads it again (one alone reads 10 bytes a cycle).
struct Slices {
	int count;        // to a row; 0: none
	int64_t row0;     // the first row
	float* top;       // {rows, count}
	u64* sum;         // {rows, kSliceBins + 2}: the first window's bins, what lies behind it, and how many elements are noted
	u64* noted;       // {rows, kNearRow}: keys
};

template <typename T>
__device__ __forceinline__ Row<T, kSliceThreads> slice_of(const SampleArgs& a, const Slices& x) {
	Row<T, kSliceThreads> row((const T*)a.logits + (x.row0 + blockIdx.y) * a.ld, a.V);
	const int per = (row.last + x.count - 1) / x.count;
	row.first = min((int)blockIdx.x * per, row.last);
	row.last = min(row.first + per, row.last);
	return row;
}

template <typename T>
__global__ __launch_bounds__(kSliceThreads) void sample_top_kernel(SampleArgs a, Slices x) {
	__shared__ float wave_top[kSliceWaves];
	u64* const sum = x.sum + (int64_t)blockIdx.y * (kSliceBins + 2);
	for (int i = blockIdx.x * kSliceThreads + threadIdx.x; i < kSliceBins + 2; i += x.count * kSliceThreads) sum[i] = 0;
	const float best = all_top<kSliceThreads>(thread_top(slice_of<T>(a, x)), wave_top);
	if (threadIdx.x == 0) x.top[(int64_t)blockIdx.y * x.count + blockIdx.x] = best;
}

// The largest of a row's slices, by each wave for itself.
__device__ __forceinline__ float top_of(const Slices& x, int64_t n) {
	float best = -__builtin_huge_valf();
	for (int i = threadIdx.x & 63; i < x.count; i += 64) best = fmaxf(best, x.top[n * x.count + i]);
#pragma unroll
	for (int d = 32; d; d >>= 1) best = fmaxf(best, __shfl_xor(best, d));
	return best;
}

template <typename T>
__global__ __launch_bounds__(kSliceThreads) void sample_bins_kernel(SampleArgs a, Slices x) {
	__shared__ u64 sum[kSliceBins + 1];
	__shared__ double table[kFine];
	__shared__ u64 notes[kSliceWaves * kNearWave];
	__shared__ unsigned counts[sizeof(T) == 2 ? kValues : 1];
	const int64_t n = blockIdx.y;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const Asked q(a, x.row0 + n);
	const float best = top_of(x, n);
	if (best == -__builtin_huge_valf() || !(q.temperature > 0.0f)) return;
	fill_table<kSliceThreads>(table, a.bits);
	for (int i = threadIdx.x; i <= kSliceBins; i += kSliceThreads) sum[i] = 0;
	if constexpr (sizeof(T) == 2)
		for (int i = threadIdx.x; i < kValues; i += kSliceThreads) counts[i] = 0;
	__syncthreads();
	const Weights w = weights_of(a, q, best, lds_of((const double*)table));
	Notes mine{lds_of(notes + wave * kNearWave), 0};
	constexpr int kBin = kWindow / kSliceBins;
	double tail = 0.0;
	if (w.bottom < FLT_MAX) {
		if constexpr (sizeof(T) == 2) tail = count_first<kBin>(slice_of<T>(a, x), w, q.cut(), q.top_k > 0, lds_of(sum), lds_of(counts), mine);
		else tail = add_first<kBin, true>(slice_of<T>(a, x), w, q.cut(), q.top_k > 0, lds_of(sum), mine);
	} else tail = add_window<kBin>(slice_of<T>(a, x), w, q.cut(), q.top_k > 0, 0, ~0ull, w.bottom, lds_of(sum));
	add_tail(tail, &sum[kSliceBins]);
	__syncthreads();
	u64* const to = x.sum + n * (kSliceBins + 2);
	for (int i = threadIdx.x; i <= kSliceBins; i += kSliceThreads)
		if (sum[i]) atomicAdd(to + i, sum[i]);
	const int count = __shfl(mine.count, 0);
	const bool all = count <= kNearWave && w.bottom < FLT_MAX;
	u64 at = 0;
	if (lane == 0 && (count || !all)) at = atomicAdd(to + kSliceBins + 1, all ? (u64)count : (u64)1 << 32);
	at = __shfl(at, 0);
	if (all)
		for (int i = lane; i < count; i += 64)
			if (at + i < kNearRow) x.noted[n * kNearRow + at + i] = notes[wave * kNearWave + i];
}

template <typename T, int NT, int BINS, bool SLICED>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a, Slices slices) {
	constexpr int kBin = kWindow / BINS;  // steps to a bin
	__shared__ Shared<NT, BINS, SLICED ? kNearRow : 1> s;
	const int64_t n = slices.row0 + blockIdx.x;
	const Row<T, NT> row((const T*)a.logits + n * a.ld, a.V);
	const u64* const sliced = SLICED ? slices.sum + (int64_t)blockIdx.x * (kSliceBins + 2) : nullptr;
	Noted<NT> noted{lds_of((const u64*)s.near), 0};
	bool near = false;  // what is within kNear steps is noted

	const Asked q(a, n);
	float best;
	u64 bins[SLICED ? BINS / NT : 1], tail_sum = 0, count = 0;
	if constexpr (SLICED) {  // (what the slices have left is on its way while the table is made)
		static_assert(BINS == kSliceBins, "the slices' bins");
#pragma unroll
		for (int i = 0; i < BINS / NT; ++i) bins[i] = sliced[i * NT + threadIdx.x];
		tail_sum = sliced[BINS];
		count = sliced[BINS + 1];
	}
	fill_table<NT>(s.table, a.bits);
	if (threadIdx.x == 0) s.low = ~0ull;
	if constexpr (SLICED) {
#pragma unroll
		for (int i = 0; i < BINS / NT; ++i) s.sum[i * NT + threadIdx.x] = bins[i];
		if (threadIdx.x == 0) s.tail = tail_sum;
		best = top_of(slices, blockIdx.x);
		near = count <= kNearRow;
		if (near) {
			noted.count = (int)count;
			for (int i = threadIdx.x; i < noted.count; i += NT) s.near[i] = slices.noted[(int64_t)blockIdx.x * kNearRow + i];
		}
		__syncthreads();
	} else {
		best = all_top<NT>(thread_top(row), s.wave_top);
	}
	if (best == -__builtin_huge_valf()) {  // no logit is a number above -infinity
		if (threadIdx.x == 0) {
			a.tokens[n] = -1;
			if (a.logprob) a.logprob[n] = best;
		}
		return;
	}
	if (!(q.temperature > 0.0f)) {  // the first of the largest
		row.each(best, best, [&](float, int i) { atomicMin(&s.low, (u64)i); });
		__syncthreads();
		if (threadIdx.x == 0) {
			a.tokens[n] = (int)s.low;
			if (a.logprob) a.logprob[n] = 0.0f;
		}
		return;
	}
	const Weights w = weights_of(a, q, best, lds_of((const double*)s.table));
	const bool cut = q.cut();
	u64 last = ~0ull;  // the last element's key that top-k leaves, and its distance
	int last_step = kNear;
	float lowest = w.bottom;

	// The questions in turn: the k-th element, the one that reaches top_p, the one that passes u.
	u64 sum = 0;            // the weights of what is kept
	int window = 0;
	u64 base = 0;           // ahead of the window
	int filled = -1;        // what the bins hold: 1 numbers of elements, 0 sums of weights
	bool complete = false;  // the list has every element from the first to the last that is kept
	Found f{0, 0, 0};
#pragma clang loop unroll(disable)
	for (int question = 0; question < 3; ++question) {
		const bool number = question == 0;
		if (question == 0 && q.top_k == 0) continue;
		if (question == 1 && !(q.top_p < 1.0f)) continue;
		u64 x = 0;
		const auto ask = [&] {
			x = question == 0 ? (u64)q.top_k : question == 1 ? max(1ull, part_of(q.top_p, sum, true)) : q.u < 1.0f ? part_of(q.u, sum, false) + 1 : sum;
		};
		bool found = true;
		if (!complete) {
			bool fill = filled != (number ? 1 : 0);
			if (fill) {
				window = 0;
				base = 0;
			}
#pragma clang loop unroll(disable)
			for (;;) {
				if (fill) {
					// the window's bins, and with the first one the weights behind it
					if (!SLICED || filled >= 0) {  // (else they are there)
						for (int i = threadIdx.x; i < BINS; i += NT) s.sum[i] = 0;
						if (threadIdx.x == 0) s.tail = 0;
						__syncthreads();
						double tail;
						if (!SLICED && filled < 0 && w.bottom < FLT_MAX) {
							Notes none{nullptr, 0};
							tail = add_first<kBin, false>(row, w, cut, number, lds_of(s.sum), none);
						} else if (SLICED && near && last_step < kNear) {
							tail = add_window<kBin>(noted, w, cut, number, window, last, lowest, lds_of(s.sum));
						} else {
							tail = add_window<kBin>(row, w, cut, number, window, last, lowest, lds_of(s.sum));
						}
						add_tail(tail, &s.tail);
					}
					__syncthreads();
					scan_bins(s, s.sum);
					if (!number && filled != 0) sum = s.sum[BINS] + s.tail;
					filled = number ? 1 : 0;
				}
				ask();
				fill = true;
				if (x <= base) {
					window = 0;
					base = 0;
				} else if (x - base > s.sum[BINS]) {
					if (window == 64 * kFine / kWindow - 1) {  // fewer than top_k have a weight (2^-52 is the least)
						found = false;
						break;
					}
					base += s.sum[BINS];
					++window;
				} else {
					break;
				}
				__syncthreads();
			}
			if (!found) continue;
			// its bin's elements into the list: with top-k all up to it, where they are few
			const int b = find_bin(s, s.sum, x - base);
			complete = number && window == 0 && s.sum[b + 1] <= kList / 2;
			u64 ahead = complete ? 0 : base + s.sum[b];
			Range r;
			r.begin = complete ? 0 : window * kWindow + b * kBin;
			r.end = window * kWindow + (b + 1) * kBin;
			r.high = r.begin == 0 ? __builtin_huge_valf() : w.at(r.begin - 1.0, 1.0);
			r.low = fmaxf(lowest, w.at(r.end + 1.0, -1.0));
			r.from = 0;
			r.to = last;
#pragma clang loop unroll(disable)
			for (;;) {
				if (threadIdx.x == 0) {
					s.listed = 0;
					s.low = ~0ull;
					s.high = 0;
				}
				__syncthreads();
				const List list{lds_of(s.list), lds_of(&s.listed), lds_of(&s.low), lds_of(&s.high)};
				if (SLICED && near && r.end <= kNear) gather(noted, w, cut, r, list);
				else gather(row, w, cut, r, list);
				__syncthreads();
				if (s.listed <= kList) break;
				// more than the list holds: the keys' range is divided, and the part with the element taken
				r.from = s.low;
				r.to = s.high;
				int shift = 0;
				while ((r.to - r.from) >> shift >= BINS) ++shift;
				for (int i = threadIdx.x; i < BINS; i += NT) s.part[i] = 0;
				__syncthreads();
				if (SLICED && near && r.end <= kNear) divide(noted, w, cut, number, r, shift, lds_of(s.part));
				else divide(row, w, cut, number, r, shift, lds_of(s.part));
				__syncthreads();
				scan_bins(s, s.part);
				const int sub = find_bin(s, s.part, x - ahead);
				ahead += s.part[sub];
				r.to = min(r.to, r.from + ((((u64)sub + 1) << shift) - 1));
				r.from = r.from + ((u64)sub << shift);
			}
			order_list(s, number ? 0 : ahead, number ? (unsigned)ahead : 0);
		} else {
			ask();
		}
		for (int i = threadIdx.x; i < (int)s.listed; i += NT) {
			const u64 from = number ? (u64)s.rank[i] : s.before[i], own = number ? 1 : s.list[i].mass;
			if (from < x && x <= from + own) s.found = Found{s.list[i].key, s.before[i], s.list[i].mass};
		}
		__syncthreads();
		f = s.found;
		__syncthreads();
		if (question < 2) sum = f.before + f.mass;
		if (number && !complete) {  // the other questions are about what top-k leaves
			last = f.key;
			lowest = fmaxf(lowest, logit_of((unsigned)(last >> 32)));
			last_step = -Weights::back(Weights::whole(w.steps(lowest)));
		}
	}
	if (threadIdx.x == 0) {
		a.tokens[n] = (int)(unsigned)f.key;
		const double far = w.steps(logit_of((unsigned)(f.key >> 32))) * (kLn2 / kFine);
		if (a.logprob) a.logprob[n] = (float)(-far - log(__builtin_ldexp((double)sum, -a.bits)));
	}
}

// Slices of a row: as many as bring 512 workgroups together, of 1024 words (16 KB) at least.
int slices_of(int64_t rows, int64_t V, int64_t size) {
	const int64_t words = (V * size + 15) / 16;
	return V > 8192 && rows ? (int)std::max<int64_t>(1, std::min(512 / rows, words / 1024)) : 0;
}

template <typename T>
hipError_t launch(const SampleArgs& a, hipStream_t s) {
	Slices x{a.slices, 0, nullptr, nullptr, nullptr};
	if (!a.slices) {
		sample_kernel<T, 256, 512, false><<<(unsigned)a.rows, 256, 0, s>>>(a, x);
		return hipGetLastError();
	}
	const int64_t at_once = std::min(a.rows, kSliceRows);
	x.sum = (u64*)a.scratch;
	x.noted = x.sum + at_once * (kSliceBins + 2);
	x.top = (float*)(x.noted + at_once * kNearRow);
	for (; x.row0 < a.rows; x.row0 += at_once) {
		const unsigned rows = (unsigned)std::min(at_once, a.rows - x.row0);
		sample_top_kernel<T><<<dim3(x.count, rows), kSliceThreads, 0, s>>>(a, x);
		sample_bins_kernel<T><<<dim3(x.count, rows), kSliceThreads, 0, s>>>(a, x);
		sample_kernel<T, 1024, kSliceBins, true><<<rows, 1024, 0, s>>>(a, x);
	}
	return hipGetLastError();
}

}  // namespace

size_t sample_scratch(int64_t rows, int64_t V, int type, int& slices) {
	slices = slices_of(rows, V, type == kF32 ? 4 : 2);
	return slices ? (size_t)std::min(rows, kSliceRows) * ((kSliceBins + 2 + kNearRow) * sizeof(u64) + slices * 4) : 0;
}

hipError_t sample(const SampleArgs& a, int type, hipStream_t s) {
	return type == kF32 ? launch<float>(a, s) : launch<__bf16>(a, s);
}

}  // namespace nnh
