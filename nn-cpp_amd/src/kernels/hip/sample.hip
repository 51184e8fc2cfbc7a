// sample.hip - the choice of a token from a row of logits under temperature, min-p, top-k and top-p (sample.hpp).
//
// With the row's logits in descending order (equal ones by their index), w = exp((z - max) / temperature) and prefix sums W of w, each
// filter keeps a prefix: min-p those with w >= min_p; top-k the first k; top-p the shortest whose sum reaches top_p of what the other
// two left. The token is the first of the kept prefix whose sum passes u of the prefix's. So every step asks one question: which
// element has before < X <= before + own, with `before` the sum (or the number) of the elements ahead of it; nothing is sorted.
//
// Weights are whole numbers: w 2^bits rounded to the nearest, bits 45 for a vocabulary of 128000. Their sums are exact, so they do
// not depend on an order, and the products with u and top_p are taken exactly too (128 bits): what rounds is each w alone, by half of
// 2^-bits beside the largest weight of 1, and a choice differs from that of exact weights only where a sum is nearer than that to its border.
//
// A workgroup takes a row. A pass finds the maximum and keeps the row's beginning in LDS, one sums weights (with top-k: counts) by bins
// of a share of a factor of two, in the order wanted: a window of 16 factors of two, in which the element nearly always is, the rest in
// registers. Then the element asked for is in a known bin, whose elements go into a list in LDS and are ordered by comparing each with
// each. With top-k the list takes all elements up to the k-th where they are few, and the later questions are answered there. A bin with
// more than the list holds is divided further by the order's own key (32 bits of the logit, then the index).
// The exponential: 2^-d = 2^-n 2^-(k/1024) 2^-r from a table of 1024 and the power series to r^3 (|r| <= 3.4e-4: off by 2^-50 of it).
//
// Bound by vector instructions (a pass of sums has about 25 an element, most of them in 64 bits, at the rate of 32) once the row has
// been read: logits that cannot count (below the least weight, or of no bin asked for) are left by two comparisons.
#include <cfloat>
#include <cmath>

#include "sample.hpp"

namespace nnh {

namespace {

typedef unsigned long long u64;

constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.6931471805599453094;
constexpr int kFine = 1024;          // steps to a factor of two, entries of the table
constexpr int kWindow = 16 * kFine;  // steps that the bins cover
constexpr int kList = 512;           // elements whose order is found by comparing them

struct alignas(16) Word {
	unsigned x[4];
};
struct alignas(16) Item {
	u64 key, mass;
};

struct Found {
	u64 key, before, mass;  // of the element: its place in the order, the sum ahead of it, its own
};

template <int NT, int BINS>
struct Shared {
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

template <typename T, bool VEC, int NT, int CACHE>
struct Row {
	static constexpr int E = 16 / (int)sizeof(T);
	const T* z;
	int V, words, kept;
	Word* cache;  // the row's first `kept` words; each thread reads those that it has stored

	__device__ __forceinline__ Word load(int w) const {
		if (VEC && (w + 1) * E <= V) return *(const Word*)(z + (int64_t)w * E);
		union {
			T e[E];
			Word w;
		} u;
#pragma unroll
		for (int i = 0; i < E; ++i) u.e[i] = w * E + i < V ? z[(int64_t)w * E + i] : (T)(-__builtin_huge_valf());
		return u.w;
	}
	// f(z, index) of every element with low <= z <= high, infinities as the largest number; FIRST stores what the others find in LDS.
	// Several words of a thread are on their way at a time.
	template <bool FIRST, typename F>
	__device__ __forceinline__ void each(float low, float high, F f) const {
		constexpr int U = VEC ? 4 : 2;
		for (int w0 = threadIdx.x; w0 < words; w0 += NT * U) {
			union {
				Word w;
				T e[E];
			} u[U];
#pragma unroll
			for (int x = 0; x < U; ++x) {
				const int w = w0 + x * NT;
				if (w >= words) continue;
				if (FIRST || w >= kept) u[x].w = load(w);
				else u[x].w = cache[w];
			}
#pragma unroll
			for (int x = 0; x < U; ++x) {
				const int w = w0 + x * NT;
				if (w >= words) break;
				if (FIRST && w < kept) cache[w] = u[x].w;
#pragma unroll
				for (int i = 0; i < E; ++i) {
					const float v = (float)u[x].e[i];
					if (v >= low && v <= high) f(fminf(v, FLT_MAX), w * E + i);
				}
			}
		}
	}
};

// A row's weights by the distance from the largest logit, in steps of 1 / kFine of a factor of two.
struct Weights {
	double top, c;
	int bits;
	double least;  // smaller ones are not kept
	const double* table;
	__device__ __forceinline__ double steps(float z) const { return fmin((top - (double)z) * c, 64.0 * kFine); }
	// The weight 2^bits 2^(-steps / kFine), rounded to a whole number, beside 2^52: the sum's last place is 1, and its low bits the number.
	__device__ __forceinline__ double beside(double steps, double whole) const {
		const int k = (int)whole;
		const double r = (steps - whole) * (-kLn2 / kFine);
		double p = __builtin_fma(r, 1.0 / 6.0, 0.5);
		p = __builtin_fma(r, p, 1.0);
		p = __builtin_fma(r, p, 1.0);
		return __builtin_ldexp(p * table[k & (kFine - 1)], bits - k / kFine) + 0x1p52;
	}
	__device__ __forceinline__ static u64 number(double beside) { return (u64)__double_as_longlong(beside) & 0xfffffffffffffull; }
	// A logit that lies so far from the largest, moved by more than any rounding here.
	__device__ __forceinline__ float at(double steps, double way) const {
		const double z = top - steps / c, room = fabs(z) * 0x1p-22 + fabs(top) * 0x1p-22 + 0x1p-140;
		return (float)fmin(fmax(z + way * room, -(double)FLT_MAX), (double)FLT_MAX);
	}
};

// What is ahead of each bin, in place.
template <int NT, int BINS>
__device__ void scan_bins(Shared<NT, BINS>& s, u64* sum) {
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
template <int NT, int BINS>
__device__ int find_bin(Shared<NT, BINS>& s, const u64* sum, u64 x) {
	for (int b = threadIdx.x; b < BINS; b += NT)
		if (sum[b] < x && x <= sum[b + 1]) s.bin = b;
	__syncthreads();
	const int b = s.bin;
	__syncthreads();
	return b;
}

// What the list's elements have ahead of them, which starts from the sum and number given.
template <int NT, int BINS>
__device__ void order_list(Shared<NT, BINS>& s, u64 mass, unsigned count) {
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

template <typename T, bool VEC, int NT, int BINS, int CACHE>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
	constexpr int kBin = kWindow / BINS;  // steps to a bin
	__shared__ Shared<NT, BINS> s;
	__shared__ Word cache[CACHE];
	const int64_t n = blockIdx.x;
	Row<T, VEC, NT, CACHE> row;
	row.z = (const T*)a.logits + n * a.ld;
	row.V = a.V;
	row.words = (a.V + row.E - 1) / row.E;
	row.kept = min(row.words, CACHE);
	row.cache = cache;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

	for (int i = threadIdx.x; i < kFine; i += NT) s.table[i] = exp2((double)i * (-1.0 / kFine));
	float best = -__builtin_huge_valf();
	{
		const float inf = __builtin_huge_valf();
		bool any = false;  // (the largest number stands for infinity in what `each` hands out)
		row.template each<true>(-FLT_MAX, inf, [&](float z, int) { best = fmaxf(best, z); });
		if (best == FLT_MAX) row.template each<false>(inf, inf, [&](float, int) { any = true; });
		if (any) best = inf;
	}
#pragma unroll
	for (int d = 32; d; d >>= 1) best = fmaxf(best, __shfl_xor(best, d));
	if (lane == 0) s.wave_top[wave] = best;
	if (threadIdx.x == 0) s.low = ~0ull;
	__syncthreads();
#pragma unroll
	for (int w = 0; w < NT / 64; ++w) best = fmaxf(best, s.wave_top[w]);
	if (best == -__builtin_huge_valf()) {  // no logit is a number above -infinity
		if (threadIdx.x == 0) {
			a.tokens[n] = -1;
			if (a.logprob) a.logprob[n] = best;
		}
		return;
	}
	const float temperature = a.temperature ? a.temperature[n] : 1.0f;
	if (!(temperature > 0.0f)) {  // the first of the largest
		row.template each<false>(best, best, [&](float, int i) { atomicMin(&s.low, (u64)i); });
		__syncthreads();
		if (threadIdx.x == 0) {
			a.tokens[n] = (int)s.low;
			if (a.logprob) a.logprob[n] = 0.0f;
		}
		return;
	}
	Weights w{fmin((double)best, (double)FLT_MAX), kFine * kLog2e / (double)temperature, a.bits, 1.0, s.table};
	const float min_p = a.min_p ? a.min_p[n] : 0.0f;
	const bool cut = min_p > 0.0f;
	if (cut) w.least = fmax(1.0, ceil(__builtin_ldexp((double)fminf(min_p, 1.0f), a.bits)));
	// Smaller logits have no weight, or less than min_p's (2^52 + least is exact). Beside an infinity, nothing else has one.
	const float bottom = best > FLT_MAX ? best : w.at(kFine * fmin((double)a.bits + 1.0, cut ? 0.001 - log2((double)fminf(min_p, 1.0f)) : 64.0), -1.0);
	const double least = w.least + 0x1p52;
	u64 last = ~0ull;  // the last element's key that top-k leaves
	float lowest = bottom;

	// The questions in turn: the k-th element, the one that reaches top_p, the one that passes u.
	const int top_k = a.top_k ? a.top_k[n] : 0;
	const float top_p = a.top_p ? a.top_p[n] : 1.0f, u = a.u[n];
	u64 sum = 0;            // the weights of what is kept
	int window = 0;
	u64 base = 0;           // ahead of the window
	int filled = -1;        // what the bins hold: 1 numbers of elements, 0 sums of weights
	bool complete = false;  // the list has every element from the first to the last that is kept
	Found f{0, 0, 0};
#pragma clang loop unroll(disable)
	for (int question = 0; question < 3; ++question) {
		const bool number = question == 0;
		if (question == 0 && !(top_k > 0 && top_k < a.V)) continue;
		if (question == 1 && !(top_p < 1.0f)) continue;
		u64 x = 0;
		const auto ask = [&] {
			x = question == 0 ? (u64)top_k : question == 1 ? max(1ull, part_of(top_p, sum, true)) : u < 1.0f ? part_of(u, sum, false) + 1 : sum;
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
					for (int i = threadIdx.x; i < BINS; i += NT) s.sum[i] = 0;
					if (threadIdx.x == 0) s.tail = 0;
					__syncthreads();
					const int from = window * kWindow;
					double tail = 0.0;  // whole numbers below 2^53
					const float high = window == 0 ? __builtin_huge_valf() : w.at(from - 1.0, 1.0);
					const float low = number || window > 0 ? fmaxf(lowest, w.at(from + kWindow + 1.0, -1.0)) : lowest;
					row.template each<false>(low, high, [&](float z, int i) {
						const double d = w.steps(z), whole = rint(d);
						const int k = (int)whole - from;
						if (k < 0) return;
						if (last != ~0ull && key_of(z, i) > last) return;
						double y = 0.0;
						if (!number || cut) {
							y = w.beside(d, whole);
							if (cut && y < least) return;
						}
						if (k < kWindow) atomicAdd(&s.sum[k / kBin], number ? 1 : w.number(y));
						else if (!number) tail += y - 0x1p52;
					});
					if (!number && window == 0) {
#pragma unroll
						for (int d = 32; d; d >>= 1) tail += __shfl_xor(tail, d);
						if (lane == 0 && tail > 0.0) atomicAdd(&s.tail, (u64)tail);
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
					if (window == 3) {  // fewer than top_k have a weight (2^-52 is the least)
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
			u64 ahead = complete ? 0 : base + s.sum[b], from = 0, to = ~0ull;
			const int begin = complete ? 0 : window * kWindow + b * kBin, end = window * kWindow + (b + 1) * kBin;
			const float high = begin == 0 ? __builtin_huge_valf() : w.at(begin - 1.0, 1.0), low = fmaxf(lowest, w.at(end + 1.0, -1.0));
#pragma clang loop unroll(disable)
			for (;;) {
				if (threadIdx.x == 0) {
					s.listed = 0;
					s.low = ~0ull;
					s.high = 0;
				}
				__syncthreads();
				u64 least_key = ~0ull, most_key = 0;
				row.template each<false>(low, high, [&](float z, int i) {
					const double d = w.steps(z), whole = rint(d);
					if (whole < begin || whole >= end) return;
					const u64 key = key_of(z, i);
					if (key < from || key > to || key > last) return;
					const double y = w.beside(d, whole);
					if (cut && y < least) return;
					const unsigned at = atomicAdd(&s.listed, 1u);
					if (at < kList) s.list[at] = Item{key, w.number(y)};
					least_key = min(least_key, key);
					most_key = max(most_key, key);
				});
				if (least_key <= most_key) {
					atomicMin(&s.low, least_key);
					atomicMax(&s.high, most_key);
				}
				__syncthreads();
				if (s.listed <= kList) break;
				// more than the list holds: the keys' range is divided, and the part with the element taken
				from = s.low;
				to = s.high;
				int shift = 0;
				while ((to - from) >> shift >= BINS) ++shift;
				for (int i = threadIdx.x; i < BINS; i += NT) s.part[i] = 0;
				__syncthreads();
				row.template each<false>(low, high, [&](float z, int i) {
					const u64 key = key_of(z, i);
					if (key < from || key > to) return;
					const double d = w.steps(z), y = w.beside(d, rint(d));
					if (cut && y < least) return;
					atomicAdd(&s.part[(key - from) >> shift], number ? 1 : w.number(y));
				});
				__syncthreads();
				scan_bins(s, s.part);
				const int sub = find_bin(s, s.part, x - ahead);
				ahead += s.part[sub];
				to = min(to, from + ((((u64)sub + 1) << shift) - 1));
				from = from + ((u64)sub << shift);
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
		}
	}
	if (threadIdx.x == 0) {
		a.tokens[n] = (int)(unsigned)f.key;
		const double far = w.steps(logit_of((unsigned)(f.key >> 32))) * (kLn2 / kFine);
		if (a.logprob) a.logprob[n] = (float)(-far - log(__builtin_ldexp((double)sum, -a.bits)));
	}
}

template <typename T, bool VEC>
hipError_t launch(const SampleArgs& a, hipStream_t s) {
	// 256 threads where they pass over a row in a few rounds; the LDS beside the bins keeps as much of a row as there is room for
	if (a.V <= 8192) sample_kernel<T, VEC, 256, 512, 1024><<<(unsigned)a.rows, 256, 0, s>>>(a);
	else sample_kernel<T, VEC, 1024, 2048, 6144><<<(unsigned)a.rows, 1024, 0, s>>>(a);
	return hipGetLastError();
}

}  // namespace

hipError_t sample(const SampleArgs& a, int type, hipStream_t s) {
	const int64_t size = type == kF32 ? 4 : 2;
	const bool vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.ld * size % 16 == 0;
	if (type == kF32) return vec ? launch<float, true>(a, s) : launch<float, false>(a, s);
	return vec ? launch<__bf16, true>(a, s) : launch<__bf16, false>(a, s);
}

}  // namespace nnh
