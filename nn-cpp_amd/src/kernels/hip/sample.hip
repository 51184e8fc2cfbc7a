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
// A workgroup takes a row. A pass finds the maximum and keeps the row's beginning in LDS, one counts and sums by bins of 1/64 of a
// factor of two, in the order wanted; then the element asked for is in a known bin. The bin's elements (or, where they are few, all
// up to it, which answers the later questions too) go into a list in LDS, whose sums are found by comparing each with each. A bin with more
// than the list holds is divided further by the order's own key (32 bits of the logit, then the index).
// The exponential: 2^-d = 2^-n 2^-(k/64) 2^-r from a table of 64 and the power series, in 64 bits.
#include <cmath>

#include "sample.hpp"

namespace nnh {

namespace {

typedef unsigned long long u64;

constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.6931471805599453094;
constexpr int kBins = 2048;   // the last one: all weights below 2^-(kBins - 1) / 64
constexpr int kList = 1024;   // elements whose order is found by comparing them

struct alignas(16) Word {
	unsigned x[4];
};
struct alignas(16) Item {
	u64 key, mass;
};

struct Found {
	u64 key, before, mass;  // of the element: its place in the order, the sum ahead of it, its own
};

template <int NT>
struct Shared {
	u64 mass[kBins + 1];  // sums ahead of each bin; the last entry: of all
	unsigned count[kBins + 1];
	u64 mass2[kBins + 1];  // of a bin that is divided further
	unsigned count2[kBins + 1];
	Item list[kList];
	u64 before[kList];
	unsigned rank[kList];
	double table[64];
	u64 wave_mass[NT / 64];
	unsigned wave_count[NT / 64];
	float wave_top[NT / 64];
	u64 low, high;
	unsigned listed;
	int bin;
	Found found;
};

template <typename T>
constexpr int per_word() { return 16 / (int)sizeof(T); }

// Descending order as ascending whole numbers (both zeros are one logit).
__device__ __forceinline__ unsigned order_of(float z) {
	const unsigned b = __float_as_uint(z + 0.0f);
	return b >> 31 ? b : 0x7fffffffu - b;
}
__device__ __forceinline__ float logit_of(unsigned o) { return __uint_as_float(o >> 31 ? o : 0x7fffffffu - o); }

// floor(f x) and ceil(f x) for 0 <= f < 1.
__device__ __forceinline__ u64 part_of(float f, u64 x, bool up) {
	const unsigned b = __float_as_uint(f), e = b >> 23;
	if (!(f > 0.0f)) return 0;
	const unsigned m = e ? (b & 0x7fffffu) | 0x800000u : b & 0x7fffffu;
	const int shift = 150 - (int)(e ? e : 1);  // f = m 2^-shift, shift at least 24
	const unsigned __int128 y = (unsigned __int128)m * x;
	if (shift >= 100) return up && y != 0 ? 1 : 0;
	const u64 q = (u64)(y >> shift);
	return q + (up && (y & (((unsigned __int128)1 << shift) - 1)) != 0 ? 1 : 0);
}

template <typename T, bool VEC, int NT, int CACHE>
struct Row {
	static constexpr int E = per_word<T>();
	const T* z;
	int V, words, kept;
	Word* cache;  // the row's first `kept` words; each thread reads those that it has stored

	__device__ __forceinline__ Word load(int w) const {
		if (VEC && (w + 1) * E <= V) return *(const Word*)(z + w * E);
		union {
			T e[E];
			Word w;
		} u;
#pragma unroll
		for (int i = 0; i < E; ++i) u.e[i] = w * E + i < V ? z[w * E + i] : (T)(-__builtin_huge_valf());
		return u.w;
	}
	// f(z, index) of every element that is a number; FIRST stores what the others find in LDS
	template <bool FIRST, typename F>
	__device__ __forceinline__ void each(F f) const {
		for (int w = threadIdx.x; w < words; w += NT) {
			union {
				Word w;
				T e[E];
			} u;
			if (FIRST || w >= kept) u.w = load(w);
			else u.w = cache[w];
			if (FIRST && w < kept) cache[w] = u.w;
#pragma unroll
			for (int i = 0; i < E; ++i) {
				const float x = (float)u.e[i];
				if (x > -__builtin_huge_valf()) f(x, w * E + i);
			}
		}
	}
};

// The weights of a row: d = (max - z) / temperature in units of log 2.
struct Weights {
	double top, c;
	int bits;
	u64 least;  // smaller ones are not kept
	const double* table;
	__device__ __forceinline__ double steps(float z) const {  // 64 d
		return (double)z == top ? 0.0 : (top - (double)z) * c;
	}
	__device__ __forceinline__ u64 mass(double steps) const {
		if (!(steps < 64.0 * 53.0)) return 0;
		const int k = (int)steps;
		const double r = (steps - (double)k) * (-kLn2 / 64.0);  // at most 0.011: r^6 / 720 is 2e-15
		double p = __builtin_fma(r, 1.0 / 120.0, 1.0 / 24.0);
		p = __builtin_fma(r, p, 1.0 / 6.0);
		p = __builtin_fma(r, p, 0.5);
		p = __builtin_fma(r, p, 1.0);
		p = __builtin_fma(r, p, 1.0);
		// 2^52 beside it, the sum's last place is 1: the nearest whole number is in its low bits
		const double y = __builtin_ldexp(p * table[k & 63], bits - (k >> 6)) + 0x1p52;
		return (u64)__double_as_longlong(y) & 0xfffffffffffffull;
	}
	__device__ __forceinline__ int bin(double steps) const { return steps < (double)(kBins - 1) ? (int)steps : kBins - 1; }
};

// Sums and numbers ahead of each bin, in place.
template <int NT>
__device__ void scan_bins(Shared<NT>& s, u64* mass, unsigned* count) {
	constexpr int per = kBins / NT, NW = NT / 64;
	static_assert(per >= 1 && per * NT == kBins, "bins to a thread");
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	u64 m[per], mt = 0;
	unsigned c[per], ct = 0;
#pragma unroll
	for (int i = 0; i < per; ++i) {
		m[i] = mass[threadIdx.x * per + i];
		c[i] = count[threadIdx.x * per + i];
		mt += m[i];
		ct += c[i];
	}
	u64 ms = mt;
	unsigned cs = ct;
#pragma unroll
	for (int d = 1; d < 64; d *= 2) {
		const u64 mo = __shfl_up(ms, d);
		const unsigned co = __shfl_up(cs, d);
		if (lane >= d) {
			ms += mo;
			cs += co;
		}
	}
	if (lane == 63) {
		s.wave_mass[wave] = ms;
		s.wave_count[wave] = cs;
	}
	__syncthreads();
	ms -= mt;
	cs -= ct;
	for (int w = 0; w < NW; ++w)
		if (w < wave) {
			ms += s.wave_mass[w];
			cs += s.wave_count[w];
		}
#pragma unroll
	for (int i = 0; i < per; ++i) {
		mass[threadIdx.x * per + i] = ms;
		count[threadIdx.x * per + i] = cs;
		ms += m[i];
		cs += c[i];
	}
	if (threadIdx.x == NT - 1) {
		mass[kBins] = ms;
		count[kBins] = cs;
	}
	__syncthreads();
}

// The bin with before < x <= before + own, by number or by sum.
template <int NT>
__device__ int find_bin(Shared<NT>& s, const u64* mass, const unsigned* count, u64 x, bool number) {
	for (int b = threadIdx.x; b < kBins; b += NT) {
		const u64 from = number ? count[b] : mass[b], to = number ? count[b + 1] : mass[b + 1];
		if (from < x && x <= to) s.bin = b;
	}
	__syncthreads();
	const int b = s.bin;
	__syncthreads();
	return b;
}

// What the list's elements have ahead of them, which starts from the sum and number given.
template <int NT>
__device__ void order_list(Shared<NT>& s, u64 mass, unsigned count) {
	const int n = s.listed;
	for (int i = threadIdx.x; i < n; i += NT) {
		s.before[i] = mass;
		s.rank[i] = count;
	}
	__syncthreads();
	// element i by NT / width threads, each with its share of the others
	int width = 64;
	while (width < n) width *= 2;
	const int shares = NT > width ? NT / width : 1, share = threadIdx.x / width, per = (n + shares - 1) / shares;
	for (int i = threadIdx.x % width; i < n; i += min(width, NT)) {
		if (share >= shares) break;
		const u64 key = s.list[i].key;
		u64 m = 0;
		unsigned c = 0;
		for (int j = share * per; j < min(n, (share + 1) * per); ++j) {
			const Item o = s.list[j];
			if (o.key < key) {
				m += o.mass;
				++c;
			}
		}
		if (m) atomicAdd(&s.before[i], m);
		if (c) atomicAdd(&s.rank[i], c);
	}
	__syncthreads();
}

template <typename T, bool VEC, int NT, int CACHE>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
	__shared__ Shared<NT> s;
	__shared__ Word cache[CACHE];
	const int64_t n = blockIdx.x;
	Row<T, VEC, NT, CACHE> row;
	row.z = (const T*)a.logits + n * a.ld;
	row.V = a.V;
	row.words = (a.V + row.E - 1) / row.E;
	row.kept = min(row.words, CACHE);
	row.cache = cache;
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

	if (threadIdx.x < 64) s.table[threadIdx.x] = exp2((double)threadIdx.x * (-1.0 / 64.0));
	for (int b = threadIdx.x; b < kBins; b += NT) {
		s.mass[b] = 0;
		s.count[b] = 0;
	}
	float best = -__builtin_huge_valf();
	row.template each<true>([&](float z, int) { best = fmaxf(best, z); });
#pragma unroll
	for (int d = 32; d; d >>= 1) best = fmaxf(best, __shfl_xor(best, d));
	if (lane == 0) s.wave_top[wave] = best;
	if (threadIdx.x == 0) {
		s.listed = 0;
		s.low = ~0ull;
	}
	__syncthreads();
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
		row.template each<false>([&](float z, int i) {
			if (z == best) atomicMin(&s.low, (u64)i);
		});
		__syncthreads();
		if (threadIdx.x == 0) {
			a.tokens[n] = (int)s.low;
			if (a.logprob) a.logprob[n] = 0.0f;
		}
		return;
	}
	Weights w{best, 64.0 * kLog2e / (double)temperature, a.bits, 1, s.table};
	const float min_p = a.min_p ? a.min_p[n] : 0.0f;
	if (min_p > 0.0f) w.least = max(1ull, (u64)ceil(__builtin_ldexp((double)fminf(min_p, 1.0f), a.bits)));

	{
		// (the last bin's elements, often most of a row's, are summed in registers)
		u64 tail = 0;
		unsigned tails = 0;
		row.template each<false>([&](float z, int) {
			const double d = w.steps(z);
			const u64 q = w.mass(d);
			if (q < w.least) return;
			const int b = w.bin(d);
			if (b == kBins - 1) {
				tail += q;
				++tails;
			} else {
				atomicAdd(&s.mass[b], q);
				atomicAdd(&s.count[b], 1u);
			}
		});
		if (tails) {
			atomicAdd(&s.mass[kBins - 1], tail);
			atomicAdd(&s.count[kBins - 1], tails);
		}
	}
	__syncthreads();
	scan_bins(s, s.mass, s.count);

	int have_from = 0, have_to = -1;  // bins whose elements are in the list
	auto gather = [&](u64 from, u64 to, int first, int last) {  // elements of these bins with a key in [from, to]
		row.template each<false>([&](float z, int i) {
			const double d = w.steps(z);
			const int b = w.bin(d);
			if (b < first || b > last) return;
			const u64 key = (u64)order_of(z) << 32 | (unsigned)i;
			if (key < from || key > to) return;
			const u64 q = w.mass(d);
			if (q < w.least) return;
			const unsigned at = atomicAdd(&s.listed, 1u);
			if (at < kList) s.list[at] = Item{key, q};
		});
		__syncthreads();
	};
	// The element with before < x <= before + own.
	auto find = [&](u64 x, bool number) -> Found {
		const int b = find_bin(s, s.mass, s.count, x, number);
		if (b < have_from || b > have_to) {
			have_from = b;
			have_to = b;
			if (s.count[b + 1] <= kList) have_from = 0;
			u64 mass = s.mass[have_from];
			unsigned count = s.count[have_from];
			const unsigned own = s.count[b + 1] - count;
			if (threadIdx.x == 0) {
				s.listed = 0;
				s.low = ~0ull;
				s.high = 0;
			}
			__syncthreads();
			if (own <= kList) {
				gather(0, ~0ull, have_from, b);
			} else {
				// the keys' range, divided until the part with the element fits the list
				u64 low = ~0ull, high = 0;
				row.template each<false>([&](float z, int i) {
					if (w.bin(w.steps(z)) != b) return;
					const u64 key = (u64)order_of(z) << 32 | (unsigned)i;
					low = min(low, key);
					high = max(high, key);
				});
				atomicMin(&s.low, low);
				atomicMax(&s.high, high);
				__syncthreads();
				low = s.low;
				high = s.high;
				for (;;) {
					int shift = 0;
					while ((high - low) >> shift >= kBins) ++shift;
					for (int i = threadIdx.x; i < kBins; i += NT) {
						s.mass2[i] = 0;
						s.count2[i] = 0;
					}
					__syncthreads();
					row.template each<false>([&](float z, int i) {
						const double d = w.steps(z);
						if (w.bin(d) != b) return;
						const u64 key = (u64)order_of(z) << 32 | (unsigned)i;
						if (key < low || key > high) return;
						const u64 q = w.mass(d);
						if (q < w.least) return;
						atomicAdd(&s.mass2[(key - low) >> shift], q);
						atomicAdd(&s.count2[(key - low) >> shift], 1u);
					});
					__syncthreads();
					scan_bins(s, s.mass2, s.count2);
					const int sub = find_bin(s, s.mass2, s.count2, x - (number ? (u64)count : mass), number);
					const unsigned in = s.count2[sub + 1] - s.count2[sub];
					mass += s.mass2[sub];
					count += s.count2[sub];
					high = min(high, low + ((((u64)sub + 1) << shift) - 1));
					low = low + ((u64)sub << shift);
					__syncthreads();
					if (in <= kList) break;
				}
				gather(low, high, b, b);
				have_to = -1;  // a part of the bin: no other question's
			}
			order_list(s, mass, count);
		}
		for (int i = threadIdx.x; i < (int)s.listed; i += NT) {
			const u64 from = number ? (u64)s.rank[i] : s.before[i], own = number ? 1 : s.list[i].mass;
			if (from < x && x <= from + own) s.found = Found{s.list[i].key, s.before[i], s.list[i].mass};
		}
		__syncthreads();
		const Found f = s.found;
		__syncthreads();
		return f;
	};

	u64 sum = s.mass[kBins];
	const int k = a.top_k ? a.top_k[n] : 0;
	if (k > 0 && (unsigned)k < s.count[kBins]) {
		const Found f = find((u64)k, true);
		sum = f.before + f.mass;
	}
	const float top_p = a.top_p ? a.top_p[n] : 1.0f;
	if (top_p < 1.0f) {
		const Found f = find(max(1ull, part_of(top_p, sum, true)), false);
		sum = f.before + f.mass;
	}
	const float u = a.u[n];
	const Found f = find(u < 1.0f ? part_of(u, sum, false) + 1 : sum, false);
	if (threadIdx.x == 0) {
		a.tokens[n] = (int)(unsigned)f.key;
		const double far = w.steps(logit_of((unsigned)(f.key >> 32))) * (kLn2 / 64.0);
		if (a.logprob) a.logprob[n] = (float)(-far - log(__builtin_ldexp((double)sum, -a.bits)));
	}
}

template <typename T, bool VEC>
hipError_t launch(const SampleArgs& a, hipStream_t s) {
	// 256 threads where they pass over a row in a few rounds; the LDS beside the bins keeps as much of a row as there is room for
	if (a.V <= 8192) sample_kernel<T, VEC, 256, 1024><<<(unsigned)a.rows, 256, 0, s>>>(a);
	else sample_kernel<T, VEC, 1024, 4096><<<(unsigned)a.rows, 1024, 0, s>>>(a);
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
