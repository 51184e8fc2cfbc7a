// paged_attention.hip - new keys and values into their pages, and how a call of attention over pages is divided.
#include "paged_attention.hpp"

#include <algorithm>

namespace nnh {

namespace attn {
template <typename T>
hipError_t paged_of(const PagedAttentionArgs& p, bool vec, hipStream_t s);
}  // namespace attn

namespace {

// A wave takes a row of one of the two: its place is worked out once, its words go 64 at a time. Bound by memory: every element
// is read and written once (16384 bf16 rows of 8 heads of 128, 22 us, a copy's rate).
template <typename T, typename W>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs p) {
	constexpr int E = (int)(sizeof(W) / sizeof(T));
	const int lane = threadIdx.x & 63;
	const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
	if (row >= p.s.rows) return;
	const int lo = sequence_with(p.s, row, lane);
	if (lo == p.s.N || row < p.s.starts[lo]) return;
	const int64_t at = (int64_t)p.s.lens[lo] - p.s.starts[lo + 1] + row;
	if (at < 0 || at >= (int64_t)p.t.width * p.t.size.d) return;
	const unsigned block = fdiv((unsigned)at, p.t.size);
	const int page = p.t.table[(int64_t)lo * p.t.width + block];
	if ((unsigned)page >= (unsigned)p.t.pages) return;
	const int64_t to = page * p.t.page + (int64_t)((unsigned)at - block * p.t.size.d) * p.t.slot;
	const bool v = blockIdx.y != 0;
	const HeadStrides& st = v ? p.vs : p.ks;
	const T* const src = (const T*)(v ? p.v : p.k) + row * st.row;
	T* const dst = (T*)(v ? p.v_pages : p.k_pages) + to;
	const int words = p.dh / E;
	for (int x = lane; x < p.Hkv * words; x += 64) {
		const int h = x / words, d = x % words * E;
		*(W*)(dst + h * p.t.head + d) = *(const W*)(src + h * st.head + d);
	}
}

struct alignas(16) Word16 {
	unsigned x[4];
};

template <typename T>
hipError_t append_of(const PagedAppendArgs& p, bool vec, hipStream_t s) {
	const dim3 grid((unsigned)(((int64_t)p.s.rows + 3) / 4), 2);
	if (vec) paged_append_kernel<T, Word16><<<grid, 256, 0, s>>>(p);
	else paged_append_kernel<T, T><<<grid, 256, 0, s>>>(p);
	return hipGetLastError();
}

}  // namespace

// Columns: a sequence of at most 64 takes the split form, whose waves share the keys, not the columns. The keys are divided so that
// three workgroups a CU come together, two in the other form, or up to four times as many (rounds_of), 256 keys to each at least; where
// the rows alone bring enough, or a sequence has room for fewer than 1024 keys (512 in the wide form), they are not: a second launch, and
// parts to memory and back, take longer than four tiles to a wave. (One token, 8 key heads: 500 keys undivided 13 us in bf16 of 128 and 18 in
// fp32 of 64, divided 24 and 30; 1000: 18 and 29, but 60 for 46 in fp32 of 128; 1900: 28 and 52. Room is not length: 500 keys under a
// table of 1024 places are divided.) (768 for 512 wanted: mixed lengths around 3000, 12 heads of
// 80, 98 -> 89 us; 1024: 86, but 128 sequences of 1000 keys 89 -> 106.) A sequence has one group at least, and one part of each group.
PagedPlan paged_attention_plan(int64_t N, int64_t rows, int64_t most, int64_t keys, int H, int Hkv, int Dh) {
	constexpr int kFew = 64, kSplitWanted = 768, kWideWanted = 512;
	PagedPlan p{kFew, {false, 5, 5, 0, 0, 0, nullptr}, {true, 7, 6, 0, 0, 0, nullptr}, 0, 0};
	if (N == 0 || rows == 0 || most == 0) return p;
	const int64_t G = H / Hkv, columns = std::min(most, rows) * G;
	const auto divide = [&](Form& f, int64_t groups, bool enough, int64_t from, int wanted, size_t& floats) {
		if (!enough && keys >= from) f.target = (wanted + Hkv - 1) / Hkv;
		const int64_t tiles = groups * ((keys + 31) / 32);
		f.pairs = (int)(groups + (f.target ? std::min<int64_t>(f.target * rounds_of(tiles, f.target), tiles / (kLeastKeys / 32) + 1) : 0));
		f.room = (int)std::min<int64_t>(1 << f.width, columns);
		floats = f.target ? (size_t)Hkv * f.pairs * f.room * (Dh + 2) : 0;
	};
	const bool split = columns <= kFew || N > 1;
	if (split) divide(p.split, std::min(2 * N, N + rows * G / 32), N * Hkv >= 8 * kSplitWanted, 1024, kSplitWanted, p.split_floats);
	else p.few = 0;
	if (columns > kFew) divide(p.wide, N + rows * G / 128, rows * G / 128 * Hkv >= kWideWanted, 512, kWideWanted, p.wide_floats);
	return p;
}

hipError_t paged_append(const PagedAppendArgs& p, int type, bool vec, hipStream_t s) {
	return type == kF32 ? append_of<float>(p, vec, s) : append_of<__bf16>(p, vec, s);
}
hipError_t paged_attention(const PagedAttentionArgs& p, int type, bool vec, hipStream_t s) {
	return type == kF32 ? attn::paged_of<float>(p, vec, s) : attn::paged_of<__bf16>(p, vec, s);
}

}  // namespace nnh
