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
// is read and written once.
template <typename T, typename W>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs p) {
	constexpr int E = (int)(sizeof(W) / sizeof(T));
	const int lane = threadIdx.x & 63;
	const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
	if (row >= p.s.rows) return;
	// the sequence that has the row, by its bounds in order
	int lo = 0, hi = p.s.N;
	while (lo < hi) {
		const int mid = (lo + hi) / 2;
		if (p.s.starts[mid + 1] <= row) lo = mid + 1;
		else hi = mid;
	}
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

// Columns: a sequence of at most 64 takes the split form, whose waves share the keys, not the columns. The parts are as many as
// bring 512 workgroups together, with 256 keys to each at least; the rows that a form has are not known here, so they are taken
// to be the most that may be.
PagedPlan paged_attention_plan(int N, int rows, int most, int keys, int H, int Hkv) {
	constexpr int kFew = 64;
	PagedPlan p{kFew, 0, 0};
	if (N == 0 || rows == 0 || most == 0) return p;
	const int64_t G = H / Hkv, columns = (int64_t)most * G;
	const auto parts = [&](int64_t groups) { return (int)std::max<int64_t>(1, std::min<int64_t>((512 + groups - 1) / groups, keys / 256)); };
	if (columns <= kFew || N > 1) p.splits = parts((std::min<int64_t>(columns, kFew) + 31) / 32 * N * Hkv);
	if (columns > kFew) p.wide_splits = parts(((int64_t)rows * G + 127) / 128 * Hkv);
	if (!p.splits) p.few = 0;
	return p;
}

hipError_t paged_append(const PagedAppendArgs& p, int type, bool vec, hipStream_t s) {
	return type == kF32 ? append_of<float>(p, vec, s) : append_of<__bf16>(p, vec, s);
}
hipError_t paged_attention(const PagedAttentionArgs& p, int type, bool vec, hipStream_t s) {
	return type == kF32 ? attn::paged_of<float>(p, vec, s) : attn::paged_of<__bf16>(p, vec, s);
}

}  // namespace nnh
