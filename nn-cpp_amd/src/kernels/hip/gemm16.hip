// gemm16.hip - which tile a bf16 product of the linear head takes (gemm16.hpp).
#include "gemm16.hpp"

#include <algorithm>

namespace nnh {

namespace g16 {

using Large = Tile<256, 256, 128, 64>;
using Small = Tile<128, 128, 64, 64>;

template <class T>
static int64_t tiles(int64_t inner, int64_t outer) { return ((inner + T::BM - 1) / T::BM) * ((outer + T::BN - 1) / T::BN); }

// 256 x 256 tiles from 200 of them on (a workgroup a CU, 256 CUs); below that, 128 x 128 ones fill the GPU better.
static bool large(int64_t inner, int64_t outer) { return tiles<Large>(inner, outer) >= 200; }

// A gradient's depth may be long where its tiles are few (dx over the vocabulary, dw over the rows): then the grid takes it
// in runs, 512 deep at least, whose sums are added afterwards in their order. 4096 x 1024 over 50257 deep: 64 large tiles in 4
// runs, where 256 small tiles without took 1026 us.
struct Cut {
	bool large;
	int64_t parts, depth;
};
static Cut cut_of(int64_t inner, int64_t outer, int64_t depth) {
	const int64_t l = std::max<int64_t>(1, tiles<Large>(inner, outer)), t = std::max<int64_t>(1, tiles<Small>(inner, outer)), most = std::max<int64_t>(1, depth / 512);
	Cut c{true, std::min((256 + l - 1) / l, most), depth};
	if (large(inner, outer)) {
		c.parts = 1;
	} else if (l * c.parts < 192) {
		c.large = false;
		c.parts = std::min((512 + t - 1) / t, most);
	}
	c.depth = ((depth + c.parts - 1) / c.parts + BK - 1) / BK * BK;
	if (c.depth > 0) c.parts = std::max<int64_t>(1, (depth + c.depth - 1) / c.depth);
	return c;
}

template <class T, bool ATR, bool BTR, int EPI>
static hipError_t launch(const Gemm16Args& a, hipStream_t s, int64_t parts = 1) {
	const int64_t blocks = tiles<T>(a.inner, a.outer);
	if (blocks == 0) return hipSuccess;
	gemm16_kernel<T, ATR, BTR, EPI><<<dim3((unsigned)blocks, (unsigned)parts), T::kThreads, 0, s>>>(a);
	return hipGetLastError();
}

// The runs' sums into the gradient, a thread to an element.
static __global__ __launch_bounds__(256) void gemm16_join_kernel(Gemm16Args a, int parts) {
	const int64_t count = (int64_t)a.outer * a.inner, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
	if (at >= count) return;
	float y = a.parts[at];
	for (int p = 1; p < parts; ++p) y += a.parts[p * count + at];
	y *= a.scale ? *a.scale * a.factor : a.factor;
	if (a.sum_in) y += a.sum[at];
	if (a.sum_out) {
		a.sum[at] = y;
	} else {
		__bf16* const o = (__bf16*)a.out + at / a.inner * a.ldo + at % a.inner;
		*o = (__bf16)(a.first ? y : y + (float)*o);
	}
}

template <class T>
static hipError_t scores(const Gemm16Args& a, int epilogue, hipStream_t s) {
	if (epilogue == kGemm16Stats) return launch<T, false, false, kGemm16Stats>(a, s);
	if (epilogue == kGemm16Keep) return launch<T, false, false, kGemm16Keep>(a, s);
	return launch<T, false, false, kGemm16Grad>(a, s);
}

}  // namespace g16

int gemm16_chunk(int64_t inner, int64_t outer) { return g16::large(inner, outer) ? g16::Large::WM : g16::Small::WM; }

hipError_t gemm16_scores(const Gemm16Args& a, int epilogue, int chunk, hipStream_t s) {
	return chunk == g16::Large::WM ? g16::scores<g16::Large>(a, epilogue, s) : g16::scores<g16::Small>(a, epilogue, s);
}

size_t gemm16_parts_floats(int64_t inner, int64_t outer, int64_t depth) {
	const g16::Cut c = g16::cut_of(inner, outer, depth);
	return c.parts > 1 ? (size_t)(c.parts * inner * outer) : 0;
}

hipError_t gemm16_out(const Gemm16Args& given, bool b_tr, hipStream_t s) {
	const g16::Cut c = g16::cut_of(given.inner, given.outer, given.depth);
	Gemm16Args a = given;
	if (c.parts == 1) a.parts = nullptr;
	a.part_depth = (int)c.depth;
	hipError_t e;
	if (c.large) e = b_tr ? g16::launch<g16::Large, true, true, kGemm16Out>(a, s, c.parts) : g16::launch<g16::Large, true, false, kGemm16Out>(a, s, c.parts);
	else e = b_tr ? g16::launch<g16::Small, true, true, kGemm16Out>(a, s, c.parts) : g16::launch<g16::Small, true, false, kGemm16Out>(a, s, c.parts);
	if (e != hipSuccess || c.parts == 1) return e;
	const int64_t count = (int64_t)a.outer * a.inner;
	g16::gemm16_join_kernel<<<(unsigned)((count + 255) / 256), 256, 0, s>>>(a, (int)c.parts);
	return hipGetLastError();
}

}  // namespace nnh
