// gemm16.hip - which tile a bf16 product of the linear head takes (gemm16.hpp).
#include "gemm16.hpp"

namespace nnh {

namespace g16 {

using Large = Tile<256, 256, 128, 64>;
using Small = Tile<128, 128, 64, 64>;

// 256 x 256 tiles from 200 of them on (a workgroup a CU, 256 CUs); below that, 128 x 128 ones fill the GPU better.
static bool large(int64_t inner, int64_t outer) { return ((inner + 255) / 256) * ((outer + 255) / 256) >= 200; }

template <class T, bool ATR, bool BTR, int EPI>
static hipError_t launch(const Gemm16Args& a, hipStream_t s) {
	const int64_t blocks = (int64_t)((a.inner + T::BM - 1) / T::BM) * ((a.outer + T::BN - 1) / T::BN);
	if (blocks == 0) return hipSuccess;
	gemm16_kernel<T, ATR, BTR, EPI><<<(unsigned)blocks, T::kThreads, 0, s>>>(a);
	return hipGetLastError();
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

hipError_t gemm16_out(const Gemm16Args& a, bool b_tr, hipStream_t s) {
	if (g16::large(a.inner, a.outer))
		return b_tr ? g16::launch<g16::Large, true, true, kGemm16Out>(a, s) : g16::launch<g16::Large, true, false, kGemm16Out>(a, s);
	return b_tr ? g16::launch<g16::Small, true, true, kGemm16Out>(a, s) : g16::launch<g16::Small, true, false, kGemm16Out>(a, s);
}

}  // namespace nnh
