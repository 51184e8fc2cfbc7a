// masked_attention.hip - masked attention's choice of kernel, and the document ranges its kernels skip tiles by.
#include "masked_attention.hpp"

#include <algorithm>

namespace nnh {

namespace attn {
template <typename T>
hipError_t forward_of(const MaskedAttentionArgs& a, bool vec, bool split, hipStream_t s);
template <typename T>
hipError_t backward_of(const MaskedAttentionArgs& a, bool vec, hipStream_t s);
}  // namespace attn

namespace {

// A wave takes one block of 64 tokens.
__global__ __launch_bounds__(256) void document_ranges_kernel(const int* docs, int N, int T, DocRange* out) {
	const int lane = threadIdx.x & 63, blocks = (T + 63) / 64;
	const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
	if (at >= (int64_t)N * blocks) return;
	const int64_t n = at / blocks;
	const int i = (int)(at % blocks) * 64 + lane;
	const int d = i < T ? docs[n * T + i] : -1;
	int lo = d < 0 ? 0x7fffffff : d, hi = d < 0 ? -1 : d;
	for (int x = 32; x; x >>= 1) {
		lo = min(lo, __shfl_xor(lo, x));
		hi = max(hi, __shfl_xor(hi, x));
	}
	const bool none = __any(d < 0 && i < T);
	if (lane == 0) out[at] = DocRange{lo, hi, none ? 1 : 0};
}

}  // namespace

hipError_t document_ranges(const int* docs, int N, int T, DocRange* out, hipStream_t s) {
	const int64_t blocks = (int64_t)N * ((T + 63) / 64);
	if (blocks == 0) return hipSuccess;
	document_ranges_kernel<<<(unsigned)((blocks + 3) / 4), 256, 0, s>>>(docs, N, T, out);
	return hipGetLastError();
}

int masked_attention_splits(int N, int Tq, int Tk, int H, int Hkv) {
	if (Tq > 32 || Tq == 0) return 0;
	const int64_t groups = ((int64_t)Tq * (H / Hkv) + 31) / 32 * N * Hkv;
	return (int)std::max<int64_t>(1, std::min<int64_t>((512 + groups - 1) / groups, Tk / 256));
}

// Parts enough for 1024 workgroups (two a CU, twice), each with 16 tiles of queries at least.
int masked_attention_parts(int N, int Tq, int Tk, int H, int Hkv) {
	const int64_t blocks = std::max<int64_t>(1, (int64_t)N * Hkv * ((Tk + 127) / 128)), steps = (int64_t)(H / Hkv) * ((Tq + 31) / 32);
	return (int)std::max<int64_t>(1, std::min<int64_t>({(1024 + blocks - 1) / blocks, steps / 16, (Tq + 31) / 32, 8}));
}

hipError_t masked_attention_forward(const MaskedAttentionArgs& a, int type, bool vec, hipStream_t s) {
	return type == kF32 ? attn::forward_of<float>(a, vec, false, s) : attn::forward_of<__bf16>(a, vec, false, s);
}
hipError_t masked_attention_split(const MaskedAttentionArgs& a, int type, bool vec, hipStream_t s) {
	return type == kF32 ? attn::forward_of<float>(a, vec, true, s) : attn::forward_of<__bf16>(a, vec, true, s);
}
hipError_t masked_attention_backward(const MaskedAttentionArgs& a, int type, bool vec, hipStream_t s) {
	return type == kF32 ? attn::backward_of<float>(a, vec, s) : attn::backward_of<__bf16>(a, vec, s);
}

}  // namespace nnh
