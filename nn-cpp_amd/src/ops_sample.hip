// ops_sample.hip - extern "C" entry point of sampling (include/nnh.h).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "abi_common.hpp"
#include "kernels/hip/sample.hpp"
#include "scratch.hpp"
#include "nnh.h"

using namespace nnh;

namespace {

constexpr uint64_t kMaxVocabulary = (uint64_t)1 << 28;
constexpr uint64_t kMaxRows = (1u << 22) - 1;  // of up to 1024 work-items each, below 2^32 together

int refuse(int code, const char* what) { return fail(code, std::string("sample: ") + what); }

}  // namespace

extern "C" {

int nnh_sample(int type, const void* logits, size_t rows, size_t V, size_t ld, const float* u, const float* temperature, const int* top_k,
               const float* top_p, const float* min_p, int* tokens, float* logprob, void* stream) {
	return guarded([&] {
		if (type != NNH_F32 && type != NNH_BF16) return refuse(NNH_ERR_INVALID, "no such element type");
		uint64_t x = 0;
		if (V == 0) return refuse(NNH_ERR_SHAPE, "an empty vocabulary");
		if (rows > kMaxRows || V > kMaxVocabulary || ld < V || !count_ok({rows, ld}, x)) return refuse(NNH_ERR_INVALID, "size out of range, or rows longer than their pitch");
		if (rows == 0) return NNH_OK;
		const uint64_t size = type == NNH_F32 ? 4 : 2;
		if (!logits || !u || !tokens) return refuse(NNH_ERR_INVALID, "logits, u and tokens are needed");
		if (reinterpret_cast<uintptr_t>(logits) % size != 0 || off_words({u, temperature, top_k, top_p, min_p, tokens, logprob}))
			return refuse(NNH_ERR_INVALID, "an array is not aligned to its elements");
		const uint64_t lb = ((rows - 1) * ld + V) * size;
		for (const void* out : {(const void*)tokens, (const void*)logprob}) {
			if (!out) continue;
			bool apart = !ranges_overlap(out, rows * 4, logits, lb);
			for (const void* in : {(const void*)u, (const void*)temperature, (const void*)top_k, (const void*)top_p, (const void*)min_p})
				apart = apart && (!in || !ranges_overlap(out, rows * 4, in, rows * 4));
			if (!apart) return refuse(NNH_ERR_ALIAS, "an output overlaps an input");
		}
		if (logprob && ranges_overlap(tokens, rows * 4, logprob, rows * 4)) return refuse(NNH_ERR_ALIAS, "the two outputs overlap");
		int bits = 62;
		while (((uint64_t)1 << (62 - bits)) < V) --bits;
		SampleArgs a{logits, (int64_t)ld, (int64_t)rows, (int)V, std::min(bits, 51), u, temperature, top_k, top_p, min_p, tokens, logprob, 0, nullptr};
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		Scratch ws(s, sample_scratch((int64_t)rows, (int64_t)V, type, a.slices));
		if (ws.status() != NNH_OK) return ws.status();
		a.scratch = ws.at<void>(0);
		return hip_status(sample(a, type, s), "sample");
	});
}

int nnh_sample_workspace_size(int type, size_t rows, size_t V, size_t* bytes) {
	return guarded([&] {
		if (type != NNH_F32 && type != NNH_BF16) return refuse(NNH_ERR_INVALID, "no such element type");
		if (rows > kMaxRows || V > kMaxVocabulary) return refuse(NNH_ERR_INVALID, "size out of range");
		int slices = 0;
		return put_bytes(bytes, sample_scratch((int64_t)rows, (int64_t)V, type, slices));
	});
}

}  // extern "C"
