// sample.hpp - one token of each row of logits (internal to libnnh).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "masked_attention.hpp"

namespace nnh {

struct SampleArgs {
	const void* logits;  // {rows, V}
	int64_t ld;
	int64_t rows;
	int V;
	int bits;  // a weight of 1 is 2^bits, so that V of them stay below 2^62
	const float *u, *temperature;  // {rows}
	const int* top_k;
	const float *top_p, *min_p;
	int* tokens;
	float* logprob;
	int slices;     // workgroups that share a row's first passes, or 0
	void* scratch;  // theirs
};

// Scratch of a call, and its slices.
size_t sample_scratch(int64_t rows, int64_t V, int type, int& slices);

hipError_t sample(const SampleArgs& a, int type, hipStream_t s);

}  // namespace nnh
