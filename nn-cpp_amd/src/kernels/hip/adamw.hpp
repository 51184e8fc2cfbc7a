// adamw.hpp - one AdamW step over many tensors, moments in 32 bits or in 8 (internal to libnnh).
//
//   g' = g scale;  m = b1 m + (1 - b1) g';  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nnh {

struct AdamWTensor {
	void* p;
	const void* g;
	void *m, *v;
	uint8_t *m_scale, *v_scale;  // 8 bits: a power of two (biased by 127) for each 64 elements
	void* copy;                  // bf16, or null
	int64_t count;
};

struct AdamWArgs {
	double beta1, beta2, lr, decay, eps;
	double first, second;        // 1 - beta^t, unless step_device is set
	double log1, log2;           // log2 of the betas
	const int* step_device;
	const float *lr_device, *grad_scale;
};

// p_type and g_type: 0 fp32, 1 bf16.
hipError_t adamw_step(const AdamWArgs& a, const AdamWTensor* tensors, size_t n, int p_type, int g_type, int bits, hipStream_t s);

}  // namespace nnh
