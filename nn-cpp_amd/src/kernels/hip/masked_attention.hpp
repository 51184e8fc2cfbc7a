// masked_attention.hpp - attention over heads that may share keys and values, with capped scores, a distance bias and
// causal, window, prefix, document and length masks; probabilities are never stored (internal to libnnh).
//
//   s = scale q.k,  c = cap tanh(s / cap) (cap > 0),  z = c - slope_h |pos - j|,  out = softmax(z over visible j) v
//   pos = q_start + i;  visible(i, j): j < k_len and the documents agree, and (causal: j <= pos; window: |pos - j| <
//   window) or j < prefix
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nnh {

enum ElemType : int { kF32 = 0, kBf16 = 1 };

// An operand's element strides: sample, row (token) and head; the elements of a head are consecutive.
struct HeadStrides {
	int64_t sample, row, head;
};

// Rows that a tile's loads reach with 32-bit offsets.
inline bool wide_row(int64_t row_bytes) { return row_bytes <= (int64_t)1 << 23; }

// What one block of 64 tokens holds: the least and largest document number (negative ones left out; lo > hi: none) and
// whether a token belongs to none.
struct DocRange {
	int lo, hi, none;
};

struct MaskedAttentionArgs {
	const void *q, *k, *v;
	HeadStrides qs, ks, vs;
	void* out;  // forward: written; backward: the forward's
	HeadStrides os;
	void* rest;  // in 16 bits, or null: what out lost in its rounding, itself in 16 bits
	HeadStrides rs;
	float* lse;  // {N, H, Tq}, natural logarithm
	int N, Tq, Tk, H, Hkv, G, dh;  // G = H / Hkv query heads to a key head
	float scale, cap;
	const float* slopes;  // {H} or null
	int causal, window;   // window 0: none
	const int *q_start, *k_lens, *prefix, *q_docs, *k_docs;  // null: 0, Tk, 0, one document
	const DocRange *q_ranges, *k_ranges;                     // {N, ceil(T / 64)}, set where documents are
	// backward
	const void* g;
	HeadStrides gs;
	float *delta, *lse2;  // {N, H, Tq}: g.out per row, and lse in units of log 2
	void *dq, *dk, *dv;
	HeadStrides dqs, dks, dvs;
	int dq_first, dk_first, dv_first;
	// the split form: {splits, N, H, Tq}, maximum, sum and dh sums of p v each; dk and dv in parts: {parts, 2, N, Hkv, Tk}, dh
	// sums each, rounded up to a multiple of 4
	float* partial;
	int splits, parts;
};

// Whether the split form (few query rows, the keys divided over the grid) takes a call, and into how many parts.
int masked_attention_splits(int N, int Tq, int Tk, int H, int Hkv);
// Workgroups that share a key tile of the backward pass.
int masked_attention_parts(int N, int Tq, int Tk, int H, int Hkv);

hipError_t document_ranges(const int* docs, int N, int T, DocRange* out, hipStream_t s);
hipError_t masked_attention_forward(const MaskedAttentionArgs& a, int type, bool vec, hipStream_t s);
hipError_t masked_attention_split(const MaskedAttentionArgs& a, int type, bool vec, hipStream_t s);
hipError_t masked_attention_backward(const MaskedAttentionArgs& a, int type, bool vec, hipStream_t s);

}  // namespace nnh
