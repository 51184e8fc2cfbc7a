// paged_attention.hpp - attention of new tokens over keys and values in pages, and the new ones' way into the pages (internal to
// libnnh). The mathematics is masked attention's (masked_attention.hpp); queries are packed rows of many sequences.
#pragma once

#include "fastdiv.hpp"
#include "masked_attention.hpp"

namespace nnh {

// Where tokens are kept: token j of sequence n in slot j % size of page table[n][j / size].
struct PageTable {
	const int* table;  // {N, width}
	int64_t page, slot, head;  // strides in elements
	FastDiv size;
	int pages, width;
};

// Rows starts[n] .. starts[n + 1] - 1 are sequence n's, the last of the lens[n] tokens that it has with them.
struct PackedRows {
	const int* starts;
	const int* lens;
	int N, rows;
};

struct PagedAppendArgs {
	const void *k, *v;
	HeadStrides ks, vs;  // (sample: unused)
	void *k_pages, *v_pages;
	PageTable t;
	PackedRows s;
	int Hkv, dh;
};

struct PagedAttentionArgs {
	MaskedAttentionArgs a;  // q, k and v (the pages), out, the rule; Tk: the most tokens that a sequence may have
	PageTable t;
	PackedRows s;
	int most;         // rows of a sequence, at most
	int few;          // sequences of so many columns (rows times the heads of a key head) or fewer take the split form
	int splits, wide_splits;  // parts that the keys of a sequence are divided into: in the split form, in the other one
	float* lse;       // {rows, H}
	float* partial;   // {parts, rows, H}: maximum, sum and dh sums of p v each
};

// How a call is divided, from what the host knows of it.
struct PagedPlan {
	int few, splits, wide_splits;  // splits or wide_splits 0: that form has no sequence to take
};
PagedPlan paged_attention_plan(int N, int rows, int most, int keys, int H, int Hkv);

hipError_t paged_append(const PagedAppendArgs& p, int type, bool vec, hipStream_t s);
hipError_t paged_attention(const PagedAttentionArgs& p, int type, bool vec, hipStream_t s);

}  // namespace nnh
