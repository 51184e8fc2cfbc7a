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

// The sequence that has a row (N: none), by a wave that looks at 64 bounds at a time.
__device__ __forceinline__ int sequence_with(const PackedRows& s, int64_t row, int lane) {
	for (int n0 = 0; n0 < s.N; n0 += 64) {
		const uint64_t behind = __ballot(n0 + lane < s.N && s.starts[n0 + lane + 1] <= row);
		if (behind != ~0ull) return n0 + __builtin_ctzll(~behind);
	}
	return s.N;
}

struct PagedAppendArgs {
	const void *k, *v;
	HeadStrides ks, vs;  // (sample: unused)
	void *k_pages, *v_pages;
	PageTable t;
	PackedRows s;
	int Hkv, dh;
};

// One of the two forms: columns in groups of 2^width, keys in tiles of 2^shift.
struct Form {
	bool wide;
	int width, shift;
	int target;      // pairs of a group and a part of the keys that are wanted, to a key head; 0: the keys are not divided
	int pairs;       // and at most so many there will be; 0: the form has no sequence to take
	int room;        // columns of a group, at most
	float* partial;  // {Hkv, pairs, room}: maximum, sum and dh sums of p v each
};

struct PagedAttentionArgs {
	MaskedAttentionArgs a;  // q, k and v (the pages), out, the rule
	PageTable t;
	PackedRows s;
	int most;          // rows of a sequence, at most
	int few;           // sequences of so many columns (rows times the heads of a key head) or fewer take the split form
	Form split, wide;
	float* lse;        // {rows, H}
};

// A pair's fixed cost is that of some ten tiles of the split form, and more pairs share the work more evenly: up to four rounds over
// the GPU, where each pair has 48 tiles.
__host__ __device__ inline int rounds_of(int64_t tiles, int target) {
	const int64_t rounds = tiles / ((int64_t)target * 48);
	return rounds < 1 ? 1 : rounds > 4 ? 4 : (int)rounds;
}
constexpr int kLeastKeys = 256;  // of a part

// How a call is divided, from what the host knows of it, and the floats of the forms' `partial`.
struct PagedPlan {
	int few;
	Form split, wide;
	size_t split_floats, wide_floats;
};
PagedPlan paged_attention_plan(int64_t N, int64_t rows, int64_t most, int64_t keys, int H, int Hkv, int Dh);

hipError_t paged_append(const PagedAppendArgs& p, int type, bool vec, hipStream_t s);
hipError_t paged_attention(const PagedAttentionArgs& p, int type, bool vec, hipStream_t s);

}  // namespace nnh
