// linear_cross_entropy.hpp - softmax cross entropy of a linear head (internal to libnnh).
//
//   z = x w^T + b,  lse_i = log sum_v exp z_iv,  loss_i = lse_i - z_i,t_i
//   dz_iv = f_i (exp(z_iv - lse_i) - [v = t_i]),  dx = dz w,  dw = dz^T x,  db = sum_i dz_i
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace nnh {

// The products in bf16 (gemm16.hpp). What each leaves:
//   kGemm16Stats  z's maximum and sum of exponentials to each chunk of columns, and the targets' z
//   kGemm16Keep   also exp(z - the chunk's maximum)
//   kGemm16Grad   dz
//   kGemm16Out    a gradient
enum Gemm16Epilogue : int { kGemm16Stats, kGemm16Keep, kGemm16Grad, kGemm16Out };

struct Gemm16Args {
	const void *a, *b;  // bf16
	int64_t lda, ldb;
	int inner, outer, depth;
	void* out;  // bf16
	int64_t ldo;
	// scores
	const void* bias;  // {inner}, bf16, or null
	const int* targets;
	int first_inner;   // the vocabulary index of column 0
	float* stats;      // {outer, chunks}: maximum, sum
	int chunks;
	float* hit;
	const float *lse, *weight;
	// a gradient
	const float* scale;  // device, or null
	float factor;
	float* sum;  // {outer, inner}: what earlier pieces of the vocabulary add up to
	int sum_in, sum_out, first;
	int whole_words;  // out's rows start and end at multiples of 16 bytes (inner = ldo)
	const uint64_t* live;  // a bit for each depth, 64 to a word, where A's rows without it are to be left out (null: none)
	float* parts;  // {n, outer, inner}: sums of runs of the depth, where the grid takes it in n runs of part_depth
	int part_depth;
};

// Columns to a chunk of the statistics, by the outputs' size (the tile's choice).
int gemm16_chunk(int64_t inner, int64_t outer);
hipError_t gemm16_scores(const Gemm16Args& a, int epilogue, int chunk, hipStream_t s);
// A gradient: A's depth is its row axis; B's too where b_tr.
hipError_t gemm16_out(const Gemm16Args& a, bool b_tr, hipStream_t s);
// Floats of a.parts that such a product takes.
size_t gemm16_parts_floats(int64_t inner, int64_t outer, int64_t depth);

// rows x cols elements into rows of ldd (zeros behind cols).
hipError_t pack16(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, hipStream_t s);

// lse and losses from the chunks' statistics (stats {rows, chunks}, hit {rows}); 0 for a row without a target. A target that
// the vocabulary does not have makes its loss NaN.
hipError_t ce_join(const float* stats, int chunks, const float* hit, const int* targets, int64_t rows, int64_t vocab, float* lse,
                   float* loss, hipStream_t s);
// The same over whole rows of fp32 scores z {rows, cols} (columns first .. of the vocabulary), joined to what running {rows, 3}
// (maximum, sum, target's z) holds where `more`; the last piece writes lse and loss.
hipError_t ce_rows32(const float* z, int64_t rows, int64_t cols, int64_t first, int64_t vocab, const int* targets, float* running,
                     bool more, bool last, float* lse, float* loss, hipStream_t s);
// z {rows, cols} into dz in place, fp32; and (xs not null) x {rows, D} into xs, zeros for the rows without a weight.
hipError_t ce_grad32(float* z, int64_t rows, int64_t cols, int64_t first, const int* targets, const float* lse, const float* weight,
                     const float* scale, const float* x, float* xs, int64_t D, hipStream_t s);
// exp(z - the chunk's maximum) into dz in place, bf16, rows of ldz.
hipError_t ce_grad16(void* z, int64_t ldz, int64_t rows, int64_t vocab, const float* stats, int chunks, int chunk, const int* targets,
                     const float* lse, const float* hit, const float* weight, hipStream_t s);
// Per-row factors of dz and, of a mean or sum, the loss and the gradients' common factor. reduction: 0 none, 1 mean, 2 sum.
//   weight[i]: 0 for a row without a target, else 1 (none: g[i]); live: a bit for each row, whether it has one
//   factor: 1 (none), g / count (mean; 0 without targets), g (sum); g null: 1
//   total: the mean or sum of loss (null: not wanted; mean of nothing is NaN)
hipError_t ce_reduce(const float* loss, const int* targets, int64_t rows, int64_t vocab, int reduction, const float* g, float* total,
                     float* weight, uint64_t* live, float* factor, hipStream_t s);
// db (+)= factor * column sums of dz {rows, cols}, rows of ld; type 0 fp32, 1 bf16.
hipError_t ce_bias(const void* dz, int64_t ld, int64_t rows, int64_t cols, int type, const float* factor, void* db, bool first, float* partial,
                   hipStream_t s);
size_t ce_bias_partial_floats(int64_t rows, int64_t cols);

}  // namespace nnh
