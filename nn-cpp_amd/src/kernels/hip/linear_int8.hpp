// linear_int8.hpp - a linear layer on 8-bit integers (internal to libnnh): rows quantised with a scale each, products summed in int32,
// y = sum * row scale * column scale + bias.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "masked_attention.hpp"

namespace nnh {

struct QuantizeArgs {
	const void* x;
	int64_t ldx;
	int64_t rows;
	int D;
	int8_t* codes;
	int64_t ldc;
	int pad;  // zeros are stored behind a row's codes up to here
	float* scale;
};

struct LinearInt8Args {
	const int8_t *w, *x;  // {V, D} and {rows, D}: rows that begin at multiples of 16 bytes, x's zero up to a multiple of 64
	int64_t ldw, ldx;
	int rows, D, V;
	const float *w_scale, *x_scale;
	const void* bias;  // {V} of y's type, or null
	void* y;
	int64_t ldy;
	int whole_words;  // y's rows can be stored in 16-byte words
	// the few rows' own form: rows to quantise (null where they have no elements), in the place of x and x_scale
	int whole;
	const void* rows_in;
	int64_t ld_in;
	int wide_in;      // they can be read in 16-byte words
	int* parts;       // {parts, rows, V}: sums of runs of the depth, or null
	int part_units;   // a run's depth, in units of 2 codes
};

// Whether a product takes the form for few rows, and whether that quantises them itself (whole).
bool linear_int8_few(int64_t rows, int64_t V);
bool linear_int8_whole(int64_t rows, int64_t D);
// Elements of LinearInt8Args::parts.
size_t linear_int8_parts(int64_t rows, int64_t D, int64_t V);

hipError_t quantize_rows(const QuantizeArgs& a, int type, hipStream_t s);
hipError_t linear_int8(const LinearInt8Args& a, int type, hipStream_t s);

}  // namespace nnh
