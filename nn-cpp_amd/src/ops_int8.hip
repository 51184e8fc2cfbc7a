// ops_int8.hip - extern "C" entry points of linears in 8-bit integers (include/nnh.h).
#include <hip/hip_runtime.h>

#include "abi_common.hpp"
#include "kernels/hip/linear_int8.hpp"
#include "scratch.hpp"
#include "nnh.h"

using namespace nnh;

namespace {

constexpr uint64_t kMaxDim = (uint64_t)1 << 30;
constexpr uint64_t kMaxDepth = ((uint64_t)1 << 17) - 1;  // 128 * 128 * kMaxDepth is below 2^31
constexpr uint64_t kMaxBlocks = (1u << 24) - 1;          // of 256 work-items each, below 2^32 together

int refuse(int code, const char* what) { return fail(code, std::string("linear in 8 bits: ") + what); }
bool off(const void* p, uint64_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }
uint64_t size_of(int type) { return type == NNH_F32 ? 4 : 2; }
uint64_t up(uint64_t x, uint64_t to) { return (x + to - 1) / to * to; }
// Bytes from the first to the last element of some rows.
uint64_t extent(uint64_t rows, uint64_t row, uint64_t ld, uint64_t size) { return rows && row ? ((rows - 1) * ld + row) * size : 0; }

int check_matrix(const void* p, uint64_t rows, uint64_t row, uint64_t ld, uint64_t size, const char* what) {
	uint64_t x = 0;
	if (ld < row || ld > kMaxElems || !mad_ok(rows, ld, 0, x)) return refuse(NNH_ERR_INVALID, (std::string(what) + ": rows longer than their pitch, or an extent out of range").c_str());
	if (rows == 0 || row == 0) return NNH_OK;
	if (!p) return refuse(NNH_ERR_INVALID, (std::string(what) + " is null").c_str());
	if (off(p, size)) return refuse(NNH_ERR_INVALID, (std::string(what) + " is not aligned to its elements").c_str());
	return NNH_OK;
}

struct Plan {
	size_t codes = 0, scale = 0, parts = 0, total = 0;
	uint64_t pitch = 0;
	bool cut = false;
};
Plan plan_of(uint64_t rows, uint64_t D, uint64_t V) {
	Plan p;
	if (rows == 0 || V == 0 || linear_int8_whole((int64_t)rows, (int64_t)D)) return p;
	WorkspacePlan w;
	p.pitch = up(D, 64);
	p.codes = w.add(rows * p.pitch);
	p.scale = w.add(rows * 4);
	const size_t parts = linear_int8_parts((int64_t)rows, (int64_t)D, (int64_t)V);
	p.cut = parts > 0;
	if (p.cut) p.parts = w.add(parts * 4);
	p.total = w.total;
	return p;
}

int check_sizes(uint64_t rows, uint64_t D, uint64_t V) {
	if (rows > kMaxBlocks || V > kMaxBlocks || D > kMaxDepth)
		return refuse(NNH_ERR_INVALID, "size out of range (a depth of at most 131071 keeps the sums within 32 bits)");
	return NNH_OK;
}

}  // namespace

extern "C" {

int nnh_quantize_rows(int type, const void* x, size_t rows, size_t D, size_t ldx, signed char* codes, size_t ldc, float* scale, void* stream) {
	return guarded([&] {
		if (type != NNH_F32 && type != NNH_BF16) return refuse(NNH_ERR_INVALID, "no such element type");
		if (rows > kMaxBlocks || D > kMaxDim) return refuse(NNH_ERR_INVALID, "size out of range");
		int rc = check_matrix(x, rows, D, ldx, size_of(type), "x");
		if (rc == NNH_OK) rc = check_matrix(codes, rows, D, ldc, 1, "codes");
		if (rc != NNH_OK || rows == 0) return rc;
		if (!scale || off(scale, 4)) return refuse(NNH_ERR_INVALID, "the scales are null or not aligned to their elements");
		const uint64_t xb = extent(rows, D, ldx, size_of(type)), cb = extent(rows, D, ldc, 1);
		if (ranges_overlap(x, xb, codes, cb) || ranges_overlap(x, xb, scale, rows * 4) || ranges_overlap(codes, cb, scale, rows * 4))
			return refuse(NNH_ERR_ALIAS, "an output overlaps the input or the other output");
		const QuantizeArgs a{x, (int64_t)ldx, (int64_t)rows, (int)D, reinterpret_cast<int8_t*>(codes), (int64_t)ldc, (int)D, scale};
		return hip_status(quantize_rows(a, type, reinterpret_cast<hipStream_t>(stream)), "quantize rows");
	});
}

int nnh_linear_int8_workspace_size(size_t rows, size_t D, size_t V, size_t* bytes) {
	return guarded([&] {
		const int rc = check_sizes(rows, D, V);
		return rc != NNH_OK ? rc : put_bytes(bytes, plan_of(rows, D, V).total);
	});
}

int nnh_linear_int8(int type, const void* x, size_t rows, size_t D, size_t ldx, const signed char* w, size_t ldw, const float* w_scale, size_t V,
                    const void* bias, void* y, size_t ldy, void* stream) {
	return guarded([&] {
		if (type != NNH_F32 && type != NNH_BF16) return refuse(NNH_ERR_INVALID, "no such element type");
		int rc = check_sizes(rows, D, V);
		if (rc != NNH_OK) return rc;
		const uint64_t size = size_of(type);
		rc = check_matrix(x, rows, D, ldx, size, "x");
		if (rc == NNH_OK) rc = check_matrix(w, V, D, ldw, 1, "w");
		if (rc == NNH_OK) rc = check_matrix(y, rows, V, ldy, size, "y");
		if (rc != NNH_OK || rows == 0 || V == 0) return rc;
		if (D > 0 && (off(w, 16) || ldw % 16 != 0)) return refuse(NNH_ERR_INVALID, "the weight's rows must begin at multiples of 16 bytes");
		if (!w_scale || off(w_scale, 4)) return refuse(NNH_ERR_INVALID, "the weight's scales are null or not aligned to their elements");
		if (off(bias, size)) return refuse(NNH_ERR_INVALID, "the bias is not aligned to its elements");
		const uint64_t yb = extent(rows, V, ldy, size);
		if (ranges_overlap(y, yb, x, extent(rows, D, ldx, size)) || ranges_overlap(y, yb, w, D ? V * ldw : 0) || ranges_overlap(y, yb, w_scale, V * 4) ||
		    (bias && ranges_overlap(y, yb, bias, V * size)))
			return refuse(NNH_ERR_ALIAS, "y overlaps an input");
		const Plan p = plan_of(rows, D, V);
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		Scratch ws(s, p.total);
		if (ws.status() != NNH_OK) return ws.status();
		LinearInt8Args a{};
		if (linear_int8_whole((int64_t)rows, (int64_t)D)) {
			a.whole = 1;
			a.rows_in = x;
			a.ld_in = (int64_t)ldx;
			a.wide_in = !off(x, 16) && ldx * size % 16 == 0 && D % 8 == 0;
		} else {
			const QuantizeArgs q{x, (int64_t)ldx, (int64_t)rows, (int)D, ws.at<int8_t>(p.codes), (int64_t)p.pitch, (int)p.pitch, ws.at<float>(p.scale)};
			rc = hip_status(quantize_rows(q, type, s), "linear in 8 bits");
			if (rc != NNH_OK) return rc;
			a.x = q.codes;
			a.x_scale = q.scale;
		}
		a.w = reinterpret_cast<const int8_t*>(w);
		a.ldw = (int64_t)ldw;
		a.ldx = (int64_t)p.pitch;
		a.rows = (int)rows;
		a.D = (int)D;
		a.V = (int)V;
		a.w_scale = w_scale;
		a.bias = bias;
		a.y = y;
		a.ldy = (int64_t)ldy;
		a.whole_words = !off(y, 16) && ldy * size % 16 == 0 && V * size % 16 == 0;
		a.parts = p.cut ? ws.at<int>(p.parts) : nullptr;
		return hip_status(linear_int8(a, type, s), "linear in 8 bits");
	});
}

}  // extern "C"
