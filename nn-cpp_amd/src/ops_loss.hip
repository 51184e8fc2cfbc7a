// ops_loss.hip - extern "C" entry points of the linear head's softmax cross entropy (include/nnh.h).
//
// Scores are made in pieces of the vocabulary and never kept: the forward keeps their statistics (bf16: they never leave the
// product's kernel), the backward makes a piece again, turns it into its gradient in scratch and takes the piece's part of dx
// and all of its dw and db from that, four products in all. The two in one call (train) make the scores once where all of
// them fit kKeep bytes of scratch, three products: bf16 keeps exp(z - its chunk's maximum), fp32 the scores.
//
// bf16's dz is rounded to bf16, the products' operand type (their sums and the common factor are fp32); train rounds what it keeps
// too, so that a probability in dz has two roundings there where backward gives it one. The target's element is made from its own
// score, not from what was kept: near a probability of 1 its difference from 1 is all of it. Against 64 bits the gradients of 4096 rows
// and 50257 words are off by 0.0017 of their norm, as fp32 products rounded once are.
//
// Scratch: a piece takes kPiece bytes, or 256 words' scores where these are more (from 2^20 rows on in fp32, 2^21 in bf16: rows are
// not cut); fp32 gradients add a copy of x, bf16 ones of several pieces a sum of dx.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "abi_common.hpp"
#include "kernels/hip/gemm.hpp"
#include "kernels/hip/linear_cross_entropy.hpp"
#include "scratch.hpp"
#include "nnh.h"

using namespace nnh;

namespace {

constexpr uint64_t kPiece = (uint64_t)1 << 30, kKeep = (uint64_t)4 << 30;  // bytes of scores in scratch
constexpr uint64_t kMaxBlocks = (1u << 23) - 1;                            // of 512 work-items, below 2^32 together

enum Call { kForward = 0, kBackward = 1, kTrain = 2 };

struct Head {
	int type;
	const void *x, *w, *bias;
	const int* targets;
	size_t rows, D, V;
	size_t size() const { return type == NNH_F32 ? 4 : 2; }
};

// Where a call's scratch lies, and how the vocabulary is cut.
struct Plan {
	bool keep = false;
	int64_t piece = 0, pieces = 1, ldz = 0, ldx = 0;  // ldx: D, or the packed row
	int chunk = 0, chunks = 0;
	int64_t part = 0;  // floats of the fp32 products' depth-cut partials
	size_t z = 0, stats = 0, hit = 0, running = 0, loss = 0, lse = 0, weight = 0, factor = 0, sum = 0, bias = 0, px = 0, pw = 0, partials = 0, parts = 0, live = 0, xs = 0, total = 0;
};

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

Plan plan_of(const Head& h, Call call, bool pack_x, bool pack_w) {
	Plan p;
	WorkspacePlan ws;
	const int64_t rows = (int64_t)h.rows, V = (int64_t)h.V, D = (int64_t)h.D, size = (int64_t)h.size();
	p.keep = call == kTrain && (uint64_t)rows * up(V, 64) * size <= kKeep;
	p.piece = p.keep ? V : std::min<int64_t>(V, std::max<int64_t>(256, (int64_t)(kPiece / size) / std::max<int64_t>(rows, 1) / 256 * 256));
	p.pieces = (V + p.piece - 1) / p.piece;
	p.ldx = up(D, 8);
	const bool forward = call != kBackward, backward = call != kForward;
	if (h.type == NNH_F32) {
		p.ldz = p.piece;
		p.z = ws.add((size_t)(rows * p.ldz) * 4);
		if (forward && p.pieces > 1) p.running = ws.add((size_t)rows * 12);
		const auto need = [&](int64_t m, int64_t n, int64_t k) { p.part = std::max(p.part, gemm_workspace_floats(m, n, k, 1)); };
		for (const int64_t cols : {p.piece, V - (p.pieces - 1) * p.piece}) {
			need(rows, cols, D);
			if (backward) {
				need(cols, D, rows);
				need(rows, D, cols);
			}
		}
		p.partials = ws.add((size_t)p.part * 4);
	} else {
		p.ldz = up(p.piece, 64);
		if (backward) p.z = ws.add((size_t)(rows * p.ldz) * 2);
		if (forward) {
			p.chunk = gemm16_chunk(V, rows);
			p.chunks = (int)((V + p.chunk - 1) / p.chunk);
			p.stats = ws.add((size_t)(rows * p.chunks) * 8);
			p.hit = ws.add((size_t)rows * 4);
		}
		if (backward && p.pieces > 1) p.sum = ws.add((size_t)(rows * D) * 4);
		size_t parts = 0;
		for (const int64_t cols : {p.piece, V - (p.pieces - 1) * p.piece})
			if (backward) parts = std::max({parts, gemm16_parts_floats(D, rows, cols), gemm16_parts_floats(D, cols, rows)});
		p.parts = ws.add(parts * 4);
		if (pack_x) p.px = ws.add((size_t)(rows * p.ldx) * 2);
		if (pack_w) p.pw = ws.add((size_t)(V * p.ldx) * 2);
	}
	if (forward) p.loss = ws.add((size_t)rows * 4);
	if (call == kTrain) p.lse = ws.add((size_t)rows * 4);
	if (backward) {
		p.weight = ws.add((size_t)rows * 4);
		p.live = ws.add((size_t)((rows + 63) / 64) * 8);
		if (h.type == NNH_F32) p.xs = ws.add((size_t)(rows * D) * 4);
		p.factor = ws.add(4);
		p.bias = ws.add(std::max(ce_bias_partial_floats(rows, p.piece), ce_bias_partial_floats(rows, V - (p.pieces - 1) * p.piece)) * 4);
	}
	p.total = ws.total;
	return p;
}

int check_head(const Head& h, int reduction) {
	if (h.type != NNH_F32 && h.type != NNH_BF16) return fail(NNH_ERR_INVALID, "linear cross entropy: no such element type");
	if (reduction < NNH_REDUCE_NONE || reduction > NNH_REDUCE_SUM) return fail(NNH_ERR_INVALID, "linear cross entropy: no such reduction");
	if (h.V == 0 || h.D == 0) return fail(NNH_ERR_SHAPE, "linear cross entropy: the vocabulary and the rows must not be empty");
	const size_t lim = (size_t)1 << 31;
	if (h.rows >= lim - 256 || h.V >= lim - 256 || h.D >= lim - 256 || !count_ok({h.rows, h.D}) || !count_ok({h.V, h.D}) || !count_ok({h.rows, h.V}))
		return fail(NNH_ERR_INVALID, "linear cross entropy: size out of range");
	const uint64_t r = (h.rows + 127) / 128, v = (h.V + 127) / 128, d = (h.D + 127) / 128;
	if (r * v > kMaxBlocks || r * d > kMaxBlocks || v * d > kMaxBlocks || h.rows > ((size_t)1 << 24) - 1)
		return fail(NNH_ERR_INVALID, "linear cross entropy: size out of range");
	return NNH_OK;
}

int check_inputs(const Head& h, std::initializer_list<const void*> words) {
	if (!h.w || (h.rows > 0 && (!h.x || !h.targets))) return fail(NNH_ERR_INVALID, "linear cross entropy: null pointer");
	for (const void* p : {h.x, h.w, h.bias})
		if (reinterpret_cast<uintptr_t>(p) % h.size() != 0) return fail(NNH_ERR_INVALID, "linear cross entropy: a pointer is not aligned to its elements");
	if (off_words({h.targets}) || off_words(words)) return fail(NNH_ERR_INVALID, "linear cross entropy: a pointer is not aligned to its elements");
	return NNH_OK;
}

struct Range {
	const void* p;
	uint64_t bytes;
};

int check_apart(const std::vector<Range>& outs, const std::vector<Range>& ins) {
	for (size_t i = 0; i < outs.size(); ++i) {
		for (const Range& x : ins)
			if (ranges_overlap(outs[i].p, outs[i].bytes, x.p, x.bytes)) return fail(NNH_ERR_ALIAS, "linear cross entropy: an output overlaps an input");
		for (size_t j = 0; j < i; ++j)
			if (ranges_overlap(outs[i].p, outs[i].bytes, outs[j].p, outs[j].bytes)) return fail(NNH_ERR_ALIAS, "linear cross entropy: two outputs overlap");
	}
	return NNH_OK;
}

std::vector<Range> inputs_of(const Head& h) {
	const uint64_t s = h.size();
	return {{h.x, h.rows * h.D * s}, {h.w, h.V * h.D * s}, {h.bias, h.V * s}, {h.targets, h.rows * 4}};
}

bool packed(const Head& h, const void* p) { return h.type == NNH_BF16 && (h.D % 8 != 0 || reinterpret_cast<uintptr_t>(p) % 16 != 0); }

struct Gradients {
	const float* g;
	void* dx;
	int dx_first;
	void* dw;
	int dw_first;
	void* db;
	int db_first;
};

// One call's work.
struct Run {
	Head h;
	Plan p;
	int reduction;
	const Scratch& ws;
	hipStream_t s;
	const void *x, *w;  // as the products read them
	int64_t ldx, ldw;

	int begin() {
		x = h.x;
		w = h.w;
		ldx = ldw = (int64_t)h.D;
		hipError_t e = hipSuccess;
		if (packed(h, h.x) && h.rows) {
			ldx = p.ldx;
			x = ws.at<void>(p.px);
			e = pack16(h.x, (int64_t)h.D, ws.at<void>(p.px), ldx, (int64_t)h.rows, (int64_t)h.D, s);
		}
		if (e == hipSuccess && packed(h, h.w)) {
			ldw = p.ldx;
			w = ws.at<void>(p.pw);
			e = pack16(h.w, (int64_t)h.D, ws.at<void>(p.pw), ldw, (int64_t)h.V, (int64_t)h.D, s);
		}
		return hip_status(e, "linear cross entropy");
	}

	int64_t cols(int64_t piece) const { return std::min(p.piece, (int64_t)h.V - piece * p.piece); }

	int product32(int ta, int tb, size_t m, size_t n, size_t k, const float* a, size_t lda, const float* b, size_t ldb, float* c, int acc,
	              const float* bias) {
		nnh_epilogue ep{bias ? NNH_BIAS_COL : NNH_BIAS_NONE, 0, bias, nullptr};
		GemmCall g;
		const int rc = build_gemm(ta, tb, m, n, k, a, lda, b, ldb, c, n, acc, nullptr, &ep, g);
		if (rc != NNH_OK) return rc;
		return hip_status(gemm_launch(g, s, -1, ws.at<float>(p.partials)), "linear cross entropy");
	}
	int scores32(int64_t piece) {
		const size_t from = (size_t)(piece * p.piece), n = (size_t)cols(piece);
		return product32(0, 1, h.rows, n, h.D, (const float*)h.x, h.D, (const float*)h.w + from * h.D, h.D, ws.at<float>(p.z), 0,
		                 h.bias ? (const float*)h.bias + from : nullptr);
	}
	Gemm16Args scores16(int64_t from, int64_t n) const {
		Gemm16Args a{};
		a.a = (const uint16_t*)w + from * ldw;
		a.b = x;
		a.lda = ldw;
		a.ldb = ldx;
		a.inner = (int)n;
		a.outer = (int)h.rows;
		a.depth = (int)p.ldx;
		if (!packed(h, h.x) || !packed(h, h.w)) a.depth = (int)h.D;  // a multiple of 8 then
		a.bias = h.bias ? (const uint16_t*)h.bias + from : nullptr;
		a.targets = h.targets;
		a.first_inner = (int)from;
		return a;
	}

	int whole(const void* out) const { return h.D % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0; }

	// lse and each row's loss; with p.keep the scores stay in scratch.
	int forward(float* lse, float* loss) {
		if (h.rows == 0) return NNH_OK;
		const int64_t rows = (int64_t)h.rows, V = (int64_t)h.V;
		if (h.type == NNH_F32) {
			for (int64_t i = 0; i < p.pieces; ++i) {
				const int rc = scores32(i);
				if (rc != NNH_OK) return rc;
				const hipError_t e = ce_rows32(ws.at<float>(p.z), rows, cols(i), i * p.piece, V, h.targets, ws.at<float>(p.running), i > 0,
				                               i + 1 == p.pieces, lse, loss, s);
				if (e != hipSuccess) return hip_status(e, "linear cross entropy");
			}
			return NNH_OK;
		}
		Gemm16Args a = scores16(0, V);  // all of the vocabulary: only statistics leave the product (or, kept, one piece is all)
		a.stats = ws.at<float>(p.stats);
		a.chunks = p.chunks;
		a.hit = ws.at<float>(p.hit);
		a.out = p.keep ? ws.at<void>(p.z) : nullptr;
		a.ldo = p.ldz;
		hipError_t e = gemm16_scores(a, p.keep ? kGemm16Keep : kGemm16Stats, p.chunk, s);
		if (e == hipSuccess) e = ce_join(a.stats, p.chunks, a.hit, h.targets, rows, V, lse, loss, s);
		return hip_status(e, "linear cross entropy");
	}

	// The gradients, weight and factor being in scratch.
	int backward(const float* lse, const Gradients& d) {
		const int64_t rows = (int64_t)h.rows, D = (int64_t)h.D;
		const float *weight = ws.at<float>(p.weight), *factor = ws.at<float>(p.factor);
		for (int64_t i = 0; i < p.pieces; ++i) {
			const int64_t from = i * p.piece, n = cols(i);
			hipError_t e = hipSuccess;
			if (h.type == NNH_F32) {
				float *const z = ws.at<float>(p.z), *const xs = ws.at<float>(p.xs);
				int rc = p.keep ? NNH_OK : scores32(i);
				if (rc == NNH_OK) rc = hip_status(ce_grad32(z, rows, n, from, h.targets, lse, weight, factor, (const float*)h.x, d.dw && i == 0 ? xs : nullptr, D, s), "linear cross entropy");
				if (rc == NNH_OK && d.dx && rows)
					rc = product32(0, 0, h.rows, h.D, (size_t)n, z, (size_t)n, (const float*)h.w + from * D, h.D, (float*)d.dx, i > 0 || !d.dx_first, nullptr);
				if (rc == NNH_OK && d.dw)
					rc = product32(1, 0, (size_t)n, h.D, h.rows, z, (size_t)n, xs, h.D, (float*)d.dw + from * D, !d.dw_first, nullptr);
				if (rc != NNH_OK) return rc;
				if (d.db) e = ce_bias(z, n, rows, n, 0, nullptr, (float*)d.db + from, d.db_first != 0, ws.at<float>(p.bias), s);
			} else {
				void* const z = ws.at<void>(p.z);
				if (rows && p.keep) {
					e = ce_grad16(z, p.ldz, rows, (int64_t)h.V, ws.at<float>(p.stats), p.chunks, p.chunk, h.targets, lse, ws.at<float>(p.hit), weight, s);
				} else if (rows) {
					Gemm16Args a = scores16(from, n);
					a.lse = lse;
					a.weight = weight;
					a.out = z;
					a.ldo = p.ldz;
					e = gemm16_scores(a, kGemm16Grad, gemm16_chunk(n, rows), s);
				}
				Gemm16Args o{};
				o.inner = (int)D;
				o.scale = factor;
				o.factor = 1.0f;
				o.ldo = D;
				o.parts = ws.at<float>(p.parts);
				if (e == hipSuccess && d.dx && rows) {
					Gemm16Args a = o;  // dx = dz w
					a.a = (const uint16_t*)w + from * ldw;
					a.lda = ldw;
					a.b = z;
					a.ldb = p.ldz;
					a.outer = (int)rows;
					a.depth = (int)n;
					a.out = d.dx;
					a.first = d.dx_first;
					a.sum = ws.at<float>(p.sum);
					a.sum_in = i > 0;
					a.sum_out = i + 1 < p.pieces;
					a.whole_words = whole(a.out);
					e = gemm16_out(a, false, s);
				}
				if (e == hipSuccess && d.dw) {
					Gemm16Args a = o;  // dw = dz^T x
					a.a = x;
					a.lda = ldx;
					a.b = z;
					a.ldb = p.ldz;
					a.outer = (int)n;
					a.depth = (int)rows;
					a.out = (uint16_t*)d.dw + from * D;
					a.first = d.dw_first;
					a.live = ws.at<uint64_t>(p.live);
					a.whole_words = whole(a.out);
					e = gemm16_out(a, true, s);
				}
				if (e == hipSuccess && d.db) e = ce_bias(z, p.ldz, rows, n, 1, factor, (uint16_t*)d.db + from, d.db_first != 0, ws.at<float>(p.bias), s);
			}
			if (e != hipSuccess) return hip_status(e, "linear cross entropy");
		}
		return NNH_OK;
	}
};

int check_gradients(const Head& h, const Gradients& d, std::vector<Range>& outs) {
	const uint64_t s = h.size();
	for (const void* p : {d.dx, d.dw, d.db})
		if (reinterpret_cast<uintptr_t>(p) % s != 0) return fail(NNH_ERR_INVALID, "linear cross entropy: a pointer is not aligned to its elements");
	outs.push_back({d.dx, h.rows * h.D * s});
	outs.push_back({d.dw, h.V * h.D * s});
	outs.push_back({d.db, h.V * s});
	return NNH_OK;
}

}  // namespace

extern "C" {

int nnh_linear_cross_entropy_workspace_size(int type, size_t rows, size_t D, size_t V, int call, int aligned, size_t* bytes) {
	return guarded([&] {
		Head h{type, nullptr, nullptr, nullptr, nullptr, rows, D, V};
		const int rc = check_head(h, NNH_REDUCE_NONE);
		if (rc != NNH_OK) return rc;
		if (call < kForward || call > kTrain) return fail(NNH_ERR_INVALID, "linear cross entropy: no such call");
		const bool pack = type == NNH_BF16 && (D % 8 != 0 || !aligned);
		return query_both_modes(bytes, [&](size_t* b) { return put_bytes(b, plan_of(h, (Call)call, pack, pack).total); });
	});
}

int nnh_linear_cross_entropy_forward(int type, const void* x, size_t rows, size_t D, const void* w, size_t V, const void* bias,
                                     const int* targets, int reduction, float* loss, float* lse, void* stream) {
	return guarded([&] {
		NumericsScope numerics_scope(stream);
		const Head h{type, x, w, bias, targets, rows, D, V};
		int rc = check_head(h, reduction);
		if (rc == NNH_OK) rc = check_inputs(h, {loss, lse});
		if (rc != NNH_OK) return rc;
		if ((!lse && rows) || (!loss && (rows || reduction != NNH_REDUCE_NONE))) return fail(NNH_ERR_INVALID, "linear cross entropy: null pointer");
		rc = check_apart({{loss, (reduction == NNH_REDUCE_NONE ? rows : 1) * 4}, {lse, rows * 4}}, inputs_of(h));
		if (rc != NNH_OK) return rc;
		if (rows == 0 && reduction == NNH_REDUCE_NONE) return NNH_OK;
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		const Plan p = plan_of(h, kForward, packed(h, x), packed(h, w));
		Scratch ws(s, p.total);
		if (ws.status() != NNH_OK) return ws.status();
		Run r{h, p, reduction, ws, s, nullptr, nullptr, 0, 0};
		rc = r.begin();
		float* const each = reduction == NNH_REDUCE_NONE ? loss : ws.at<float>(p.loss);
		if (rc == NNH_OK) rc = r.forward(lse, each);
		if (rc == NNH_OK && reduction != NNH_REDUCE_NONE)
			rc = hip_status(ce_reduce(each, targets, (int64_t)rows, (int64_t)V, reduction, nullptr, loss, nullptr, nullptr, nullptr, s), "linear cross entropy");
		return rc;
	});
}

int nnh_linear_cross_entropy_backward(int type, const float* g, const void* x, size_t rows, size_t D, const void* w, size_t V,
                                      const void* bias, const int* targets, const float* lse, int reduction, void* dx, int dx_first,
                                      void* dw, int dw_first, void* db, int db_first, void* stream) {
	return guarded([&] {
		NumericsScope numerics_scope(stream);
		const Head h{type, x, w, bias, targets, rows, D, V};
		const Gradients d{g, dx, dx_first, dw, dw_first, db, db_first};
		std::vector<Range> outs, ins = inputs_of(h);
		int rc = check_head(h, reduction);
		if (rc == NNH_OK) rc = check_inputs(h, {g, lse});
		if (rc == NNH_OK && rows && !lse) rc = fail(NNH_ERR_INVALID, "linear cross entropy: null pointer");
		if (rc == NNH_OK) rc = check_gradients(h, d, outs);
		ins.push_back({lse, rows * 4});
		ins.push_back({g, (reduction == NNH_REDUCE_NONE ? rows : 1) * 4});
		if (rc == NNH_OK) rc = check_apart(outs, ins);
		if (rc != NNH_OK || (!dx && !dw && !db)) return rc;
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		const Plan p = plan_of(h, kBackward, packed(h, x), packed(h, w));
		Scratch ws(s, p.total);
		if (ws.status() != NNH_OK) return ws.status();
		Run r{h, p, reduction, ws, s, nullptr, nullptr, 0, 0};
		rc = r.begin();
		if (rc == NNH_OK)
			rc = hip_status(ce_reduce(nullptr, targets, (int64_t)rows, (int64_t)V, reduction, g, nullptr, ws.at<float>(p.weight), ws.at<uint64_t>(p.live), ws.at<float>(p.factor), s),
			                "linear cross entropy");
		return rc == NNH_OK ? r.backward(lse, d) : rc;
	});
}

int nnh_linear_cross_entropy_train(int type, const float* g, const void* x, size_t rows, size_t D, const void* w, size_t V,
                                   const void* bias, const int* targets, int reduction, float* loss, void* dx, int dx_first, void* dw,
                                   int dw_first, void* db, int db_first, void* stream) {
	return guarded([&] {
		NumericsScope numerics_scope(stream);
		const Head h{type, x, w, bias, targets, rows, D, V};
		const Gradients d{g, dx, dx_first, dw, dw_first, db, db_first};
		std::vector<Range> outs, ins = inputs_of(h);
		int rc = check_head(h, reduction);
		if (rc == NNH_OK) rc = check_inputs(h, {g, loss});
		if (rc == NNH_OK && !loss && (rows || reduction != NNH_REDUCE_NONE)) rc = fail(NNH_ERR_INVALID, "linear cross entropy: null pointer");
		if (rc == NNH_OK) rc = check_gradients(h, d, outs);
		outs.push_back({loss, (reduction == NNH_REDUCE_NONE ? rows : 1) * 4});
		ins.push_back({g, (reduction == NNH_REDUCE_NONE ? rows : 1) * 4});
		if (rc == NNH_OK) rc = check_apart(outs, ins);
		if (rc != NNH_OK) return rc;
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		const Plan p = plan_of(h, kTrain, packed(h, x), packed(h, w));
		Scratch ws(s, p.total);
		if (ws.status() != NNH_OK) return ws.status();
		Run r{h, p, reduction, ws, s, nullptr, nullptr, 0, 0};
		rc = r.begin();
		float* const each = reduction == NNH_REDUCE_NONE ? loss : ws.at<float>(p.loss);
		float* const lse = ws.at<float>(p.lse);
		if (rc == NNH_OK) rc = r.forward(lse, each);
		if (rc == NNH_OK)
			rc = hip_status(ce_reduce(each, targets, (int64_t)rows, (int64_t)V, reduction, g, reduction == NNH_REDUCE_NONE ? nullptr : loss,
			                          ws.at<float>(p.weight), ws.at<uint64_t>(p.live), ws.at<float>(p.factor), s),
			                "linear cross entropy");
		return rc == NNH_OK ? r.backward(lse, d) : rc;
	});
}

}  // extern "C"
