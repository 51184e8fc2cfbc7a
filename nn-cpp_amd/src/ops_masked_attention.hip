// ops_masked_attention.hip - extern "C" entry points of masked attention (include/nnh.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "abi_common.hpp"
#include "kernels/hip/masked_attention.hpp"
#include "scratch.hpp"
#include "nnh.h"

using namespace nnh;

namespace {

constexpr size_t kMaxRows = (size_t)1 << 30;   // positions and their differences stay within an int
constexpr uint64_t kMaxBlocks = (1u << 24) - 1;  // of 256 work-items each, below 2^32 together

struct Geom {
	int type;
	size_t N, Tq, Tk, H, Hkv, Dh;
	size_t size() const { return type == kF32 ? 4 : 2; }
};

// One operand: {N, T, H, Dh} at its strides.
struct Operand {
	const nnh_head_tensor* t;
	size_t T, H;
	const char* name;
	uint64_t span = 0;  // elements from the first to the last, plus one
};

int check_geometry(const Geom& g) {
	if (g.type != NNH_F32 && g.type != NNH_BF16) return fail(NNH_ERR_INVALID, "masked attention: no such element type");
	if (g.H == 0 || g.Hkv == 0 || g.H % g.Hkv != 0 || g.Dh == 0)
		return fail(NNH_ERR_SHAPE, "masked attention: the key heads must divide the query heads, heads must not be empty");
	if (g.Dh > 128) return fail(NNH_ERR_INVALID, "masked attention: heads of more than 128 elements are not supported");
	uint64_t qb = 0, kb = 0;
	if (g.N > kMaxRows || g.Tq > kMaxRows || g.Tk > kMaxRows || g.H > kMaxRows ||
	    !count_ok({g.N, g.H, (g.Tq + 31) / 32}, qb) || !count_ok({g.N, g.Hkv, (g.Tk + 31) / 32}, kb) || qb > kMaxBlocks || kb > kMaxBlocks)
		return fail(NNH_ERR_INVALID, "masked attention: size out of range");
	return NNH_OK;
}

int check_operand(const Geom& g, Operand& o, bool output) {
	const std::string what = std::string("masked attention: ") + o.name;
	o.span = 0;
	if (g.N == 0 || o.T == 0) return NNH_OK;
	if (!o.t || !o.t->data) return fail(NNH_ERR_INVALID, what + " is null");
	if (reinterpret_cast<uintptr_t>(o.t->data) % g.size() != 0) return fail(NNH_ERR_INVALID, what + " is not aligned to its elements");
	const size_t sizes[3] = {g.N, o.T, o.H}, strides[3] = {o.t->sample, o.t->row, o.t->head};
	uint64_t last = 0;
	for (int d = 0; d < 3; ++d)
		if (strides[d] > kMaxElems || !mad_ok(sizes[d] - 1, strides[d], last, last)) return fail(NNH_ERR_INVALID, what + ": extent out of range");
	o.span = last + g.Dh;
	if (output) {  // every element has a place of its own
		int order[3] = {0, 1, 2};
		std::sort(order, order + 3, [&](int x, int y) { return strides[x] < strides[y]; });
		uint64_t inner = g.Dh;
		for (int x = 0; x < 3; ++x) {
			const int d = order[x];
			if (sizes[d] == 1) continue;
			if (strides[d] < inner) return fail(NNH_ERR_ALIAS, what + ": its elements overlap each other");
			inner += (sizes[d] - 1) * strides[d];
		}
	}
	return NNH_OK;
}

// What a 16-bit out lost in its rounding.
int check_rest(const Geom& g, Operand& o, bool output) {
	if (g.type == NNH_F32) return fail(NNH_ERR_INVALID, "masked attention: rest is for 16-bit types");
	return check_operand(g, o, output);
}

HeadStrides strides_of(const nnh_head_tensor* t) {
	return t ? HeadStrides{(int64_t)t->sample, (int64_t)t->row, (int64_t)t->head} : HeadStrides{0, 0, 0};
}

// Whether rows of the operand can be moved in 16-byte words.
bool wide(const Geom& g, const Operand& o) {
	if (!o.t || !o.span) return true;
	const size_t e = 16 / g.size();
	return reinterpret_cast<uintptr_t>(o.t->data) % 16 == 0 && o.t->sample % e == 0 && o.t->row % e == 0 && o.t->head % e == 0 &&
	       wide_row((int64_t)(o.t->row * g.size()));
}

int check_rule(const Geom& g, const nnh_attention_rule* r, MaskedAttentionArgs& a) {
	if (!r) return fail(NNH_ERR_INVALID, "masked attention: the rule is null");
	if (!(r->scale >= 0.0f) || !std::isfinite(r->scale) || !(r->cap >= 0.0f) || !std::isfinite(r->cap))
		return fail(NNH_ERR_INVALID, "masked attention: scale and cap must be finite and not negative");
	if (r->window > kMaxRows) return fail(NNH_ERR_INVALID, "masked attention: window out of range");
	const bool pairs = g.N > 0 && g.Tq > 0 && g.Tk > 0;  // else there is nothing to keep apart, and an empty side's array may be null
	if (pairs && !r->q_docs != !r->k_docs) return fail(NNH_ERR_INVALID, "masked attention: documents need both the queries' and the keys'");
	if (off_words({r->slopes, r->q_start, r->k_lens, r->prefix, r->q_docs, r->k_docs}))
		return fail(NNH_ERR_INVALID, "masked attention: an array of the rule is not aligned to its elements");
	a.scale = r->scale > 0.0f ? r->scale : 1.0f / std::sqrt((float)g.Dh);
	a.cap = r->cap;
	a.slopes = r->slopes;
	a.causal = r->causal ? 1 : 0;
	a.window = (int)r->window;
	a.q_start = r->q_start;
	a.k_lens = r->k_lens;
	a.prefix = r->prefix;
	a.q_docs = pairs ? r->q_docs : nullptr;
	a.k_docs = pairs ? r->k_docs : nullptr;
	a.N = (int)g.N;
	a.Tq = (int)g.Tq;
	a.Tk = (int)g.Tk;
	a.H = (int)g.H;
	a.Hkv = (int)g.Hkv;
	a.G = (int)(g.H / g.Hkv);
	a.dh = (int)g.Dh;
	return NNH_OK;
}

// A range of memory that a call reads or writes.
struct Range {
	const void* p;
	uint64_t bytes;
};

std::vector<Range> rule_ranges(const Geom& g, const MaskedAttentionArgs& a) {
	const uint64_t n = g.N * 4;
	return {{a.slopes, g.H * 4}, {a.q_start, n}, {a.k_lens, n}, {a.prefix, n}, {a.q_docs, n * g.Tq}, {a.k_docs, n * g.Tk}};
}

int check_apart(const std::vector<Range>& outs, const std::vector<Range>& ins) {
	for (const Range& o : outs)
		for (const Range& i : ins)
			if (ranges_overlap(o.p, o.bytes, i.p, i.bytes)) return fail(NNH_ERR_ALIAS, "masked attention: an output overlaps an input or another output");
	return NNH_OK;
}

Range range_of(const Geom& g, const Operand& o) { return {o.span ? o.t->data : nullptr, o.span * g.size()}; }

// Two gradients that share a buffer: rows of one stride, in places of their own (dq, dk and dv beside each other).
bool beside(const Geom& g, const Operand& x, const Operand& y) {
	if (!x.span || !y.span || !ranges_overlap(x.t->data, x.span * g.size(), y.t->data, y.span * g.size())) return true;
	if (x.t->row != y.t->row || x.t->sample != y.t->sample || x.t->row == 0 || x.t->sample % x.t->row != 0) return false;
	const intptr_t bytes = static_cast<const char*>(y.t->data) - static_cast<const char*>(x.t->data), row = (intptr_t)(x.t->row * g.size());
	if (bytes % (intptr_t)g.size() != 0) return false;
	const uint64_t off = (uint64_t)(((bytes % row) + row) % row) / g.size();
	const uint64_t sx = (x.H - 1) * x.t->head + g.Dh, sy = (y.H - 1) * y.t->head + g.Dh;
	return sx <= off && off + sy <= x.t->row;
}

struct Plan {
	size_t q_ranges = 0, k_ranges = 0, partial = 0, delta = 0, lse2 = 0, total = 0;
	int splits = 0, parts = 1;
};

Plan plan_of(const Geom& g, bool docs, bool backward) {
	Plan p;
	WorkspacePlan w;
	if (g.N == 0) return p;
	if (docs) {
		p.q_ranges = w.add(g.N * ((g.Tq + 63) / 64) * sizeof(DocRange));
		p.k_ranges = w.add(g.N * ((g.Tk + 63) / 64) * sizeof(DocRange));
	}
	if (backward) {
		p.delta = w.add(g.N * g.H * g.Tq * 4);
		p.lse2 = w.add(g.N * g.H * g.Tq * 4);
		p.parts = masked_attention_parts((int)g.N, (int)g.Tq, (int)g.Tk, (int)g.H, (int)g.Hkv);
		if (p.parts > 1) p.partial = w.add((size_t)p.parts * 2 * g.N * g.Hkv * g.Tk * ((g.Dh + 3) / 4 * 4) * 4);
	} else {
		p.splits = masked_attention_splits((int)g.N, (int)g.Tq, (int)g.Tk, (int)g.H, (int)g.Hkv);
		if (p.splits > 1) p.partial = w.add((size_t)p.splits * g.N * g.H * g.Tq * (g.Dh + 2) * 4);
	}
	p.total = w.total;
	return p;
}

int run_ranges(MaskedAttentionArgs& a, const Plan& p, const Scratch& ws, hipStream_t s) {
	if (!a.q_docs) return NNH_OK;
	DocRange* q = ws.at<DocRange>(p.q_ranges);
	DocRange* k = ws.at<DocRange>(p.k_ranges);
	hipError_t e = document_ranges(a.q_docs, a.N, a.Tq, q, s);
	const bool same = a.q_docs == a.k_docs && a.Tq == a.Tk;
	if (e == hipSuccess && !same) e = document_ranges(a.k_docs, a.N, a.Tk, k, s);
	a.q_ranges = q;
	a.k_ranges = same ? q : k;
	return hip_status(e, "masked attention");
}

}  // namespace

extern "C" {

int nnh_masked_attention_workspace_size(size_t N, size_t Tq, size_t Tk, size_t H, size_t Hkv, size_t Dh, int documents,
                                        int backward, size_t* bytes) {
	return guarded([&] {
		const Geom g{NNH_F32, N, Tq, Tk, H, Hkv, Dh};
		const int rc = check_geometry(g);
		return rc != NNH_OK ? rc : put_bytes(bytes, plan_of(g, documents != 0, backward != 0).total);
	});
}

int nnh_masked_attention_forward(int type, size_t N, size_t Tq, size_t Tk, size_t H, size_t Hkv, size_t Dh,
                                 const nnh_head_tensor* q, const nnh_head_tensor* k, const nnh_head_tensor* v,
                                 const nnh_attention_rule* rule, const nnh_head_tensor* out, const nnh_head_tensor* rest,
                                 float* lse, void* stream) {
	return guarded([&] {
		const Geom g{type, N, Tq, Tk, H, Hkv, Dh};
		MaskedAttentionArgs a{};
		int rc = check_geometry(g);
		if (rc == NNH_OK) rc = check_rule(g, rule, a);
		Operand in[3] = {{q, Tq, H, "q"}, {k, Tk, Hkv, "k"}, {v, Tk, Hkv, "v"}}, o{out, Tq, H, "out"}, lost{rest, Tq, H, "rest"};
		for (Operand& x : in)
			if (rc == NNH_OK) rc = check_operand(g, x, false);
		if (rc == NNH_OK) rc = check_operand(g, o, true);
		if (rc == NNH_OK && rest) rc = check_rest(g, lost, true);
		if (rc != NNH_OK) return rc;
		if (N == 0 || Tq == 0) return NNH_OK;
		if (!lse) return fail(NNH_ERR_INVALID, "masked attention: lse is null");
		if (off_words({lse})) return fail(NNH_ERR_INVALID, "masked attention: lse is not aligned to its elements");
		const Range stats{lse, (uint64_t)N * H * Tq * 4};
		std::vector<Range> ins = rule_ranges(g, a);
		for (const Operand& x : in) ins.push_back(range_of(g, x));
		rc = check_apart({range_of(g, o), range_of(g, lost), stats}, ins);
		if (rc == NNH_OK) rc = check_apart({stats}, {range_of(g, o), range_of(g, lost)});
		if (rc == NNH_OK) rc = check_apart({range_of(g, o)}, {range_of(g, lost)});
		if (rc != NNH_OK) return rc;
		a.q = q->data;
		a.k = Tk ? k->data : nullptr;
		a.v = Tk ? v->data : nullptr;
		a.out = out->data;
		a.lse = lse;
		a.qs = strides_of(q);
		a.ks = strides_of(k);
		a.vs = strides_of(v);
		a.os = strides_of(out);
		a.rest = rest ? rest->data : nullptr;
		a.rs = strides_of(rest);
		const bool vec = Dh * g.size() % 16 == 0 && wide(g, in[0]) && wide(g, in[1]) && wide(g, in[2]) && wide(g, o) && wide(g, lost);
		const Plan p = plan_of(g, a.q_docs != nullptr, false);
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		Scratch ws(s, p.total);
		if (ws.status() != NNH_OK) return ws.status();
		rc = run_ranges(a, p, ws, s);
		if (rc != NNH_OK) return rc;
		a.splits = p.splits;
		if (p.splits > 1) a.partial = ws.at<float>(p.partial);
		return hip_status(p.splits ? masked_attention_split(a, type, vec, s) : masked_attention_forward(a, type, vec, s), "masked attention");
	});
}

int nnh_masked_attention_backward(int type, size_t N, size_t Tq, size_t Tk, size_t H, size_t Hkv, size_t Dh,
                                  const nnh_head_tensor* g_, const nnh_head_tensor* q, const nnh_head_tensor* k,
                                  const nnh_head_tensor* v, const nnh_head_tensor* out, const nnh_head_tensor* rest, const float* lse,
                                  const nnh_attention_rule* rule, const nnh_head_tensor* dq, int dq_first,
                                  const nnh_head_tensor* dk, int dk_first, const nnh_head_tensor* dv, int dv_first,
                                  void* stream) {
	return guarded([&] {
		const Geom g{type, N, Tq, Tk, H, Hkv, Dh};
		MaskedAttentionArgs a{};
		int rc = check_geometry(g);
		if (rc == NNH_OK) rc = check_rule(g, rule, a);
		if (rc != NNH_OK) return rc;
		if (N == 0 || (!dq && !dk && !dv)) return NNH_OK;
		Operand in[5] = {{g_, Tq, H, "g"}, {q, Tq, H, "q"}, {k, Tk, Hkv, "k"}, {v, Tk, Hkv, "v"}, {out, Tq, H, "out"}}, lost{rest, Tq, H, "rest"};
		Operand grad[3] = {{dq, Tq, H, "dq"}, {dk, Tk, Hkv, "dk"}, {dv, Tk, Hkv, "dv"}};
		for (Operand& x : in)
			if (rc == NNH_OK) rc = check_operand(g, x, false);
		if (rc == NNH_OK && rest) rc = check_rest(g, lost, false);
		for (Operand& x : grad)
			if (rc == NNH_OK && x.t) rc = check_operand(g, x, true);
		if (rc != NNH_OK) return rc;
		if (Tq && !lse) return fail(NNH_ERR_INVALID, "masked attention: lse is null");
		if (off_words({lse})) return fail(NNH_ERR_INVALID, "masked attention: lse is not aligned to its elements");
		std::vector<Range> ins = rule_ranges(g, a), outs;
		for (const Operand& x : in) ins.push_back(range_of(g, x));
		ins.push_back({lse, (uint64_t)N * H * Tq * 4});
		ins.push_back(range_of(g, lost));
		for (const Operand& x : grad) outs.push_back(range_of(g, x));
		rc = check_apart(outs, ins);
		if (rc != NNH_OK) return rc;
		if (!beside(g, grad[0], grad[1]) || !beside(g, grad[0], grad[2]) || !beside(g, grad[1], grad[2]))
			return fail(NNH_ERR_ALIAS, "masked attention: two gradients overlap");
		auto data = [](const nnh_head_tensor* t) { return t ? t->data : nullptr; };
		a.q = data(q);
		a.k = data(k);
		a.v = data(v);
		a.g = data(g_);
		a.out = data(out);
		a.lse = const_cast<float*>(lse);
		a.dq = data(dq);
		a.dk = data(dk);
		a.dv = data(dv);
		a.qs = strides_of(q);
		a.ks = strides_of(k);
		a.vs = strides_of(v);
		a.gs = strides_of(g_);
		a.os = strides_of(out);
		a.rest = data(rest);
		a.rs = strides_of(rest);
		a.dqs = strides_of(dq);
		a.dks = strides_of(dk);
		a.dvs = strides_of(dv);
		a.dq_first = dq_first;
		a.dk_first = dk_first;
		a.dv_first = dv_first;
		bool vec = Dh * g.size() % 16 == 0 && wide(g, lost);
		for (const Operand& x : in) vec = vec && wide(g, x);
		for (const Operand& x : grad) vec = vec && wide(g, x);
		const Plan p = plan_of(g, a.q_docs != nullptr, true);
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		Scratch ws(s, p.total);
		if (ws.status() != NNH_OK) return ws.status();
		a.delta = ws.at<float>(p.delta);
		a.lse2 = ws.at<float>(p.lse2);
		a.parts = p.parts;
		a.partial = ws.at<float>(p.partial);
		rc = run_ranges(a, p, ws, s);
		if (rc != NNH_OK) return rc;
		return hip_status(masked_attention_backward(a, type, vec, s), "masked attention backward");
	});
}

}  // extern "C"
