// ops_paged.hip - extern "C" entry points of the paged cache: new tokens into it, attention over it (include/nnh.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "abi_common.hpp"
#include "kernels/hip/paged_attention.hpp"
#include "scratch.hpp"
#include "nnh.h"

using namespace nnh;

namespace {

constexpr size_t kMost = (size_t)1 << 30;        // positions, rows and pages stay within an int
constexpr uint64_t kMaxBlocks = (1u << 24) - 1;  // of 256 work-items each, below 2^32 together

int refuse(int code, const char* what) { return fail(code, std::string("paged cache: ") + what); }

struct Range {
	const void* p;
	uint64_t bytes;
};

int check_apart(const std::vector<Range>& outs, const std::vector<Range>& ins) {
	for (const Range& o : outs)
		for (const Range& i : ins)
			if (ranges_overlap(o.p, o.bytes, i.p, i.bytes)) return refuse(NNH_ERR_ALIAS, "an output overlaps an input or another output");
	return NNH_OK;
}

// Elements of a head at some strides: their extent in elements, and whether each has a place of its own.
struct Layout {
	uint64_t span = 0;
	bool apart = true;
	uint64_t inner[4] = {0, 0, 0, 0}, stride[4] = {0, 0, 0, 0};  // by rising stride: what a step of that stride has to pass
	int levels = 0;
};

int layout_of(size_t dh, std::initializer_list<size_t> sizes, std::initializer_list<size_t> strides, Layout& l, const char* what) {
	std::vector<std::pair<uint64_t, uint64_t>> d;
	uint64_t last = 0;
	auto st = strides.begin();
	for (size_t n : sizes) {
		if (*st > kMaxElems || !mad_ok(n - 1, *st, last, last)) return refuse(NNH_ERR_INVALID, (std::string(what) + ": extent out of range").c_str());
		if (n > 1) d.push_back({*st, n});
		++st;
	}
	l.span = last + dh;
	std::sort(d.begin(), d.end());
	uint64_t inner = dh;
	for (const auto& x : d) {
		if (x.first < inner) l.apart = false;
		l.inner[l.levels] = inner;
		l.stride[l.levels++] = x.first;
		inner += (x.second - 1) * x.first;
	}
	return NNH_OK;
}

// Two buffers of one layout whose extents overlap but whose elements do not: keys and values side by side in a page, a slot or a head.
bool side_by_side(const Layout& l, const void* x, const void* y, uint64_t size) {
	const char *p = static_cast<const char*>(x), *q = static_cast<const char*>(y);
	if (!ranges_overlap(p, l.span * size, q, l.span * size)) return true;
	const uint64_t bytes = p < q ? q - p : p - q;
	if (bytes % size != 0) return false;
	for (int i = 0; i < l.levels; ++i)
		if (bytes / size >= l.inner[i] && bytes / size + l.inner[i] <= l.stride[i]) return true;
	return false;
}

uint64_t size_of(int type) { return type == NNH_F32 ? 4 : 2; }

bool off(const void* p, uint64_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

// What both calls are given.
struct Call {
	int type;
	size_t N, rows, Hkv, Dh;
	const nnh_paged_cache* cache;
	const int *starts, *lens;
	Layout pages;
	bool any_page() const { return cache->pages > 0 && cache->width > 0; }
	uint64_t keys() const { return (uint64_t)cache->width * cache->page_size; }
	std::vector<Range> lists() const { return {{starts, (N + 1) * 4}, {lens, N * 4}, {cache->table, N * cache->width * 4}}; }
	Range k() const { return {any_page() ? cache->k : nullptr, pages.span * size_of(type)}; }
	Range v() const { return {any_page() ? cache->v : nullptr, pages.span * size_of(type)}; }
};

int check_call(Call& c) {
	if (c.type != NNH_F32 && c.type != NNH_BF16) return refuse(NNH_ERR_INVALID, "no such element type");
	if (!c.cache) return refuse(NNH_ERR_INVALID, "the cache is null");
	if (c.Hkv == 0 || c.Dh == 0 || c.cache->page_size == 0) return refuse(NNH_ERR_SHAPE, "heads and pages must not be empty");
	uint64_t x = 0;
	if (c.N >= kMost || c.rows > kMost || c.cache->pages > kMost || c.Hkv > kMost || c.Dh > kMost || !count_ok({c.cache->width, c.cache->page_size}, x) ||
	    c.cache->width > kMost || c.cache->page_size > kMost || x > kMost || !count_ok({c.N, c.cache->width}, x))
		return refuse(NNH_ERR_INVALID, "size out of range");
	if (c.N == 0 || c.rows == 0) return NNH_OK;
	if (!c.starts || !c.lens) return refuse(NNH_ERR_INVALID, "starts and lens are needed");
	if (off_words({c.starts, c.lens, c.cache->table})) return refuse(NNH_ERR_INVALID, "an array is not aligned to its elements");
	if (!c.any_page()) return NNH_OK;
	if (!c.cache->table || !c.cache->k || !c.cache->v) return refuse(NNH_ERR_INVALID, "the cache's pages or its table are null");
	if (off(c.cache->k, size_of(c.type)) || off(c.cache->v, size_of(c.type))) return refuse(NNH_ERR_INVALID, "a page is not aligned to its elements");
	return layout_of(c.Dh, {c.cache->pages, c.cache->page_size, c.Hkv}, {c.cache->page, c.cache->slot, c.cache->head}, c.pages, "the pages");
}

// Packed rows {rows, heads, Dh} at their strides.
int check_rows(const Call& c, const nnh_head_tensor* t, size_t heads, const char* name, bool output, Layout& l) {
	const std::string what = name;
	if (!t || !t->data) return refuse(NNH_ERR_INVALID, (what + " is null").c_str());
	if (off(t->data, size_of(c.type))) return refuse(NNH_ERR_INVALID, (what + " is not aligned to its elements").c_str());
	const int rc = layout_of(c.Dh, {c.rows, heads}, {t->row, t->head}, l, name);
	if (rc == NNH_OK && output && !l.apart) return refuse(NNH_ERR_ALIAS, (what + ": its elements overlap each other").c_str());
	return rc;
}

Range range_of(const Call& c, const nnh_head_tensor* t, const Layout& l) { return {t->data, l.span * size_of(c.type)}; }

// Whether everything can be moved in 16-byte words.
bool wide_strides(uint64_t size, const void* p, std::initializer_list<size_t> strides) {
	bool w = reinterpret_cast<uintptr_t>(p) % 16 == 0;
	for (size_t s : strides) w = w && s * size % 16 == 0;
	return w;
}
bool wide(const Call& c) {
	const uint64_t s = size_of(c.type);
	return c.Dh * s % 16 == 0 && wide_strides(s, c.cache->k, {c.cache->page, c.cache->slot, c.cache->head}) && reinterpret_cast<uintptr_t>(c.cache->v) % 16 == 0;
}
bool wide(const Call& c, const nnh_head_tensor* t) { return wide_strides(size_of(c.type), t->data, {t->row, t->head}); }

PageTable table_of(const Call& c) {
	const nnh_paged_cache& k = *c.cache;
	return {k.table, (int64_t)k.page, (int64_t)k.slot, (int64_t)k.head, make_fastdiv((unsigned)k.page_size), c.any_page() ? (int)k.pages : 0, (int)k.width};
}

HeadStrides strides_of(const nnh_head_tensor* t) { return {0, (int64_t)t->row, (int64_t)t->head}; }

int check_blocks(size_t N, size_t rows, size_t most, size_t H, size_t Hkv) {
	uint64_t x = 0;
	if (H > kMost || Hkv > kMost || H == 0 || Hkv == 0 || H % Hkv != 0) return refuse(NNH_ERR_SHAPE, "the key heads must divide the query heads, heads must not be empty");
	// (workgroups: a group of 32 columns or more each, two to a sequence more at most, and the 512 that the keys are divided for)
	if (most > kMost || !count_ok({rows, H}, x) || x > 4 * kMaxBlocks || !count_ok({2 * N + 1024, Hkv}, x) || x > kMaxBlocks / 2)
		return refuse(NNH_ERR_INVALID, "size out of range");
	return NNH_OK;
}

struct Room {
	PagedPlan plan;
	size_t split = 0, wide = 0, total = 0;
	Room(size_t N, size_t rows, size_t most, size_t keys, size_t H, size_t Hkv, size_t Dh) : plan(paged_attention_plan(N, rows, most, keys, (int)H, (int)Hkv, (int)Dh)) {
		WorkspacePlan w;
		split = w.add(plan.split_floats * 4);
		wide = w.add(plan.wide_floats * 4);
		total = w.total;
	}
};

}  // namespace

extern "C" {

int nnh_paged_append(int type, size_t N, size_t rows, size_t Hkv, size_t Dh, const nnh_head_tensor* k, const nnh_head_tensor* v,
                     const int* starts, const int* lens, const nnh_paged_cache* cache, void* stream) {
	return guarded([&] {
		Call c{type, N, rows, Hkv, Dh, cache, starts, lens, {}};
		int rc = check_call(c);
		if (rc != NNH_OK) return rc;
		uint64_t x = 0;
		if (rows > 4 * kMaxBlocks || !count_ok({Hkv, Dh}, x) || x > kMost) return refuse(NNH_ERR_INVALID, "size out of range");
		if (N == 0 || rows == 0) return NNH_OK;
		Layout kl, vl;
		rc = check_rows(c, k, Hkv, "k", false, kl);
		if (rc == NNH_OK) rc = check_rows(c, v, Hkv, "v", false, vl);
		if (rc != NNH_OK || !c.any_page()) return rc;
		if (!c.pages.apart || !side_by_side(c.pages, cache->k, cache->v, size_of(type))) return refuse(NNH_ERR_ALIAS, "the pages overlap each other");
		std::vector<Range> ins = c.lists();
		ins.push_back(range_of(c, k, kl));
		ins.push_back(range_of(c, v, vl));
		rc = check_apart({c.k(), c.v()}, ins);
		if (rc != NNH_OK) return rc;
		PagedAppendArgs a{};
		a.k = k->data;
		a.v = v->data;
		a.ks = strides_of(k);
		a.vs = strides_of(v);
		a.k_pages = cache->k;
		a.v_pages = cache->v;
		a.t = table_of(c);
		a.s = {starts, lens, (int)N, (int)rows};
		a.Hkv = (int)Hkv;
		a.dh = (int)Dh;
		return hip_status(paged_append(a, type, wide(c) && wide(c, k) && wide(c, v), reinterpret_cast<hipStream_t>(stream)), "paged append");
	});
}

int nnh_paged_attention_workspace_size(size_t N, size_t rows, size_t most, size_t keys, size_t H, size_t Hkv, size_t Dh, size_t* bytes) {
	return guarded([&] {
		const int rc = check_blocks(N, rows, most, H, Hkv);
		if (rc != NNH_OK) return rc;
		if (keys > kMost || N >= kMost || rows > kMost || Dh > 128) return refuse(NNH_ERR_INVALID, "size out of range");
		return put_bytes(bytes, Room(N, rows, most, keys, H, Hkv, Dh).total);
	});
}

int nnh_paged_attention(int type, size_t N, size_t rows, size_t most, size_t H, size_t Hkv, size_t Dh, const nnh_head_tensor* q,
                        const nnh_paged_cache* cache, const int* starts, const nnh_attention_rule* rule, const nnh_head_tensor* out,
                        float* lse, void* stream) {
	return guarded([&] {
		if (!rule) return refuse(NNH_ERR_INVALID, "the rule is null");
		Call c{type, N, rows, Hkv, Dh, cache, starts, rule->k_lens, {}};
		int rc = check_blocks(N, rows, most, H, Hkv);
		if (rc == NNH_OK) rc = check_call(c);
		if (rc != NNH_OK) return rc;
		if (Dh > 128) return refuse(NNH_ERR_INVALID, "heads of more than 128 elements are not supported");
		if (rule->q_start || rule->q_docs || rule->k_docs) return refuse(NNH_ERR_INVALID, "positions come from starts and k_lens, and a sequence is one document");
		if (!(rule->scale >= 0.0f) || !std::isfinite(rule->scale) || !(rule->cap >= 0.0f) || !std::isfinite(rule->cap) || rule->window > kMost)
			return refuse(NNH_ERR_INVALID, "scale, cap and window must be finite and not negative");
		if (off_words({rule->slopes, rule->prefix, lse})) return refuse(NNH_ERR_INVALID, "an array is not aligned to its elements");
		if (N == 0 || rows == 0 || most == 0) return NNH_OK;
		if (!lse) return refuse(NNH_ERR_INVALID, "lse is null");
		Layout ql, ol;
		rc = check_rows(c, q, H, "q", false, ql);
		if (rc == NNH_OK) rc = check_rows(c, out, H, "out", true, ol);
		if (rc != NNH_OK) return rc;
		const Range o = range_of(c, out, ol), stats{lse, (uint64_t)rows * H * 4};
		std::vector<Range> ins = c.lists();
		for (const Range& r : {range_of(c, q, ql), c.k(), c.v(), Range{rule->slopes, H * 4}, Range{rule->prefix, N * 4}}) ins.push_back(r);
		rc = check_apart({o, stats}, ins);
		if (rc == NNH_OK) rc = check_apart({o}, {stats});
		if (rc != NNH_OK) return rc;
		PagedAttentionArgs p{};
		MaskedAttentionArgs& a = p.a;
		a.q = q->data;
		a.k = cache->k;
		a.v = cache->v;
		a.out = out->data;
		a.qs = strides_of(q);
		a.os = strides_of(out);
		a.N = (int)N;
		a.H = (int)H;
		a.Hkv = (int)Hkv;
		a.G = (int)(H / Hkv);
		a.dh = (int)Dh;
		a.scale = rule->scale > 0.0f ? rule->scale : 1.0f / std::sqrt((float)Dh);
		a.cap = rule->cap;
		a.slopes = rule->slopes;
		a.causal = rule->causal ? 1 : 0;
		a.window = (int)rule->window;
		a.prefix = rule->prefix;
		p.t = table_of(c);
		p.s = {starts, rule->k_lens, (int)N, (int)rows};
		p.most = (int)std::min(most, rows);
		p.lse = lse;
		const Room room(N, rows, most, c.any_page() ? c.keys() : 0, H, Hkv, Dh);
		p.few = room.plan.few;
		p.split = room.plan.split;
		p.wide = room.plan.wide;
		hipStream_t s = reinterpret_cast<hipStream_t>(stream);
		Scratch ws(s, room.total);
		if (ws.status() != NNH_OK) return ws.status();
		p.split.partial = ws.at<float>(room.split);
		p.wide.partial = ws.at<float>(room.wide);
		return hip_status(paged_attention(p, type, wide(c) && wide(c, q) && wide(c, out), s), "paged attention");
	});
}

}  // extern "C"
