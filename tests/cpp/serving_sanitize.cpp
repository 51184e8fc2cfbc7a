// serving_sanitize.cpp - TEST CODE: the argument validation of the serving entry points of include/nnh.h on the host, as lm_sanitize.cpp
// does it for the language-model ones (built with -fsanitize=address,undefined; no GPU). Valid calls reach the HIP runtime and come back
// NNH_ERR_HIP, invalid ones with their code before it. Exit status 77 when a GPU is visible.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <vector>

#include "nnh.h"

namespace {

int g_failures = 0, g_calls = 0;

void expect(const char* what, int line, int got, std::initializer_list<int> allowed) {
	++g_calls;
	for (int a : allowed)
		if (got == a) return;
	std::fprintf(stderr, "FAILED: line %d: %s returned %d (%s)\n", line, what, got, nnh_last_error());
	++g_failures;
}

#define EXPECT(call, ...) expect(#call, __LINE__, (call), {__VA_ARGS__})

constexpr int OK = NNH_OK, INV = NNH_ERR_INVALID, SHAPE = NNH_ERR_SHAPE, ALIAS = NNH_ERR_ALIAS, HIP = NNH_ERR_HIP;
constexpr size_t kHuge = (size_t)1 << 62, kMax = SIZE_MAX;
const size_t kBig[] = {(size_t)1 << 31, (size_t)1 << 33, kHuge, kMax};

void paged() {
	// N 2, 7 rows, H 4, Hkv 2, Dh 16; 5 pages of 8, 3 to a sequence
	std::vector<float> q(7 * 64), k(7 * 32), v(7 * 32), o(7 * 64), lse(7 * 4 + 4), kp(5 * 8 * 32), vp(5 * 8 * 32), slopes(4);
	std::vector<int> starts(4), lens(3), table(7), prefix(2);
	const nnh_head_tensor hq{q.data(), 0, 64, 16}, hk{k.data(), 0, 32, 16}, hv{v.data(), 0, 32, 16}, ho{o.data(), 0, 64, 16};
	const nnh_paged_cache good{kp.data(), vp.data(), 8 * 32, 32, 16, 5, 8, table.data(), 3};
	nnh_paged_cache c = good;
	const auto add = [&](const nnh_head_tensor* a, const nnh_head_tensor* b) {
		return nnh_paged_append(NNH_F32, 2, 7, 2, 16, a, b, starts.data(), lens.data(), &c, nullptr);
	};
	EXPECT(add(&hk, &hv), HIP);
	EXPECT(nnh_paged_append(NNH_BF16, 2, 7, 2, 16, &hk, &hv, starts.data(), lens.data(), &c, nullptr), HIP);
	EXPECT(nnh_paged_append(2, 2, 7, 2, 16, &hk, &hv, starts.data(), lens.data(), &c, nullptr), INV);
	EXPECT(nnh_paged_append(NNH_F32, 0, 7, 2, 16, nullptr, nullptr, nullptr, nullptr, &c, nullptr), OK);
	EXPECT(nnh_paged_append(NNH_F32, 2, 0, 2, 16, nullptr, nullptr, nullptr, nullptr, &c, nullptr), OK);
	EXPECT(nnh_paged_append(NNH_F32, 2, 7, 0, 16, &hk, &hv, starts.data(), lens.data(), &c, nullptr), SHAPE);
	EXPECT(nnh_paged_append(NNH_F32, 2, 7, 2, 0, &hk, &hv, starts.data(), lens.data(), &c, nullptr), SHAPE);
	EXPECT(nnh_paged_append(NNH_F32, 2, 7, 2, 16, &hk, &hv, nullptr, lens.data(), &c, nullptr), INV);
	EXPECT(nnh_paged_append(NNH_F32, 2, 7, 2, 16, &hk, &hv, starts.data(), nullptr, &c, nullptr), INV);
	EXPECT(nnh_paged_append(NNH_F32, 2, 7, 2, 16, &hk, &hv, starts.data(), lens.data(), nullptr, nullptr), INV);
	EXPECT(nnh_paged_append(NNH_F32, 2, 7, 2, 16, &hk, &hv, reinterpret_cast<int*>(reinterpret_cast<char*>(starts.data()) + 2), lens.data(), &c, nullptr), INV);
	EXPECT(add(nullptr, &hv), INV);
	EXPECT(add(&hk, nullptr), INV);
	for (size_t big : kBig) {
		EXPECT(nnh_paged_append(NNH_F32, big, 7, 2, 16, &hk, &hv, starts.data(), lens.data(), &c, nullptr), INV);
		EXPECT(nnh_paged_append(NNH_F32, 2, big, 2, 16, &hk, &hv, starts.data(), lens.data(), &c, nullptr), INV);
		EXPECT(nnh_paged_append(NNH_F32, 2, 7, big, 16, &hk, &hv, starts.data(), lens.data(), &c, nullptr), INV);
		EXPECT(nnh_paged_append(NNH_F32, 2, 7, 2, big, &hk, &hv, starts.data(), lens.data(), &c, nullptr), INV);
		for (size_t nnh_paged_cache::*field : {&nnh_paged_cache::pages, &nnh_paged_cache::page_size, &nnh_paged_cache::width}) {
			c.*field = big;
			EXPECT(add(&hk, &hv), INV);
			c = good;
		}
		for (size_t nnh_paged_cache::*field : {&nnh_paged_cache::page, &nnh_paged_cache::slot, &nnh_paged_cache::head}) {
			c.*field = big;
			EXPECT(add(&hk, &hv), INV, ALIAS, HIP);  // (an extent that holds the rows, or none that is out of range)
			c = good;
		}
		nnh_head_tensor far = hk;
		far.row = big;
		EXPECT(add(&far, &hv), INV, ALIAS, HIP);
	}
	// no pages, or none to a sequence: nothing is stored
	c.pages = 0;
	EXPECT(add(&hk, &hv), OK);
	c = good;
	c.width = 0;
	c.table = nullptr;
	EXPECT(add(&hk, &hv), OK);
	c = good;
	c.page_size = 0;
	EXPECT(add(&hk, &hv), SHAPE);
	c = good;
	c.table = nullptr;
	EXPECT(add(&hk, &hv), INV);
	c = good;
	c.k = nullptr;
	EXPECT(add(&hk, &hv), INV);
	c = good;
	c.v = reinterpret_cast<char*>(vp.data()) + 2;
	EXPECT(add(&hk, &hv), INV);
	// places that overlap: slots, keys and values, the rows; side by side: apart
	c = good;
	c.slot = 24;
	EXPECT(add(&hk, &hv), ALIAS);
	c = good;
	c.page = 0;
	EXPECT(add(&hk, &hv), ALIAS);
	c = good;
	c.v = kp.data() + 32;
	EXPECT(add(&hk, &hv), ALIAS);
	std::vector<float> both(5 * 8 * 64);
	c = {both.data(), both.data() + 256, 512, 32, 16, 5, 8, table.data(), 3};
	EXPECT(add(&hk, &hv), HIP);
	c = {both.data(), both.data() + 32, 512, 64, 16, 5, 8, table.data(), 3};
	EXPECT(add(&hk, &hv), HIP);
	c = {both.data(), both.data() + 16, 512, 64, 32, 5, 8, table.data(), 3};
	EXPECT(add(&hk, &hv), HIP);
	c.v = both.data() + 8;
	EXPECT(add(&hk, &hv), ALIAS);
	c = good;
	nnh_head_tensor in = hk;
	in.data = kp.data() + 100;
	EXPECT(add(&in, &hv), ALIAS);
	c.table = reinterpret_cast<const int*>(vp.data());
	EXPECT(add(&hk, &hv), ALIAS);
	c = good;

	nnh_attention_rule r{};
	r.k_lens = lens.data();
	const nnh_attention_rule plain = r;
	const auto see = [&](int type, size_t N, size_t rows, size_t most, size_t H, size_t Hkv, size_t Dh, const nnh_head_tensor* a, const nnh_head_tensor* b, float* l) {
		return nnh_paged_attention(type, N, rows, most, H, Hkv, Dh, a, &c, starts.data(), &r, b, l, nullptr);
	};
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), HIP);
	EXPECT(see(NNH_BF16, 2, 7, kMax >> 40, 4, 2, 16, &hq, &ho, lse.data()), HIP);
	EXPECT(see(7, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
	EXPECT(see(NNH_F32, 0, 7, 4, 4, 2, 16, nullptr, nullptr, nullptr), OK);
	EXPECT(see(NNH_F32, 2, 0, 4, 4, 2, 16, nullptr, nullptr, nullptr), OK);
	EXPECT(see(NNH_F32, 2, 7, 0, 4, 2, 16, nullptr, nullptr, nullptr), OK);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 3, 16, &hq, &ho, lse.data()), SHAPE);
	EXPECT(see(NNH_F32, 2, 7, 4, 0, 2, 16, &hq, &ho, lse.data()), SHAPE);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 0, 16, &hq, &ho, lse.data()), SHAPE);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 0, &hq, &ho, lse.data()), SHAPE);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 129, &hq, &ho, lse.data()), INV);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, nullptr, &ho, lse.data()), INV);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, nullptr, lse.data()), INV);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, nullptr), INV);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &hq, lse.data()), ALIAS);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, o.data() + 40), ALIAS);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, reinterpret_cast<float*>(lens.data())), ALIAS);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, kp.data() + 5), ALIAS);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, reinterpret_cast<float*>(reinterpret_cast<char*>(lse.data()) + 1)), INV);
	nnh_head_tensor odd = ho;
	odd.head = 8;
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &odd, lse.data()), ALIAS);
	odd = ho;
	odd.row = 0;
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &odd, lse.data()), ALIAS);
	odd = hq;
	odd.data = reinterpret_cast<char*>(q.data()) + 2;
	EXPECT(see(NNH_F32, 2, 6, 4, 4, 2, 16, &odd, &ho, lse.data()), INV);
	EXPECT(see(NNH_BF16, 2, 6, 4, 4, 2, 16, &odd, &ho, lse.data()), HIP);
	odd.data = vp.data();
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &odd, lse.data()), ALIAS);
	for (size_t big : kBig) {
		EXPECT(see(NNH_F32, big, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
		EXPECT(see(NNH_F32, 2, big, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
		EXPECT(see(NNH_F32, 2, 7, big, 4, 2, 16, &hq, &ho, lse.data()), INV);
		EXPECT(see(NNH_F32, 2, 7, 4, big, 1, 16, &hq, &ho, lse.data()), INV, SHAPE);
		EXPECT(see(NNH_F32, 2, 7, 4, big, big, 16, &hq, &ho, lse.data()), INV, SHAPE);
		EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, big, &hq, &ho, lse.data()), INV);
		r.window = big;
		EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
		r = plain;
		size_t bytes = 0;
		EXPECT(nnh_paged_attention_workspace_size(big, 7, 4, 24, 4, 2, 16, &bytes), INV);
		EXPECT(nnh_paged_attention_workspace_size(2, big, 4, 24, 4, 2, 16, &bytes), INV);
		EXPECT(nnh_paged_attention_workspace_size(2, 7, 4, big, 4, 2, 16, &bytes), INV);
	}
	r.k_lens = nullptr;
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
	for (const int* nnh_attention_rule::*field : {&nnh_attention_rule::q_start, &nnh_attention_rule::q_docs, &nnh_attention_rule::k_docs}) {
		r = plain;
		r.*field = prefix.data();
		EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
	}
	r = plain;
	r.prefix = prefix.data();
	r.slopes = slopes.data();
	r.causal = 1;
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), HIP);
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, slopes.data()), ALIAS);
	for (float bad : {-1.0f, __builtin_nanf(""), __builtin_huge_valf()}) {
		r = plain;
		r.cap = bad;
		EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
		r = plain;
		r.scale = bad;
		EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), INV);
	}
	r = plain;
	EXPECT(nnh_paged_attention(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &c, starts.data(), nullptr, &ho, lse.data(), nullptr), INV);
	EXPECT(nnh_paged_attention(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, nullptr, starts.data(), &r, &ho, lse.data(), nullptr), INV);
	EXPECT(nnh_paged_attention(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &c, nullptr, &r, &ho, lse.data(), nullptr), INV);
	c.pages = 0;  // (rows that see nothing: a kernel's work all the same)
	c.k = c.v = nullptr;
	EXPECT(see(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &ho, lse.data()), HIP);
	size_t bytes = 0;
	EXPECT(nnh_paged_attention_workspace_size(2, 7, 4, 24, 4, 2, 16, nullptr), INV);
	EXPECT(nnh_paged_attention_workspace_size(2, 7, 4, 24, 4, 3, 16, &bytes), SHAPE);
	EXPECT(nnh_paged_attention_workspace_size(0, 0, 0, 0, 4, 2, 16, &bytes), OK);
	EXPECT(nnh_paged_attention_workspace_size(1, 1, 1, (size_t)1 << 30, 128, 1, 128, &bytes), OK);
}

void int8() {
	std::vector<float> x(20 * 40), y(20 * 12), scale(20), ws(12), bias(12);
	std::vector<signed char> room(20 * 48 + 16), wroom(12 * 48 + 16);
	signed char* const codes = room.data() + (16 - reinterpret_cast<uintptr_t>(room.data()) % 16) % 16;
	signed char* const w = wroom.data() + (16 - reinterpret_cast<uintptr_t>(wroom.data()) % 16) % 16;
	const auto rows = [&](int type, const void* from, size_t n, size_t D, size_t ldx, signed char* to, size_t ldc, float* s) {
		return nnh_quantize_rows(type, from, n, D, ldx, to, ldc, s, nullptr);
	};
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, codes, 48, scale.data()), HIP);
	EXPECT(rows(NNH_BF16, x.data(), 20, 40, 80, codes, 40, scale.data()), HIP);
	EXPECT(rows(NNH_F32, nullptr, 0, 40, 40, nullptr, 48, nullptr), OK);
	EXPECT(rows(NNH_F32, nullptr, 20, 0, 0, nullptr, 0, scale.data()), HIP);  // (scales of 0)
	EXPECT(rows(5, x.data(), 20, 40, 40, codes, 48, scale.data()), INV);
	EXPECT(rows(NNH_F32, nullptr, 20, 40, 40, codes, 48, scale.data()), INV);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, nullptr, 48, scale.data()), INV);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, codes, 48, nullptr), INV);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 39, codes, 48, scale.data()), INV);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, codes, 39, scale.data()), INV);
	EXPECT(rows(NNH_F32, reinterpret_cast<char*>(x.data()) + 2, 10, 40, 40, codes, 48, scale.data()), INV);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, reinterpret_cast<signed char*>(x.data()) + 100, 48, scale.data()), ALIAS);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, codes, 48, x.data() + 4), ALIAS);
	EXPECT(rows(NNH_F32, x.data(), 20, 40, 40, reinterpret_cast<signed char*>(scale.data()), 48, scale.data()), ALIAS);
	const auto lin = [&](int type, const void* from, size_t n, size_t D, size_t ldx, const signed char* c, size_t ldw, const float* s, size_t V, const void* b, void* to,
	                     size_t ldy) { return nnh_linear_int8(type, from, n, D, ldx, c, ldw, s, V, b, to, ldy, nullptr); };
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), 12, bias.data(), y.data(), 12), HIP);
	EXPECT(lin(NNH_F32, x.data(), 3, 40, 40, w, 48, ws.data(), 12, nullptr, y.data(), 12), HIP);
	EXPECT(lin(NNH_BF16, x.data(), 20, 40, 40, w, 48, ws.data(), 12, nullptr, y.data(), 24), HIP);
	EXPECT(lin(NNH_F32, nullptr, 0, 40, 40, w, 48, ws.data(), 12, nullptr, nullptr, 12), OK);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, nullptr, 48, nullptr, 0, nullptr, nullptr, 0), OK);
	EXPECT(lin(NNH_F32, nullptr, 20, 0, 0, nullptr, 0, ws.data(), 12, bias.data(), y.data(), 12), HIP);  // (the bias)
	EXPECT(lin(4, x.data(), 20, 40, 40, w, 48, ws.data(), 12, nullptr, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, nullptr, 20, 40, 40, w, 48, ws.data(), 12, nullptr, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, nullptr, 48, ws.data(), 12, nullptr, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, nullptr, 12, nullptr, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), 12, nullptr, nullptr, 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 39, w, 48, ws.data(), 12, nullptr, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 32, ws.data(), 12, nullptr, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 40, ws.data(), 12, nullptr, y.data(), 12), INV);       // rows off 16 bytes
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w + 8, 48, ws.data(), 11, nullptr, y.data(), 12), INV);   // the first one too
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), 12, nullptr, y.data(), 11), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), 12, reinterpret_cast<char*>(bias.data()) + 2, y.data(), 12), INV);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), 12, nullptr, x.data() + 10, 12), ALIAS);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), 12, y.data() + 1, y.data(), 12), ALIAS);
	EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, y.data() + 2, 12, nullptr, y.data(), 12), ALIAS);
	EXPECT(lin(NNH_F32, x.data(), 2, 40, 40, w, 48, ws.data(), 12, nullptr, w + 16, 12), ALIAS);
	EXPECT(lin(NNH_F32, x.data(), 1, (size_t)1 << 17, (size_t)1 << 17, w, (size_t)1 << 17, ws.data(), 12, nullptr, y.data(), 12), INV);  // sums past 32 bits
	size_t bytes = 0;
	for (size_t big : kBig) {
		EXPECT(rows(NNH_F32, x.data(), big, 40, 40, codes, 48, scale.data()), INV);
		EXPECT(rows(NNH_F32, x.data(), 20, big, big, codes, big, scale.data()), INV);
		EXPECT(rows(NNH_F32, x.data(), 20, 40, big, codes, 48, scale.data()), INV, ALIAS, HIP);
		EXPECT(lin(NNH_F32, x.data(), big, 40, 40, w, 48, ws.data(), 12, nullptr, y.data(), 12), INV);
		EXPECT(lin(NNH_F32, x.data(), 20, big, big, w, big, ws.data(), 12, nullptr, y.data(), 12), INV);
		EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, 48, ws.data(), big, nullptr, y.data(), big), INV);
		EXPECT(lin(NNH_F32, x.data(), 20, 40, 40, w, big, ws.data(), 12, nullptr, y.data(), 12), INV, ALIAS, HIP);
		EXPECT(nnh_linear_int8_workspace_size(big, 40, 12, &bytes), INV);
		EXPECT(nnh_linear_int8_workspace_size(20, big, 12, &bytes), INV);
		EXPECT(nnh_linear_int8_workspace_size(20, 40, big, &bytes), INV);
	}
	EXPECT(nnh_linear_int8_workspace_size(20, 40, 12, nullptr), INV);
	EXPECT(nnh_linear_int8_workspace_size(((size_t)1 << 24) - 1, 131071, ((size_t)1 << 24) - 1, &bytes), OK);
	EXPECT(nnh_linear_int8_workspace_size(0, 0, 0, &bytes), OK);
}

void choice() {
	std::vector<float> z(6 * 50), u(6), t(6), p(6), m(6), lp(6);
	std::vector<int> k(6), tokens(6);
	const auto take = [&](int type, const void* logits, size_t rows, size_t V, size_t ld, const float* uu, const float* temp, int* out, float* l) {
		return nnh_sample(type, logits, rows, V, ld, uu, temp, k.data(), p.data(), m.data(), out, l, nullptr);
	};
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), tokens.data(), lp.data()), HIP);
	EXPECT(take(NNH_BF16, z.data(), 6, 50, 100, u.data(), nullptr, tokens.data(), nullptr), HIP);
	EXPECT(nnh_sample(NNH_F32, z.data(), 6, 50, 50, u.data(), nullptr, nullptr, nullptr, nullptr, tokens.data(), nullptr, nullptr), HIP);
	EXPECT(take(NNH_F32, nullptr, 0, 50, 50, nullptr, nullptr, nullptr, nullptr), OK);
	EXPECT(take(NNH_F32, z.data(), 6, 0, 50, u.data(), t.data(), tokens.data(), lp.data()), SHAPE);
	EXPECT(take(9, z.data(), 6, 50, 50, u.data(), t.data(), tokens.data(), lp.data()), INV);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 49, u.data(), t.data(), tokens.data(), lp.data()), INV);
	EXPECT(take(NNH_F32, nullptr, 6, 50, 50, u.data(), t.data(), tokens.data(), lp.data()), INV);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, nullptr, t.data(), tokens.data(), lp.data()), INV);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), nullptr, lp.data()), INV);
	EXPECT(take(NNH_F32, reinterpret_cast<char*>(z.data()) + 2, 5, 50, 50, u.data(), t.data(), tokens.data(), lp.data()), INV);
	EXPECT(take(NNH_F32, z.data(), 5, 50, 50, reinterpret_cast<float*>(reinterpret_cast<char*>(u.data()) + 2), t.data(), tokens.data(), lp.data()), INV);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), tokens.data(), z.data() + 8), ALIAS);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), tokens.data(), u.data()), ALIAS);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), tokens.data(), t.data() + 2), ALIAS);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), k.data(), lp.data()), ALIAS);
	EXPECT(take(NNH_F32, z.data(), 6, 50, 50, u.data(), t.data(), tokens.data(), reinterpret_cast<float*>(tokens.data())), ALIAS);
	size_t bytes = 0;
	for (size_t big : kBig) {
		EXPECT(take(NNH_F32, z.data(), big, 50, 50, u.data(), t.data(), tokens.data(), lp.data()), INV);
		EXPECT(take(NNH_F32, z.data(), 6, big, big, u.data(), t.data(), tokens.data(), lp.data()), INV);
		EXPECT(take(NNH_F32, z.data(), 1, 50, big, u.data(), t.data(), tokens.data(), lp.data()), INV, HIP);
		EXPECT(nnh_sample_workspace_size(NNH_F32, big, 50, &bytes), INV);
		EXPECT(nnh_sample_workspace_size(NNH_F32, 6, big, &bytes), INV);
	}
	EXPECT(nnh_sample_workspace_size(NNH_F32, 6, 50, nullptr), INV);
	EXPECT(nnh_sample_workspace_size(3, 6, 50, &bytes), INV);
	EXPECT(nnh_sample_workspace_size(NNH_BF16, (1 << 22) - 1, (size_t)1 << 28, &bytes), OK);
	EXPECT(nnh_sample_workspace_size(NNH_F32, 0, 0, &bytes), OK);
}

}  // namespace

int main() {
	int devices = 0;
	if (hipGetDeviceCount(&devices) == hipSuccess && devices > 0) {
		std::printf("skipped: a GPU is visible (this test passes host buffers where device pointers belong)\n");
		return 77;
	}
	paged();
	int8();
	choice();
	if (g_failures) {
		std::fprintf(stderr, "%d of %d calls returned an unexpected code\n", g_failures, g_calls);
		return 1;
	}
	std::printf("serving validation: %d calls, every code as expected\n", g_calls);
	return 0;
}
