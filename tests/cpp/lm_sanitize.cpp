// lm_sanitize.cpp - TEST CODE: the argument validation of the language-model entry points of include/nnh.h on the host, as
// abi_sanitize.cpp does it for the others (built with -fsanitize=address,undefined; no GPU). Valid calls reach the HIP
// runtime and come back NNH_ERR_HIP, invalid ones with their code before it. Exit status 77 when a GPU is visible.
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <vector>

#include "nnh.h"

namespace {

int g_failures = 0, g_calls = 0;

void expect(const char* what, int got, std::initializer_list<int> allowed) {
	++g_calls;
	for (int a : allowed)
		if (got == a) return;
	std::fprintf(stderr, "FAILED: %s returned %d (%s)\n", what, got, nnh_last_error());
	++g_failures;
}

#define EXPECT(call, ...) expect(#call, (call), {__VA_ARGS__})

constexpr int OK = NNH_OK, INV = NNH_ERR_INVALID, SHAPE = NNH_ERR_SHAPE, ALIAS = NNH_ERR_ALIAS, HIP = NNH_ERR_HIP;
constexpr size_t kHuge = (size_t)1 << 62, kMax = SIZE_MAX;

void attention() {
	// N 2, T 8, H 4, Hkv 2, Dh 16
	std::vector<float> q(1024), k(512), v(512), o(1024), g(1024), dq(1024), dk(512), dv(512), lse(64);
	std::vector<int> docs(16), lens(2);
	const auto head = [](float* p, size_t heads) { return nnh_head_tensor{p, 8 * heads * 16, heads * 16, 16}; };
	const nnh_head_tensor hq = head(q.data(), 4), hk = head(k.data(), 2), hv = head(v.data(), 2), ho = head(o.data(), 4),
	                      hg = head(g.data(), 4), hdq = head(dq.data(), 4), hdk = head(dk.data(), 2), hdv = head(dv.data(), 2);
	nnh_attention_rule r{};
	const auto fwd = [&](int type, size_t N, size_t Tq, size_t Tk, size_t H, size_t Hkv, size_t Dh, const nnh_head_tensor* a,
	                     const nnh_head_tensor* b, const nnh_head_tensor* c, const nnh_head_tensor* out, float* l) {
		return nnh_masked_attention_forward(type, N, Tq, Tk, H, Hkv, Dh, a, b, c, &r, out, nullptr, l, nullptr);
	};
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), HIP);
	EXPECT(fwd(NNH_F32, 0, 8, 8, 4, 2, 16, nullptr, nullptr, nullptr, nullptr, nullptr), OK);
	EXPECT(fwd(NNH_F32, 2, 0, 8, 4, 2, 16, nullptr, &hk, &hv, nullptr, nullptr), OK);
	EXPECT(fwd(2, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 3, 16, &hq, &hk, &hv, &ho, lse.data()), SHAPE);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 0, 2, 16, &hq, &hk, &hv, &ho, lse.data()), SHAPE);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 0, 16, &hq, &hk, &hv, &ho, lse.data()), SHAPE);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 0, &hq, &hk, &hv, &ho, lse.data()), SHAPE);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 129, &hq, &hk, &hv, &ho, lse.data()), INV);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, nullptr, &hk, &hv, &ho, lse.data()), INV);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, nullptr), INV);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &hq, lse.data()), ALIAS);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, o.data()), ALIAS);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, k.data()), ALIAS);
	for (size_t big : {kHuge, kMax, (size_t)1 << 31, (size_t)1 << 33}) {
		EXPECT(fwd(NNH_F32, big, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
		EXPECT(fwd(NNH_F32, 2, big, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
		EXPECT(fwd(NNH_F32, 2, 8, big, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
		EXPECT(fwd(NNH_F32, 2, 8, 8, big, 1, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
		nnh_head_tensor far = hq;
		far.sample = big > kHuge / 2 ? kMax : big;
		EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &far, &hk, &hv, &ho, lse.data()), INV, HIP, ALIAS);  // (its span may hold the output)
		far = ho;
		far.row = kMax - big % 7;
		EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &far, lse.data()), INV);
	}
	nnh_head_tensor same = ho;
	same.sample = 0;
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &same, lse.data()), ALIAS);
	same = ho;
	same.head = 8;
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &same, lse.data()), ALIAS);
	nnh_head_tensor odd = hq;
	odd.data = reinterpret_cast<char*>(q.data()) + 2;
	EXPECT(fwd(NNH_F32, 1, 4, 8, 4, 2, 16, &odd, &hk, &hv, &ho, lse.data()), INV);
	EXPECT(fwd(NNH_BF16, 1, 4, 8, 4, 2, 16, &odd, &hk, &hv, &ho, lse.data()), HIP);
	EXPECT(nnh_masked_attention_forward(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, nullptr, &ho, nullptr, lse.data(), nullptr), INV);
	EXPECT(nnh_masked_attention_forward(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &r, &ho, &hg, lse.data(), nullptr), INV);  // a rest of 32 bits
	const auto rest = [&](nnh_head_tensor x) { return nnh_masked_attention_forward(NNH_BF16, 1, 8, 8, 4, 2, 16, &hq, &hk, &hv, &r, &ho, &x, lse.data(), nullptr); };
	EXPECT(rest(hg), HIP);
	EXPECT(rest(ho), ALIAS);
	EXPECT(rest(hv), ALIAS);
	EXPECT(rest({nullptr, 512, 64, 16}), INV);
	EXPECT(rest({g.data(), 512, 64, 8}), ALIAS);
	EXPECT(rest({lse.data(), 0, 0, 16}), ALIAS);
	r.q_docs = docs.data();
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
	r.k_docs = docs.data();
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), HIP);
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, reinterpret_cast<float*>(docs.data())), ALIAS);
	r = nnh_attention_rule{};
	for (float bad : {-1.0f, __builtin_nanf(""), __builtin_huge_valf()}) {
		r.cap = bad;
		EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
		r.cap = 0.0f;
		r.scale = bad;
		EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
		r.scale = 0.0f;
	}
	r.window = kHuge;
	EXPECT(fwd(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &ho, lse.data()), INV);
	r.window = 0;
	const auto bwd = [&](const nnh_head_tensor* a, const nnh_head_tensor* b, const nnh_head_tensor* c) {
		return nnh_masked_attention_backward(NNH_F32, 2, 8, 8, 4, 2, 16, &hg, &hq, &hk, &hv, &ho, nullptr, lse.data(), &r, a, 1, b, 1, c, 1, nullptr);
	};
	EXPECT(bwd(&hdq, &hdk, &hdv), HIP);
	EXPECT(bwd(nullptr, nullptr, nullptr), OK);
	EXPECT(bwd(nullptr, &hdk, nullptr), HIP);
	EXPECT(bwd(&hdq, &hdk, &hdk), ALIAS);
	EXPECT(bwd(&hq, &hdk, &hdv), ALIAS);
	EXPECT(bwd(&hdq, &hdk, &hg), ALIAS);
	// beside each other in rows of 8 heads: apart; one head too far: not
	std::vector<float> all(2 * 8 * 8 * 16);
	nnh_head_tensor x{all.data(), 8 * 128, 128, 16}, y{all.data() + 64, 8 * 128, 128, 16}, z{all.data() + 96, 8 * 128, 128, 16};
	EXPECT(bwd(&x, &y, &z), HIP);
	y.data = all.data() + 48;
	EXPECT(bwd(&x, &y, &z), ALIAS);
	size_t bytes = 0;
	EXPECT(nnh_masked_attention_workspace_size(2, 8, 8, 4, 2, 16, 1, 1, &bytes), OK);
	EXPECT(nnh_masked_attention_workspace_size(2, 8, 8, 4, 2, 16, 1, 1, nullptr), INV);
	EXPECT(nnh_masked_attention_workspace_size(2, 8, 8, 4, 3, 16, 1, 1, &bytes), SHAPE);
	EXPECT(nnh_masked_attention_workspace_size(kMax, kMax, kMax, kMax, 1, 16, 1, 0, &bytes), INV);
	EXPECT(nnh_masked_attention_workspace_size((size_t)1 << 22, 32, (size_t)1 << 30, 1, 1, 16, 0, 0, &bytes), OK, INV);
}

void loss() {
	std::vector<float> x(8 * 16), w(20 * 16), b(20), out(8), lse(8), dx(8 * 16), dw(20 * 16), db(20), g(8);
	std::vector<int> t(8);
	const auto fwd = [&](int type, size_t rows, size_t D, size_t V, int reduction, float* l) {
		return nnh_linear_cross_entropy_forward(type, x.data(), rows, D, w.data(), V, b.data(), t.data(), reduction, l, lse.data(), nullptr);
	};
	EXPECT(fwd(NNH_F32, 8, 16, 20, NNH_REDUCE_NONE, out.data()), HIP);
	EXPECT(fwd(NNH_BF16, 8, 16, 20, NNH_REDUCE_MEAN, out.data()), HIP);
	EXPECT(fwd(3, 8, 16, 20, NNH_REDUCE_MEAN, out.data()), INV);
	EXPECT(fwd(NNH_F32, 8, 16, 20, 3, out.data()), INV);
	EXPECT(fwd(NNH_F32, 8, 16, 0, NNH_REDUCE_MEAN, out.data()), SHAPE);
	EXPECT(fwd(NNH_F32, 8, 0, 20, NNH_REDUCE_MEAN, out.data()), SHAPE);
	EXPECT(fwd(NNH_F32, 8, 16, 20, NNH_REDUCE_MEAN, nullptr), INV);
	EXPECT(fwd(NNH_F32, 8, 16, 20, NNH_REDUCE_MEAN, x.data()), ALIAS);
	EXPECT(fwd(NNH_F32, 8, 16, 20, NNH_REDUCE_MEAN, lse.data() + 3), ALIAS);
	EXPECT(fwd(NNH_F32, 0, 16, 20, NNH_REDUCE_NONE, nullptr), OK);
	for (size_t big : {kHuge, kMax, (size_t)1 << 31, (size_t)1 << 30}) {
		EXPECT(fwd(NNH_F32, big, 16, 20, NNH_REDUCE_MEAN, out.data()), INV);
		EXPECT(fwd(NNH_F32, 8, big, 20, NNH_REDUCE_MEAN, out.data()), INV);
		EXPECT(fwd(NNH_F32, (size_t)1 << 20, 16, big, NNH_REDUCE_MEAN, out.data()), INV);
	}
	EXPECT(nnh_linear_cross_entropy_forward(NNH_F32, nullptr, 8, 16, w.data(), 20, nullptr, t.data(), 1, out.data(), lse.data(), nullptr), INV);
	EXPECT(nnh_linear_cross_entropy_forward(NNH_F32, x.data(), 8, 16, nullptr, 20, nullptr, t.data(), 1, out.data(), lse.data(), nullptr), INV);
	EXPECT(nnh_linear_cross_entropy_forward(NNH_F32, x.data(), 8, 16, w.data(), 20, nullptr, nullptr, 1, out.data(), lse.data(), nullptr), INV);
	EXPECT(nnh_linear_cross_entropy_forward(NNH_BF16, reinterpret_cast<char*>(x.data()) + 1, 8, 16, w.data(), 20, nullptr, t.data(), 1, out.data(), lse.data(), nullptr), INV);
	const auto bwd = [&](float* a, float* c, float* d) {
		return nnh_linear_cross_entropy_backward(NNH_F32, g.data(), x.data(), 8, 16, w.data(), 20, b.data(), t.data(), lse.data(), NNH_REDUCE_NONE, a, 1, c, 1, d, 1, nullptr);
	};
	EXPECT(bwd(dx.data(), dw.data(), db.data()), HIP);
	EXPECT(bwd(nullptr, nullptr, nullptr), OK);
	EXPECT(bwd(x.data(), dw.data(), db.data()), ALIAS);
	EXPECT(bwd(dx.data(), dx.data(), db.data()), ALIAS);
	EXPECT(bwd(dx.data(), dw.data(), g.data()), ALIAS);
	EXPECT(nnh_linear_cross_entropy_backward(NNH_F32, nullptr, x.data(), 8, 16, w.data(), 20, nullptr, t.data(), nullptr, 1, dx.data(), 1, dw.data(), 1, nullptr, 1, nullptr), INV);
	EXPECT(nnh_linear_cross_entropy_train(NNH_F32, nullptr, x.data(), 8, 16, w.data(), 20, b.data(), t.data(), 1, out.data(), dx.data(), 1, dw.data(), 1, db.data(), 1, nullptr), HIP);
	EXPECT(nnh_linear_cross_entropy_train(NNH_F32, nullptr, x.data(), 8, 16, w.data(), 20, b.data(), t.data(), 1, nullptr, dx.data(), 1, dw.data(), 1, db.data(), 1, nullptr), INV);
	EXPECT(nnh_linear_cross_entropy_train(NNH_F32, nullptr, x.data(), 8, 16, w.data(), 20, b.data(), t.data(), 1, dx.data(), dx.data(), 1, dw.data(), 1, db.data(), 1, nullptr), ALIAS);
	size_t bytes = 0;
	for (int type : {NNH_F32, NNH_BF16})
		for (int call = 0; call < 3; ++call) {
			EXPECT(nnh_linear_cross_entropy_workspace_size(type, 8192, 4096, 128000, call, 1, &bytes), OK);
			EXPECT(nnh_linear_cross_entropy_workspace_size(type, 1 << 20, 33, 5, call, 0, &bytes), OK);
			EXPECT(nnh_linear_cross_entropy_workspace_size(type, 0, 4, 5, call, 0, &bytes), OK);
			EXPECT(nnh_linear_cross_entropy_workspace_size(type, kMax, 4, 5, call, 0, &bytes), INV);
		}
	EXPECT(nnh_linear_cross_entropy_workspace_size(NNH_F32, 8, 4, 5, 3, 0, &bytes), INV);
	EXPECT(nnh_linear_cross_entropy_workspace_size(NNH_F32, 8, 4, 5, 0, 0, nullptr), INV);
}

void adamw() {
	std::vector<float> p(64), g(64), m(64), v(64), q(64), scale(1);
	std::vector<unsigned char> cm(64), cv(64), sm(1), sv(1);
	nnh_adamw o{};
	o.bits = 32;
	o.lr = 1e-3;
	o.beta1 = 0.9;
	o.beta2 = 0.99;
	o.step = 1;
	nnh_adamw_tensor t[2] = {{p.data(), g.data(), m.data(), v.data(), nullptr, nullptr, nullptr, 64}, {p.data(), g.data(), m.data(), v.data(), nullptr, nullptr, nullptr, 64}};
	EXPECT(nnh_adamw_step(&o, t, 1, nullptr), HIP);
	EXPECT(nnh_adamw_step(&o, nullptr, 0, nullptr), OK);
	EXPECT(nnh_adamw_step(nullptr, t, 1, nullptr), INV);
	EXPECT(nnh_adamw_step(&o, nullptr, 1, nullptr), INV);
	EXPECT(nnh_adamw_step(&o, t, 2, nullptr), ALIAS);  // the same tensor twice
	t[1] = {q.data(), g.data(), nullptr, nullptr, nullptr, nullptr, nullptr, 64};
	EXPECT(nnh_adamw_step(&o, t, 2, nullptr), INV);
	t[1].count = 0;
	EXPECT(nnh_adamw_step(&o, t, 2, nullptr), HIP);
	nnh_adamw_tensor x = t[0];
	x.g = p.data() + 32;
	EXPECT(nnh_adamw_step(&o, &x, 1, nullptr), ALIAS);
	x = t[0];
	x.count = kHuge;
	EXPECT(nnh_adamw_step(&o, &x, 1, nullptr), INV);
	x = t[0];
	x.p = reinterpret_cast<char*>(p.data()) + 2;
	EXPECT(nnh_adamw_step(&o, &x, 1, nullptr), INV);
	o.grad_scale = m.data() + 5;
	EXPECT(nnh_adamw_step(&o, t, 1, nullptr), ALIAS);
	o.grad_scale = scale.data();
	EXPECT(nnh_adamw_step(&o, t, 1, nullptr), HIP);
	const nnh_adamw fine = o;
	const auto with = [&](auto change) {
		o = fine;
		change();
		return nnh_adamw_step(&o, t, 1, nullptr);
	};
	EXPECT(with([&] { o.bits = 16; }), INV);
	EXPECT(with([&] { o.p_type = 2; }), INV);
	EXPECT(with([&] { o.g_type = -1; }), INV);
	EXPECT(with([&] { o.beta1 = 1.0; }), INV);
	EXPECT(with([&] { o.beta2 = -0.1; }), INV);
	EXPECT(with([&] { o.beta2 = __builtin_nan(""); }), INV);
	EXPECT(with([&] { o.eps = -1.0; }), INV);
	EXPECT(with([&] { o.lr = __builtin_huge_val(); }), INV);
	EXPECT(with([&] { o.weight_decay = __builtin_nan(""); }), INV);
	EXPECT(with([&] { o.step = 0; }), INV);
	EXPECT(with([&] { o.beta1 = o.beta2 = 0.0; }), HIP);
	o = fine;
	o.bits = 8;
	EXPECT(nnh_adamw_step(&o, t, 1, nullptr), INV);
	x = {p.data(), g.data(), cm.data(), cv.data(), sm.data(), sv.data(), nullptr, 64};
	EXPECT(nnh_adamw_step(&o, &x, 1, nullptr), HIP);
	x.v_scale = sm.data();
	EXPECT(nnh_adamw_step(&o, &x, 1, nullptr), ALIAS);
}

}  // namespace

int main() {
	int devices = 0;
	if (hipGetDeviceCount(&devices) == hipSuccess && devices > 0) {
		std::printf("skipped: a GPU is visible (this test passes host buffers where device pointers belong)\n");
		return 77;
	}
	attention();
	loss();
	adamw();
	if (g_failures) {
		std::fprintf(stderr, "%d of %d calls returned an unexpected code\n", g_failures, g_calls);
		return 1;
	}
	std::printf("language-model validation: %d calls, every code as expected\n", g_calls);
	return 0;
}
