// lm_align_sanitize.cpp - TEST CODE: the language-model entry points of include/nnh.h refuse arrays of 32-bit elements that do not
// begin at a multiple of 4 bytes, on the host (as lm_sanitize.cpp). Exit status 77 when a GPU is visible.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <vector>

#include "nnh.h"

namespace {

int g_failures = 0, g_calls = 0;

void expect(const char* what, int got, int want) {
	++g_calls;
	if (got == want) return;
	std::fprintf(stderr, "FAILED: %s returned %d, not %d (%s)\n", what, got, want, nnh_last_error());
	++g_failures;
}

template <typename T>
T* off(T* p, int bytes) {
	return reinterpret_cast<T*>(reinterpret_cast<uintptr_t>(p) + bytes);
}

}  // namespace

int main() {
	int devices = 0;
	if (hipGetDeviceCount(&devices) == hipSuccess && devices > 0) {
		std::printf("skipped: a GPU is visible (this test passes host buffers where device pointers belong)\n");
		return 77;
	}
	std::vector<float> q(1024), k(512), v(512), o(1024), g(1024), dq(1024), lse(80), slopes(8);
	std::vector<int> whole[5];
	for (auto& x : whole) x.resize(32);
	const auto head = [](float* p, size_t heads) { return nnh_head_tensor{p, 8 * heads * 16, heads * 16, 16}; };
	const nnh_head_tensor hq = head(q.data(), 4), hk = head(k.data(), 2), hv = head(v.data(), 2), ho = head(o.data(), 4), hg = head(g.data(), 4), hdq = head(dq.data(), 4);
	for (int bytes = 0; bytes < 4; ++bytes) {
		const int want = bytes ? NNH_ERR_INVALID : NNH_ERR_HIP;
		for (int which = 0; which < 7; ++which) {
			const auto moved = [&](int i) { return off(whole[i].data(), which == i ? bytes : 0); };
			nnh_attention_rule r{};
			r.q_start = moved(0);
			r.k_lens = moved(1);
			r.prefix = moved(2);
			r.q_docs = moved(3);
			r.k_docs = moved(4);
			r.slopes = off(slopes.data(), which == 5 ? bytes : 0);
			float* const l = off(lse.data(), which == 6 ? bytes : 0);
			expect("attention forward", nnh_masked_attention_forward(NNH_BF16, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &r, &ho, nullptr, l, nullptr), want);
			expect("attention backward", nnh_masked_attention_backward(NNH_BF16, 2, 8, 8, 4, 2, 16, &hg, &hq, &hk, &hv, &ho, nullptr, l, &r, &hdq, 1, nullptr, 1, nullptr, 1, nullptr), want);
		}
		std::vector<float> x(128), w(320), out(16), dw(320), up(16);
		std::vector<int> t(16);
		for (int which = 0; which < 4; ++which) {
			const int* const y = off(t.data(), which == 0 ? bytes : 0);
			float* const l = off(lse.data(), which == 1 ? bytes : 0);
			float* const loss = off(out.data(), which == 2 ? bytes : 0);
			const float* const d = off(up.data(), which == 3 ? bytes : 0);
			expect("loss forward", nnh_linear_cross_entropy_forward(NNH_BF16, x.data(), 8, 16, w.data(), 20, nullptr, y, 0, loss, l, nullptr), which == 3 ? NNH_ERR_HIP : want);
			expect("loss backward", nnh_linear_cross_entropy_backward(NNH_BF16, d, x.data(), 8, 16, w.data(), 20, nullptr, y, l, 0, nullptr, 1, dw.data(), 1, nullptr, 1, nullptr), which == 2 ? NNH_ERR_HIP : want);
			expect("loss train", nnh_linear_cross_entropy_train(NNH_BF16, d, x.data(), 8, 16, w.data(), 20, nullptr, y, 0, loss, nullptr, 1, dw.data(), 1, nullptr, 1, nullptr), which == 1 ? NNH_ERR_HIP : want);
		}
		for (int which = 0; which < 3; ++which) {
			nnh_adamw a{};
			a.bits = 32;
			a.beta1 = 0.9;
			a.beta2 = 0.99;
			a.step = 1;
			a.step_device = off(whole[0].data(), which == 0 ? bytes : 0);
			a.lr_device = off(up.data(), which == 1 ? bytes : 0);
			a.grad_scale = off(out.data(), which == 2 ? bytes : 0);
			const nnh_adamw_tensor one{q.data(), k.data(), o.data(), g.data(), nullptr, nullptr, nullptr, 64};
			expect("adamw", nnh_adamw_step(&a, &one, 1, nullptr), want);
		}
	}
	if (g_failures) {
		std::fprintf(stderr, "%d of %d calls returned an unexpected code\n", g_failures, g_calls);
		return 1;
	}
	std::printf("alignment: %d calls, every code as expected\n", g_calls);
	return 0;
}
