// lm_nomem.cpp - TEST CODE: the language-model entry points of include/nnh.h where the host has no memory left. Each call is one that
// is refused after its lists are made (an output over an input), and runs with its k-th allocation failing for every k: it must
// come back with a code, since nothing may be thrown across the C boundary (std::terminate there ends this program).
#include <cstdio>
#include <cstdlib>
#include <new>
#include <vector>

#include "nnh.h"

namespace {
thread_local long g_left = -1;  // allocations until one fails; negative: none does
thread_local bool g_failed = false;
}  // namespace

void* operator new(std::size_t n) {
	if (g_left == 0) {
		g_failed = true;
		throw std::bad_alloc();
	}
	if (g_left > 0) --g_left;
	if (void* p = std::malloc(n ? n : 1)) return p;
	throw std::bad_alloc();
}
void operator delete(void* p) noexcept { std::free(p); }
void operator delete(void* p, std::size_t) noexcept { std::free(p); }

namespace {

int g_failures = 0, g_calls = 0;

template <typename F>
void exhaust(const char* what, int code, F call) {
	for (long k = 0; k < 200; ++k) {
		g_failed = false;
		g_left = k;
		const int rc = call();
		g_left = -1;
		++g_calls;
		const bool end = !g_failed;
		if (rc != (end ? code : NNH_ERR_INVALID) && rc != code) {
			std::fprintf(stderr, "FAILED: %s with allocation %ld failing returned %d (%s)\n", what, k, rc, nnh_last_error());
			++g_failures;
		}
		if (end) return;
	}
	std::fprintf(stderr, "FAILED: %s makes more than 200 allocations\n", what);
	++g_failures;
}

}  // namespace

int main() {
	std::vector<float> q(1024), k(512), v(512), o(1024), g(1024), lse(64), big(4096);
	const auto head = [](float* p, size_t heads) { return nnh_head_tensor{p, 8 * heads * 16, heads * 16, 16}; };
	const nnh_head_tensor hq = head(q.data(), 4), hk = head(k.data(), 2), hv = head(v.data(), 2), ho = head(o.data(), 4), hg = head(g.data(), 4);
	nnh_head_tensor same = ho;
	same.sample = 0;
	nnh_attention_rule r{};
	exhaust("attention forward", NNH_ERR_ALIAS, [&] { return nnh_masked_attention_forward(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &r, &hq, nullptr, lse.data(), nullptr); });
	exhaust("attention forward, out in one place", NNH_ERR_ALIAS, [&] { return nnh_masked_attention_forward(NNH_F32, 2, 8, 8, 4, 2, 16, &hq, &hk, &hv, &r, &same, nullptr, lse.data(), nullptr); });
	exhaust("attention backward", NNH_ERR_ALIAS, [&] { return nnh_masked_attention_backward(NNH_F32, 2, 8, 8, 4, 2, 16, &hg, &hq, &hk, &hv, &ho, nullptr, lse.data(), &r, &hq, 1, nullptr, 1, nullptr, 1, nullptr); });
	exhaust("attention workspace", NNH_ERR_SHAPE, [&] {
		size_t bytes = 0;
		return nnh_masked_attention_workspace_size(2, 8, 8, 4, 3, 16, 1, 1, &bytes);
	});
	std::vector<float> x(128), w(320), out(8), dw(320);
	std::vector<int> t(8);
	exhaust("loss forward", NNH_ERR_ALIAS, [&] { return nnh_linear_cross_entropy_forward(NNH_F32, x.data(), 8, 16, w.data(), 20, nullptr, t.data(), 0, out.data(), out.data(), nullptr); });
	exhaust("loss backward", NNH_ERR_ALIAS, [&] { return nnh_linear_cross_entropy_backward(NNH_F32, nullptr, x.data(), 8, 16, w.data(), 20, nullptr, t.data(), lse.data(), 0, x.data(), 1, dw.data(), 1, nullptr, 1, nullptr); });
	exhaust("loss train", NNH_ERR_ALIAS, [&] { return nnh_linear_cross_entropy_train(NNH_F32, nullptr, x.data(), 8, 16, w.data(), 20, nullptr, t.data(), 0, out.data(), x.data(), 1, dw.data(), 1, nullptr, 1, nullptr); });
	exhaust("loss workspace", NNH_ERR_INVALID, [&] {
		size_t bytes = 0;
		return nnh_linear_cross_entropy_workspace_size(NNH_F32, 8, 4, 5, 3, 0, &bytes);
	});
	nnh_adamw a{};
	a.bits = 32;
	a.beta1 = 0.9;
	a.beta2 = 0.99;
	a.step = 1;
	const nnh_adamw_tensor one{big.data(), big.data() + 32, big.data() + 1024, big.data() + 2048, nullptr, nullptr, nullptr, 64};
	exhaust("adamw", NNH_ERR_ALIAS, [&] { return nnh_adamw_step(&a, &one, 1, nullptr); });
	if (g_failures) return 1;
	std::printf("without memory: %d calls, each with a code\n", g_calls);
	return 0;
}
