// serving_nomem.cpp - TEST CODE: the serving entry points of include/nnh.h where the host has no memory left. Each call is one that
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
	std::vector<float> q(7 * 64), k(7 * 32), v(7 * 32), lse(28), kp(5 * 8 * 32), vp(5 * 8 * 32), x(20 * 40), s(20), y(20 * 12), u(20);
	std::vector<int> starts(3), lens(2), table(6), tokens(20);
	std::vector<signed char> codes(20 * 48);
	const nnh_head_tensor hq{q.data(), 0, 64, 16}, hk{k.data(), 0, 32, 16}, hv{v.data(), 0, 32, 16}, inside{kp.data(), 0, 32, 16};
	const nnh_paged_cache c{kp.data(), vp.data(), 8 * 32, 32, 16, 5, 8, table.data(), 3};
	nnh_attention_rule r{};
	r.k_lens = lens.data();
	exhaust("append", NNH_ERR_ALIAS, [&] { return nnh_paged_append(NNH_F32, 2, 7, 2, 16, &inside, &hv, starts.data(), lens.data(), &c, nullptr); });
	exhaust("append", NNH_ERR_INVALID, [&] { return nnh_paged_append(NNH_F32, 2, 7, 2, 16, &hk, nullptr, starts.data(), lens.data(), &c, nullptr); });
	exhaust("attention", NNH_ERR_ALIAS, [&] { return nnh_paged_attention(NNH_F32, 2, 7, 4, 4, 2, 16, &hq, &c, starts.data(), &r, &hq, lse.data(), nullptr); });
	exhaust("quantize", NNH_ERR_ALIAS, [&] { return nnh_quantize_rows(NNH_F32, x.data(), 20, 40, 40, codes.data(), 48, x.data(), nullptr); });
	exhaust("linear", NNH_ERR_ALIAS, [&] { return nnh_linear_int8(NNH_F32, x.data(), 20, 0, 40, nullptr, 0, s.data(), 12, y.data(), y.data(), 12, nullptr); });
	exhaust("sample", NNH_ERR_ALIAS, [&] {
		return nnh_sample(NNH_F32, x.data(), 20, 40, 40, u.data(), nullptr, nullptr, nullptr, nullptr, tokens.data(), u.data(), nullptr);
	});
	if (g_failures) return 1;
	std::printf("without memory: %d calls, each with a code\n", g_calls);
	return 0;
}
