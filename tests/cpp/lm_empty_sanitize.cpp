// lm_empty_sanitize.cpp - TEST CODE: the masked attention entry points of include/nnh.h with documents where one side has no
// elements, whose array may then be null, on the host (as lm_sanitize.cpp: valid calls come back NNH_OK, with nothing to do, or
// NNH_ERR_HIP from the runtime). Exit status 77 when a GPU is visible.
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

}  // namespace

int main() {
	int devices = 0;
	if (hipGetDeviceCount(&devices) == hipSuccess && devices > 0) {
		std::printf("skipped: a GPU is visible (this test passes host buffers where device pointers belong)\n");
		return 77;
	}
	std::vector<float> q(1024), k(512), v(512), o(1024), g(1024), dq(1024), dk(512), dv(512), lse(64);
	std::vector<int> docs(16);
	const auto head = [](float* p, size_t heads) { return nnh_head_tensor{p, 8 * heads * 16, heads * 16, 16}; };
	const nnh_head_tensor hq = head(q.data(), 4), hk = head(k.data(), 2), hv = head(v.data(), 2), ho = head(o.data(), 4),
	                      hg = head(g.data(), 4), hdq = head(dq.data(), 4), hdk = head(dk.data(), 2), hdv = head(dv.data(), 2);
	for (int which = 0; which < 4; ++which) {  // the arrays given: none, the queries', the keys', both
		nnh_attention_rule r{};
		r.q_docs = which & 1 ? docs.data() : nullptr;
		r.k_docs = which & 2 ? docs.data() : nullptr;
		const auto fwd = [&](size_t N, size_t Tq, size_t Tk) {
			return nnh_masked_attention_forward(NNH_F32, N, Tq, Tk, 4, 2, 16, Tq ? &hq : nullptr, Tk ? &hk : nullptr, Tk ? &hv : nullptr, &r, Tq ? &ho : nullptr, nullptr, lse.data(), nullptr);
		};
		const auto bwd = [&](size_t N, size_t Tq, size_t Tk) {
			return nnh_masked_attention_backward(NNH_F32, N, Tq, Tk, 4, 2, 16, &hg, &hq, &hk, &hv, &ho, nullptr, lse.data(), &r, &hdq, 1, &hdk, 1, &hdv, 1, nullptr);
		};
		expect("forward, no keys", fwd(2, 8, 0), NNH_ERR_HIP);
		expect("forward, no queries", fwd(2, 0, 8), NNH_OK);
		expect("forward, no samples", fwd(0, 8, 8), NNH_OK);
		expect("backward, no keys", bwd(2, 8, 0), NNH_ERR_HIP);
		expect("backward, no queries", bwd(2, 0, 8), NNH_ERR_HIP);
		expect("backward, no samples", bwd(0, 8, 8), NNH_OK);
		const int both = which == 0 || which == 3 ? NNH_ERR_HIP : NNH_ERR_INVALID;
		expect("forward", fwd(2, 8, 8), both);
		expect("backward", bwd(2, 8, 8), both);
	}
	if (g_failures) {
		std::fprintf(stderr, "%d of %d calls returned an unexpected code\n", g_failures, g_calls);
		return 1;
	}
	std::printf("empty sides: %d calls, every code as expected\n", g_calls);
	return 0;
}
