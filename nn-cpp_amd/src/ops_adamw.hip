// ops_adamw.hip - extern "C" entry point of the AdamW step (include/nnh.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "abi_common.hpp"
#include "kernels/hip/adamw.hpp"
#include "nnh.h"

using namespace nnh;

namespace {

// A range that the step reads (out false) or writes.
struct Range {
	uintptr_t from, to;
	bool out;
};

// No written range overlaps another range, the same tensor given twice included.
bool apart(std::vector<Range>& r) {
	std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.from < y.from; });
	uintptr_t end = 0, out_end = 0;  // the furthest end so far, and of what is written
	for (const Range& x : r) {
		if (x.from < out_end || (x.out && x.from < end)) return false;
		end = std::max(end, x.to);
		if (x.out) out_end = std::max(out_end, x.to);
	}
	return true;
}

int step(const nnh_adamw* o, const nnh_adamw_tensor* tensors, size_t n, void* stream) {
	if (!o || (n > 0 && !tensors)) return fail(NNH_ERR_INVALID, "adamw: null pointer");
	if ((o->p_type != NNH_F32 && o->p_type != NNH_BF16) || (o->g_type != NNH_F32 && o->g_type != NNH_BF16))
		return fail(NNH_ERR_INVALID, "adamw: no such element type");
	if (o->bits != 32 && o->bits != 8) return fail(NNH_ERR_INVALID, "adamw: moments are kept in 32 or 8 bits");
	const auto share = [](double b) { return b >= 0.0 && b < 1.0; };
	if (!share(o->beta1) || !share(o->beta2) || !(o->eps >= 0.0) || !std::isfinite(o->eps) || !std::isfinite(o->lr) ||
	    !std::isfinite(o->weight_decay))
		return fail(NNH_ERR_INVALID, "adamw: the betas must be in [0, 1), eps not negative, lr and weight_decay finite");
	if (!o->step_device && o->step == 0) return fail(NNH_ERR_INVALID, "adamw: steps count from 1");
	if (off_words({o->step_device, o->lr_device, o->grad_scale})) return fail(NNH_ERR_INVALID, "adamw: a pointer is not aligned to its elements");
	const uint64_t ps = o->p_type == NNH_F32 ? 4 : 2, gs = o->g_type == NNH_F32 ? 4 : 2, ss = o->bits == 32 ? 4 : 1;
	std::vector<AdamWTensor> t;
	std::vector<Range> ranges;
	t.reserve(n);
	ranges.reserve(7 * n + 3);
	const auto add = [&](const void* p, uint64_t bytes, bool out) {
		if (p) ranges.push_back({reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes, out});
	};
	add(o->step_device, 4, false);
	add(o->lr_device, 4, false);
	add(o->grad_scale, 4, false);
	for (size_t i = 0; i < n; ++i) {
		const nnh_adamw_tensor& x = tensors[i];
		if (x.count == 0) continue;
		if (!count_ok({x.count})) return fail(NNH_ERR_INVALID, "adamw: size out of range (above 2^60 elements)");
		if (!x.p || !x.g || !x.m || !x.v || (o->bits == 8 && (!x.m_scale || !x.v_scale))) return fail(NNH_ERR_INVALID, "adamw: null pointer");
		const auto off = [](const void* p, uint64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; };
		if (off(x.p, ps) || off(x.g, gs) || off(x.m, ss) || off(x.v, ss) || off(x.copy, 2))
			return fail(NNH_ERR_INVALID, "adamw: a pointer is not aligned to its elements");
		add(x.p, x.count * ps, true);
		add(x.g, x.count * gs, false);
		add(x.m, x.count * ss, true);
		add(x.v, x.count * ss, true);
		if (o->bits == 8) {
			add(x.m_scale, (x.count + 63) / 64, true);
			add(x.v_scale, (x.count + 63) / 64, true);
		}
		add(x.copy, x.count * 2, true);
		t.push_back({x.p, x.g, x.m, x.v, x.m_scale, x.v_scale, x.copy, (int64_t)x.count});
	}
	if (!apart(ranges)) return fail(NNH_ERR_ALIAS, "adamw: what the step writes overlaps something else that it uses");
	AdamWArgs a{};
	a.beta1 = o->beta1;
	a.beta2 = o->beta2;
	a.lr = o->lr;
	a.decay = o->weight_decay;
	a.eps = o->eps;
	a.first = 1.0 - std::pow(o->beta1, (double)o->step);
	a.second = 1.0 - std::pow(o->beta2, (double)o->step);
	a.log1 = std::log2(o->beta1);  // beta 0: -infinity, and 2^-infinity is the 0 that its powers are
	a.log2 = std::log2(o->beta2);
	a.step_device = o->step_device;
	a.lr_device = o->lr_device;
	a.grad_scale = o->grad_scale;
	return hip_status(adamw_step(a, t.data(), t.size(), o->p_type, o->g_type, o->bits, reinterpret_cast<hipStream_t>(stream)), "adamw");
}

}  // namespace

extern "C" {

int nnh_adamw_step(const nnh_adamw* o, const nnh_adamw_tensor* tensors, size_t n, void* stream) {
	return guarded([&] { return step(o, tensors, n, stream); });
}

}  // extern "C"
