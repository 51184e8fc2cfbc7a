// lm_edges_harness.cpp - TEST CODE: calls of include/nn_hip_modules.hpp's language-model layer that change something between its
// steps, for tests/test_lm_edges.py. Return codes: 0 ok, 2 nn::hip::TensorShapeError, 1 any other exception.
#include <stdexcept>
#include <string>
#include <vector>

#include "nn_hip.hpp"
#include "nn_hip_modules.hpp"

using namespace nn::hip;

namespace {

std::string g_last_error;

template <typename F>
int guard(F f) {
	try {
		f();
		return 0;
	} catch (const TensorShapeError& e) {
		g_last_error = e.what();
		return 2;
	} catch (const std::exception& e) {
		g_last_error = e.what();
		return 1;
	}
}

}  // namespace

extern "C" {

const char* edges_last_error(void) { return g_last_error.c_str(); }

// A step of AdamW over a parameter of n elements, and another after a change: 0 none, 1 the options' bits are the other kind, 2 the
// parameter has twice its elements (and a gradient like it), 3 half of them. The parameter after the steps that ran into p {n}.
int edges_adamw_changed(size_t n, int bits, int change, float* p, size_t* steps) {
	return guard([&] {
		const std::vector<float> ones(2 * n, 1.0f);
		const Value v = Value::leaf(Tensor::from_host({n}, ones.data()), true);
		bool first = false;
		v.grad_accum(first).fill_(0.5f);
		AdamWOptions o;
		o.bits = bits;
		AdamW optimizer({v}, o);
		optimizer.step();
		v.data().to_host(p);
		const size_t now = change == 2 ? 2 * n : change == 3 ? n / 2 : n;
		if (change == 1) optimizer.options().bits = 40 - bits;
		if (change > 1) {
			v.data() = Tensor::from_host({now}, ones.data());
			v.grad() = Tensor::from_host({now}, ones.data());
		}
		try {
			optimizer.step();
			v.data().to_host(p);
		} catch (...) {
			*steps = optimizer.steps();
			throw;
		}
		*steps = optimizer.steps();
	});
}

// linear_cross_entropy over nodes that are given twice: which 0 x is the weight too ({V, D}), 1 x of one row is the bias too (x {D}, bias
// {V}, D = V), 2 all apart. add: the leaves' gradients hold ones before. loss {1}, and the gradients of x, weight and bias (of a node
// given twice: the sum, in its first place).
int edges_loss_shared(int which, int add, size_t V, size_t D, const float* x, const float* w, const float* b, const int* targets, float* loss,
                      float* dx, float* dw, float* db) {
	return guard([&] {
		const size_t rows = which == 1 ? 1 : V;
		const Value X = Value::leaf(Tensor::from_host(which == 1 ? std::vector<size_t>{D} : std::vector<size_t>{rows, D}, x), true);
		const Value W = which == 0 ? X : Value::leaf(Tensor::from_host({V, D}, w), true);
		const Value B = which == 1 ? X : Value::leaf(Tensor::from_host({V}, b), true);
		const IntTensor y = IntTensor::from_host(which == 1 ? std::vector<size_t>{} : std::vector<size_t>{rows}, targets);
		bool first = false;
		if (add)
			for (const Value* v : {&X, &W, &B}) v->grad_accum(first).fill_(1.0f);
		Value l = linear_cross_entropy(X, W, B, y);
		l.backward();
		l.data().to_host(loss);
		X.grad().to_host(dx);
		if (which != 0) W.grad().to_host(dw);
		if (which != 1) B.grad().to_host(db);
	});
}

}  // extern "C"
