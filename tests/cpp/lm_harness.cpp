// lm_harness.cpp - TEST CODE: a language model's training steps through include/nn_hip_modules.hpp (Transformer::loss over
// packed documents, backward, AdamW), and the graphs of masked_attention and linear_cross_entropy alone, for
// tests/test_lm_training.py. Return codes: 0 ok, 2 nn::hip::TensorShapeError, 1 any other exception.
#include <cstring>
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

size_t append(const Tensor& t, float* to, size_t at) {
	if (to) t.to_host(to + at);
	return at + t.size();
}

}  // namespace

extern "C" {

const char* lm_last_error(void) { return g_last_error.c_str(); }

// `steps` training steps of a Transformer on one batch; docs null: one document a row, with the attention op. losses {steps},
// the parameters before and after, and the first step's gradients, all parameters in turn; count: their elements.
int lm_train(size_t vocab, size_t dim, size_t heads, size_t layers, size_t N, size_t T, const float* ids, const int* targets,
             const int* docs, float cap, const float* slopes, int bits, double lr, size_t steps, float* losses, float* before,
             float* grads, float* after, size_t* count) {
	return guard([&] {
		manual_seed(99);
		TransformerConfig c{vocab, dim, heads, layers, T};
		c.learned_positions = true;
		Transformer model(c);
		const std::vector<Value> parameters = model.parameters();
		AdamWOptions o;
		o.lr = lr;
		o.bits = bits;
		AdamW optimizer(parameters, o);
		const Value x = Value::leaf(Tensor::from_host({N, T}, ids));
		const IntTensor y = IntTensor::from_host({N, T}, targets);
		AttentionRule rule;
		rule.cap = cap;
		if (slopes) rule.slopes = Tensor::from_host({heads}, slopes);
		if (docs) rule.q_docs = rule.k_docs = IntTensor::from_host({N, T}, docs);
		synchronize();
		size_t at = 0;
		for (const Value& p : parameters) at = append(p.data(), before, at);
		*count = at;
		for (size_t s = 0; s < steps; ++s) {
			optimizer.zero_grad();
			Value loss = docs ? model.loss(x, y, rule) : model.loss(x, y);
			loss.backward();
			loss.data().to_host(losses + s);
			if (s == 0) {
				at = 0;
				for (const Value& p : parameters) at = append(p.grad(), grads, at);
			}
			optimizer.step();
		}
		at = 0;
		for (const Value& p : parameters) at = append(p.data(), after, at);
	});
}

// Self-attention with one node as query, key and value (the three gradients added up), and a loss over it.
int lm_shared(size_t N, size_t T, size_t heads, size_t dim, const float* x, size_t vocab, const float* w, const int* targets,
              float* loss, float* dx, float* dw) {
	return guard([&] {
		const Value a = Value::leaf(Tensor::from_host({N, T, dim}, x), true), b = Value::leaf(Tensor::from_host({vocab, dim}, w), true);
		const IntTensor y = IntTensor::from_host({N, T}, targets);
		AttentionRule rule;
		rule.causal = true;
		Value l = linear_cross_entropy(masked_attention(a, a, a, heads, heads, rule), b, Value(), y);
		l.backward();
		l.data().to_host(loss);
		a.grad().to_host(dx);
		b.grad().to_host(dw);
	});
}

// Calls that must throw: 0 shapes of masked_attention, 1 an option's shape, 2 shapes of linear_cross_entropy, 3 AdamW's bits.
int lm_refused(int which) {
	return guard([&] {
		const Value a = Value::leaf(Tensor::empty({2, 3, 8})), b = Value::leaf(Tensor::empty({2, 3, 6})), w = Value::leaf(Tensor::empty({5, 8}));
		AttentionRule rule;
		const int one[1] = {0};
		if (which == 0) masked_attention(a, b, b, 2, 2, rule);
		if (which == 1) {
			rule.k_lens = IntTensor::from_host({1}, one);
			masked_attention(a, a, a, 2, 2, rule);
		}
		if (which == 2) linear_cross_entropy(a, w, Value(), IntTensor::from_host({1}, one));
		if (which == 3) {
			AdamWOptions o;
			o.bits = 16;
			AdamW optimizer({a}, o);
		}
	});
}

}  // extern "C"
