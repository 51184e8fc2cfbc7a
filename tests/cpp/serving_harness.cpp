// serving_harness.cpp - TEST CODE: generation through include/nn_hip_modules.hpp (Decoder over a Transformer), and the serving operators
// of include/nn_hip.hpp alone, for tests/test_serving_gpu.py. Return codes: 0 ok, 2 nn::hip::TensorShapeError, 3 std::invalid_argument,
// 1 any other exception.
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
	} catch (const std::invalid_argument& e) {
		g_last_error = e.what();
		return 3;
	} catch (const std::exception& e) {
		g_last_error = e.what();
		return 1;
	}
}

Transformer model_of(size_t vocab, size_t dim, size_t heads, size_t layers, size_t max_len, bool learned) {
	manual_seed(41);
	TransformerConfig c{vocab, dim, heads, layers, max_len};
	c.learned_positions = learned;
	return Transformer(c);
}

Tensor maybe(size_t rows, const float* p) { return p ? Tensor::from_host({rows}, p) : Tensor(); }

}  // namespace

extern "C" {

const char* serving_last_error(void) { return g_last_error.c_str(); }

// The parameters in turn, then `steps` steps: turns[s] turns each, a turn being a sequence, a count of tokens and these; a count of 0
// drops the sequence. logits: {vocab} of every turn with tokens, in order; whole: the same rows of the model's own forward over all of the
// sequence's tokens (fp32). free: pages left at the end.
int serving_steps(size_t vocab, size_t dim, size_t heads, size_t layers, size_t max_len, int learned, size_t sequences, size_t page_size,
                  size_t pages, int int8, size_t steps, const int* turns, const int* sequence, const int* count, const int* tokens,
                  float* parameters, size_t* elements, float* logits, float* whole, size_t* left) {
	return guard([&] {
		Transformer model = model_of(vocab, dim, heads, layers, max_len, learned != 0);
		*elements = 0;
		for (const Value& p : model.parameters()) {
			p.data().to_host(parameters + *elements);
			*elements += p.data().size();
		}
		DecoderOptions o;
		o.sequences = sequences;
		o.page_size = page_size;
		o.pages = pages;
		o.int8 = int8 != 0;
		Decoder decoder(model, o);
		std::vector<std::vector<float>> all(sequences);
		for (size_t s = 0; s < steps; ++s) {
			std::vector<Decoder::Turn> step;
			for (int t = 0; t < turns[s]; ++t, ++sequence, ++count) {
				if (*count == 0) {
					decoder.drop(*sequence);
					all[*sequence].clear();
					continue;
				}
				step.push_back({static_cast<size_t>(*sequence), std::vector<int>(tokens, tokens + *count)});
				all[*sequence].insert(all[*sequence].end(), tokens, tokens + *count);
				tokens += *count;
			}
			const Tensor y = decoder.step(step);
			y.to_host(logits);
			logits += y.size();
			NoGradGuard none;
			for (const Decoder::Turn& t : step) {
				const std::vector<float>& ids = all[t.sequence];
				if (decoder.length(t.sequence) != ids.size()) throw std::runtime_error("a sequence's length");
				const std::vector<float> z = model.forward(Value::leaf(Tensor::from_host({1, ids.size()}, ids.data()))).data().to_host();
				std::copy(z.end() - vocab, z.end(), whole);
				whole += vocab;
			}
		}
		*left = decoder.free_pages();
	});
}

// `count` tokens to each of N prompts of `length` tokens, the first largest ones or, with a temperature, drawn.
int serving_generate(size_t vocab, size_t dim, size_t heads, size_t layers, size_t max_len, int int8, size_t N, size_t length, const int* tokens,
                     size_t count, float temperature, int top_k, int* out) {
	return guard([&] {
		Transformer model = model_of(vocab, dim, heads, layers, max_len, true);
		DecoderOptions o;
		o.sequences = N;
		o.page_size = 16;
		o.int8 = int8 != 0;
		Decoder decoder(model, o);
		std::vector<Decoder::Turn> prompts;
		for (size_t n = 0; n < N; ++n) prompts.push_back({n, std::vector<int>(tokens + n * length, tokens + (n + 1) * length)});
		SampleRule rule;
		rule.temperature = Tensor({N}, temperature);
		const std::vector<int> k(N, top_k);
		rule.top_k = IntTensor::from_host({N}, k.data());
		for (const std::vector<int>& t : decoder.generate(prompts, count, rule)) out = std::copy(t.begin(), t.end(), out);
	});
}

int serving_sample(size_t rows, size_t V, const float* logits, const float* u, const float* temperature, const int* top_k, const float* top_p,
                   const float* min_p, int* tokens, float* logprob) {
	return guard([&] {
		SampleRule rule{maybe(rows, temperature), maybe(rows, top_p), maybe(rows, min_p), top_k ? IntTensor::from_host({rows}, top_k) : IntTensor()};
		Tensor share;
		const std::vector<int> t = sample(Tensor::from_host({rows, V}, logits), Tensor::from_host({rows}, u), rule, &share).to_host();
		std::copy(t.begin(), t.end(), tokens);
		share.to_host(logprob);
	});
}

// Calls that must throw (the codes are in the test); none of them launches a kernel with what it is given.
int serving_refused(int which) {
	return guard([&] {
		Transformer model = model_of(31, 32, 2, 1, 40, false);
		DecoderOptions o;
		o.sequences = 2;
		o.page_size = 16;
		o.pages = 3;
		Decoder decoder(model, o);
		const std::vector<int> many(41, 1), most(40, 1);
		if (which == 0) decoder.step({{2, {1}}});
		if (which == 1) decoder.step({{0, {1}}, {0, {2}}});
		if (which == 2) decoder.step({{0, {}}});
		if (which == 3) decoder.step({{0, {31}}});
		if (which == 4) decoder.step({{0, {-1}}});
		if (which == 5) decoder.step({{0, many}});
		if (which == 6) decoder.step({{0, most}, {1, {1}}});  // (a fourth page)
		if (which == 7) {
			TransformerConfig c{31, 32, 2, 1, 40};
			c.causal = false;
			Decoder wrong{Transformer(c)};
		}
		if (which == 8) {
			TransformerConfig c{31, 258, 2, 1, 40};
			Decoder wrong{Transformer(c)};
		}
		if (which == 9) {
			o.page_size = 0;
			Decoder wrong(model, o);
		}
		if (which == 10) {
			QuantizedLinear l({Linear(8, 4)});
			l.forward(Value::leaf(Tensor({2, 8}, 1.0f), true));
		}
		if (which == 11) QuantizedLinear l({Linear(8, 4), Linear(9, 4)});
		const Tensor x({4, 12}, 0.0f);
		const int zero[4] = {};
		PagedCache cache(2, 4, 1, 8);
		PagedStep step{IntTensor::from_host({1, 2}, zero), IntTensor::from_host({2}, zero), IntTensor::from_host({1}, zero), 4};
		if (which == 12) paged_append(cache, {x, 5}, x, step);
		if (which == 13) paged_attention(x, cache, 2, step, AttentionRule());
		if (which == 14) {
			AttentionRule rule;
			rule.k_lens = step.lens;
			paged_attention(x, cache, 1, step, rule);
		}
		if (which == 15) {
			step.lens = IntTensor::from_host({2}, zero);
			paged_attention(x, cache, 1, step, AttentionRule());
		}
		if (which == 16) linear_int8(x, quantize({Tensor({3, 8}, 1.0f)}), Tensor());
		if (which == 17) sample(x, Tensor({3}, 0.5f));
		if (which == 18) {
			SampleRule rule;
			rule.top_p = Tensor({3}, 0.5f);
			sample(x, Tensor({4}, 0.5f), rule);
		}
		if (which == 20) decoder.generate({{0, {1, 2}}}, 40);  // 41 tokens
		if (which == 21) decoder.generate({{0, {1}}, {1, {1}}}, 17, SampleRule{Tensor({1}, 1.0f), Tensor(), Tensor(), IntTensor()});
		if (which == 22) decoder.generate({{0, {1}}, {1, {1}}}, 34);  // three pages each
		if (which == 23) decoder.drop(2);
		if (which == 24) decoder.length(2);
		if (which == 19) linear_int8(Tensor({4, 8}, 0.0f), quantize({Tensor({3, 8}, 1.0f)}), Tensor({2}, 0.0f));
	});
}

// A refused step leaves the decoder as it was: the logits of a step after one, and of the same step without.
int serving_after_refusal(float* a, float* b) {
	return guard([&] {
		Transformer model = model_of(31, 32, 2, 1, 40, false);
		for (int refused = 0; refused < 2; ++refused) {
			DecoderOptions o;
			o.sequences = 2;
			o.page_size = 4;
			o.pages = 4;
			Decoder decoder(model, o);
			decoder.step({{0, {1, 2, 3, 4, 5}}});
			if (refused) {
				const std::vector<int> nine(9, 1);
				bool thrown = false;
				try {
					decoder.step({{1, nine}});
				} catch (const std::invalid_argument&) {
					thrown = true;
				}
				if (!thrown || decoder.length(1) != 0 || decoder.free_pages() != 2) throw std::runtime_error("the refused step left something");
			}
			decoder.step({{0, {6, 7, 8}}, {1, {9}}}).to_host(refused ? b : a);
		}
	});
}

}  // extern "C"
