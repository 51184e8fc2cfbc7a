// linear_cross_entropy.hip - what the linear head's cross entropy does beside its products (linear_cross_entropy.hpp):
// statistics joined, scores turned into their gradient, sums. All of it is bound by memory or, for few rows, by latency; every
// sum has a fixed order.
#include "linear_cross_entropy.hpp"

#include <algorithm>

namespace nnh {

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f, kInf = __builtin_huge_valf();
constexpr int kThreads = 256;

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_max(float x) {
	for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
	return x;
}
__device__ __forceinline__ float wave_sum(float x) {
	for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
	return x;
}

__device__ __forceinline__ float loss_of(float lse, float hit, int target, int64_t vocab) {
	return target < 0 ? 0.0f : target >= vocab ? __builtin_nanf("") : lse - hit;
}

// A wave to a row.
__global__ __launch_bounds__(kThreads) void ce_join_kernel(const f32x2* stats, int chunks, const float* hit, const int* targets,
                                                           int64_t rows, int64_t vocab, float* lse, float* loss) {
	const int lane = threadIdx.x & 63;
	const int64_t i = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
	if (i >= rows) return;
	const f32x2* const s = stats + i * chunks;
	float top = -kInf, sum = 0.0f;
	for (int c = lane; c < chunks; c += 64) top = fmaxf(top, s[c][0]);
	top = wave_max(top);
	const float base = top == -kInf ? 0.0f : top * kLog2e;
	for (int c = lane; c < chunks; c += 64) sum += s[c][1] * exp2_of(__builtin_fmaf(s[c][0], kLog2e, -base));
	sum = wave_sum(sum);
	if (lane == 0) {
		const float l = top + logf(sum);
		lse[i] = l;
		if (loss) loss[i] = loss_of(l, targets[i] >= 0 && targets[i] < vocab ? hit[i] : 0.0f, targets[i], vocab);
	}
}

// A group of G threads (a wave, or the workgroup) to a row.
template <int G>
struct Group {
	static constexpr int kRows = kThreads / G;
	template <typename F>
	static __device__ __forceinline__ float all(float x, float* room, F f) {
		x = f(x);
		if (G == 64) return x;
		__syncthreads();
		if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = x;
		__syncthreads();
		return room[threadIdx.x & 3];
	}
};

template <int G>
__global__ __launch_bounds__(kThreads) void ce_rows32_kernel(const float* z, int64_t rows, int64_t cols, int64_t first, int64_t vocab,
                                                             const int* targets, float* running, int more, int last, float* lse, float* loss) {
	__shared__ float room[4];
	const int at = threadIdx.x % G;
	const int64_t i = (int64_t)blockIdx.x * Group<G>::kRows + threadIdx.x / G;
	const bool on = i < rows;
	const float* const row = z + (on ? i : 0) * cols;
	float top = -kInf, sum = 0.0f;
	for (int64_t v = at; v < cols; v += G) top = fmaxf(top, row[v]);
	if (G == 64) {
		top = wave_max(top);
	} else {
		top = Group<G>::all(top, room, wave_max);
		for (int w = 0; w < 4; ++w) top = fmaxf(top, room[w]);
	}
	const float base = top == -kInf ? 0.0f : top * kLog2e;
	for (int64_t v = at; v < cols; v += G) sum += exp2_of(__builtin_fmaf(row[v], kLog2e, -base));
	if (G == 64) {
		sum = wave_sum(sum);
	} else {
		Group<G>::all(sum, room, wave_sum);
		sum = room[0] + room[1] + room[2] + room[3];
	}
	if (!on || at != 0) return;
	const int t = targets[i];
	float hit = t >= first && t < first + cols ? row[t - first] : 0.0f;
	if (more) {
		const float m = running[3 * i], both = fmaxf(m, top), b2 = both == -kInf ? 0.0f : both * kLog2e;
		sum = running[3 * i + 1] * exp2_of(__builtin_fmaf(m, kLog2e, -b2)) + sum * exp2_of(__builtin_fmaf(top, kLog2e, -b2));
		top = both;
		hit += running[3 * i + 2];
	}
	if (last) {
		const float l = top + logf(sum);
		lse[i] = l;
		if (loss) loss[i] = loss_of(l, hit, t, vocab);
	} else {
		running[3 * i] = top;
		running[3 * i + 1] = sum;
		running[3 * i + 2] = hit;
	}
}

template <int G>
__global__ __launch_bounds__(kThreads) void ce_grad32_kernel(float* z, int64_t rows, int64_t cols, int64_t first, const int* targets,
                                                             const float* lse, const float* weight, const float* scale, const float* x,
                                                             float* xs, int64_t D) {
	const int64_t i = (int64_t)blockIdx.x * Group<G>::kRows + threadIdx.x / G;
	if (i >= rows) return;
	if (xs)
		for (int64_t d = threadIdx.x % G; d < D; d += G) xs[i * D + d] = weight[i] == 0.0f ? 0.0f : x[i * D + d];
	float* const row = z + i * cols;
	const float base = lse[i] * kLog2e, w = weight[i], f = w * *scale;
	const int64_t t = (int64_t)targets[i] - first;
	for (int64_t v = threadIdx.x % G; v < cols; v += G) {
		const float p = exp2_of(__builtin_fmaf(row[v], kLog2e, -base));
		row[v] = w == 0.0f ? 0.0f : (v == t ? p - 1.0f : p) * f;
	}
}

// A workgroup to a row, 16-byte words.
__global__ __launch_bounds__(kThreads) void ce_grad16_kernel(__bf16* z, int64_t ldz, int64_t vocab, const f32x2* stats, int chunks, int chunk,
                                                             const int* targets, const float* lse, const float* hit, const float* weight) {
	const int64_t i = blockIdx.x;
	__bf16* const row = z + i * ldz;
	const float w = weight[i], l = lse[i];
	const int t = targets[i];
	for (int64_t v = threadIdx.x * 8; v < ldz; v += kThreads * 8) {
		union {
			u32x4 u;
			__bf16 e[8];
		} x;
		x.u = u32x4{0, 0, 0, 0};
		if (w != 0.0f && v < vocab) {
			x.u = *(const u32x4*)(row + v);
			const float f = exp2_of((stats[i * chunks + v / chunk][0] - l) * kLog2e) * w;
#pragma unroll
			for (int j = 0; j < 8; ++j) x.e[j] = (__bf16)((float)x.e[j] * f);
			if (t >= v && t < v + 8) {  // from the target's own score: a probability near 1 keeps what is left to 1
				const float y = (exp2_of((hit[i] - l) * kLog2e) - 1.0f) * w;
#pragma unroll
				for (int j = 0; j < 8; ++j)
					if (t - v == j) x.e[j] = (__bf16)y;
			}
		}
		*(u32x4*)(row + v) = x.u;
	}
}

// One workgroup: counts and sums in 64 bits, each thread's rows in order, then the threads' in a tree.
__global__ __launch_bounds__(1024) void ce_reduce_kernel(const float* loss, const int* targets, int64_t rows, int64_t vocab, int reduction,
                                                         const float* g, float* total, float* weight, uint64_t* live, float* factor) {
	__shared__ double sums[1024];
	__shared__ int counts[1024];
	double sum = 0.0;
	int count = 0;
	for (int64_t i = threadIdx.x; i < (rows + 63) / 64 * 64; i += 1024) {  // (a wave's 64 rows together)
		const int t = i < rows ? targets[i] : -1;
		const bool on = t >= 0, used = on && t < vocab;
		count += on;
		if (loss && on) sum += (double)loss[i];
		if (weight && i < rows) weight[i] = !used ? 0.0f : reduction == 0 && g ? g[i] : 1.0f;
		const uint64_t word = __ballot(used);
		if (live && (threadIdx.x & 63) == 0) live[i / 64] = word;
	}
	if (reduction == 0) {
		if (factor && threadIdx.x == 0) *factor = 1.0f;
		return;
	}
	sums[threadIdx.x] = sum;
	counts[threadIdx.x] = count;
	__syncthreads();
	for (int d = 512; d; d >>= 1) {
		if (threadIdx.x < d) {
			sums[threadIdx.x] += sums[threadIdx.x + d];
			counts[threadIdx.x] += counts[threadIdx.x + d];
		}
		__syncthreads();
	}
	if (threadIdx.x == 0) {
		const float up = g ? *g : 1.0f;
		if (total) *total = (float)(reduction == 1 ? sums[0] / counts[0] : sums[0]);
		if (factor) *factor = reduction == 2 ? up : counts[0] ? (float)((double)up / counts[0]) : 0.0f;
	}
}

// Sums of a run of rows, a thread to a column.
template <typename T>
__global__ __launch_bounds__(kThreads) void ce_bias_kernel(const T* dz, int64_t ld, int64_t rows, int64_t cols, int64_t per, float* partial) {
	const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x, from = blockIdx.y * per, to = min(from + per, rows);
	if (v >= cols) return;
	float s[8] = {};
	int64_t i = from;
	for (; i + 8 <= to; i += 8)
#pragma unroll
		for (int j = 0; j < 8; ++j) s[j] += (float)dz[(i + j) * ld + v];
	for (; i < to; ++i) s[0] += (float)dz[i * ld + v];
	partial[blockIdx.y * cols + v] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
}

template <typename T>
__global__ __launch_bounds__(kThreads) void ce_bias_join_kernel(const float* partial, int parts, int64_t cols, const float* factor, T* db, int first) {
	const int64_t v = (int64_t)blockIdx.x * kThreads + threadIdx.x;
	if (v >= cols) return;
	float s = 0.0f;
	for (int p = 0; p < parts; ++p) s += partial[p * cols + v];
	if (factor) s *= *factor;
	db[v] = (T)(first ? s : (float)db[v] + s);
}

__global__ __launch_bounds__(kThreads) void pack16_kernel(const uint16_t* src, int64_t lds, uint16_t* dst, int64_t ldd, int64_t rows, int64_t cols) {
	const int64_t x = (int64_t)blockIdx.x * kThreads + threadIdx.x, r = x / ldd, c = x % ldd;
	if (r < rows) dst[x] = c < cols ? src[r * lds + c] : (uint16_t)0;
}

// Rows of bias sums to a part: enough parts to fill the GPU, 64 rows at least.
int64_t bias_rows(int64_t rows, int64_t cols) {
	const int64_t blocks = std::max<int64_t>(1, (cols + kThreads - 1) / kThreads), parts = std::min((512 + blocks - 1) / blocks, (rows + 63) / 64);
	return parts ? (rows + parts - 1) / parts : 1;
}
int64_t bias_parts(int64_t rows, int64_t cols) {
	const int64_t per = bias_rows(rows, cols);
	return (rows + per - 1) / per;
}

}  // namespace

hipError_t pack16(const void* src, int64_t lds, void* dst, int64_t ldd, int64_t rows, int64_t cols, hipStream_t s) {
	constexpr int64_t kRun = (int64_t)1 << 31;  // elements a launch: below 2^32 work-items
	for (int64_t r = 0; r < rows;) {
		const int64_t n = std::min(rows - r, std::max<int64_t>(1, kRun / ldd));
		pack16_kernel<<<(unsigned)((n * ldd + kThreads - 1) / kThreads), kThreads, 0, s>>>((const uint16_t*)src + r * lds, lds, (uint16_t*)dst + r * ldd, ldd, n, cols);
		const hipError_t e = hipGetLastError();
		if (e != hipSuccess) return e;
		r += n;
	}
	return hipSuccess;
}

hipError_t ce_join(const float* stats, int chunks, const float* hit, const int* targets, int64_t rows, int64_t vocab, float* lse, float* loss,
                   hipStream_t s) {
	if (rows == 0) return hipSuccess;
	ce_join_kernel<<<(unsigned)((rows + 3) / 4), kThreads, 0, s>>>((const f32x2*)stats, chunks, hit, targets, rows, vocab, lse, loss);
	return hipGetLastError();
}

hipError_t ce_rows32(const float* z, int64_t rows, int64_t cols, int64_t first, int64_t vocab, const int* targets, float* running, bool more,
                     bool last, float* lse, float* loss, hipStream_t s) {
	if (rows == 0) return hipSuccess;
	if (cols <= 1024) ce_rows32_kernel<64><<<(unsigned)((rows + 3) / 4), kThreads, 0, s>>>(z, rows, cols, first, vocab, targets, running, more, last, lse, loss);
	else ce_rows32_kernel<256><<<(unsigned)rows, kThreads, 0, s>>>(z, rows, cols, first, vocab, targets, running, more, last, lse, loss);
	return hipGetLastError();
}

hipError_t ce_grad32(float* z, int64_t rows, int64_t cols, int64_t first, const int* targets, const float* lse, const float* weight, const float* scale,
                     const float* x, float* xs, int64_t D, hipStream_t s) {
	if (rows == 0) return hipSuccess;
	if (cols <= 1024) ce_grad32_kernel<64><<<(unsigned)((rows + 3) / 4), kThreads, 0, s>>>(z, rows, cols, first, targets, lse, weight, scale, x, xs, D);
	else ce_grad32_kernel<256><<<(unsigned)rows, kThreads, 0, s>>>(z, rows, cols, first, targets, lse, weight, scale, x, xs, D);
	return hipGetLastError();
}

hipError_t ce_grad16(void* z, int64_t ldz, int64_t rows, int64_t vocab, const float* stats, int chunks, int chunk, const int* targets, const float* lse,
                     const float* hit, const float* weight, hipStream_t s) {
	if (rows == 0) return hipSuccess;
	ce_grad16_kernel<<<(unsigned)rows, kThreads, 0, s>>>((__bf16*)z, ldz, vocab, (const f32x2*)stats, chunks, chunk, targets, lse, hit, weight);
	return hipGetLastError();
}

hipError_t ce_reduce(const float* loss, const int* targets, int64_t rows, int64_t vocab, int reduction, const float* g, float* total, float* weight,
                     uint64_t* live, float* factor, hipStream_t s) {
	ce_reduce_kernel<<<1, 1024, 0, s>>>(loss, targets, rows, vocab, reduction, g, total, weight, live, factor);
	return hipGetLastError();
}

size_t ce_bias_partial_floats(int64_t rows, int64_t cols) { return (size_t)(bias_parts(rows, cols) * cols); }

hipError_t ce_bias(const void* dz, int64_t ld, int64_t rows, int64_t cols, int type, const float* factor, void* db, bool first, float* partial,
                   hipStream_t s) {
	if (cols == 0) return hipSuccess;
	const int64_t per = bias_rows(rows, cols), parts = bias_parts(rows, cols);
	const unsigned blocks = (unsigned)((cols + kThreads - 1) / kThreads);
	if (parts > 0) {
		const dim3 grid(blocks, (unsigned)parts);
		if (type == 0) ce_bias_kernel<float><<<grid, kThreads, 0, s>>>((const float*)dz, ld, rows, cols, per, partial);
		else ce_bias_kernel<__bf16><<<grid, kThreads, 0, s>>>((const __bf16*)dz, ld, rows, cols, per, partial);
		const hipError_t e = hipGetLastError();
		if (e != hipSuccess) return e;
	}
	if (type == 0) ce_bias_join_kernel<float><<<blocks, kThreads, 0, s>>>(partial, (int)parts, cols, factor, (float*)db, first);
	else ce_bias_join_kernel<__bf16><<<blocks, kThreads, 0, s>>>(partial, (int)parts, cols, factor, (__bf16*)db, first);
	return hipGetLastError();
}

}  // namespace nnh
