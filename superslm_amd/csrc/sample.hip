// The next token by sampling (cache_ops.h): kernels, launches and the C entry.
#include <hip/hip_runtime.h>

#include "../../include/sslm_hip.h"
#include "attention_util.h"
#include "cache_ops.h"
#include "entry_util.h"

namespace sslm {

using sslm_launch::SampleArgs;
using sslm_launch::Sampling;

// ceil(total share / 2^16) and floor(total random / 2^32) for totals below 2^62
__device__ __forceinline__ uint64_t share_of(uint64_t total, uint32_t share) { return (total >> 16) * share + (((total & 0xffff) * share + 0xffff) >> 16); }
__device__ __forceinline__ uint64_t random_of(uint64_t total, uint32_t random) { return (total >> 32) * random + (((total & 0xffffffffu) * random) >> 32); }

__device__ __forceinline__ bool sampling_ok(const Sampling& s, int vocab) {
	if (s.q_ln2 < 1 || s.q_b < 0 || s.q_b >= ((int64_t)1 << 24) || s.q_ln2 > 2 * s.q_b + 1 || s.q_c < 0 || s.q_c > ((int64_t)1 << 47)) return false;
	const int64_t w0 = s.q_b * s.q_b + s.q_c;
	return w0 >= 1 && w0 <= ((int64_t)1 << 47) && __umul64hi(w0, vocab) == 0 && (uint64_t)w0 * vocab < (uint64_t)1 << 62 && s.top_k >= 0 && s.top_p >= 0 && s.top_p <= 65536 &&
	       s.min_p >= 0 && s.min_p <= 65536;
}

// The weight of a logit d below the row's largest, in doubles, each value exact: sa_exp's form (attention_util.h)
// for a d of up to 2^32, and nothing from 30 q_ln2 on.
struct Weight {
	double ninv, half, l, b, c;
	int64_t lim;
};
__device__ __forceinline__ Weight weight_of(const Sampling& s) {
	Weight w;
	w.l = (double)s.q_ln2;
	w.ninv = 1.0 / w.l;
	w.half = 0.5 * w.ninv;
	w.b = (double)s.q_b;
	w.c = (double)s.q_c;
	w.lim = 30 * s.q_ln2;
	return w;
}
__device__ __forceinline__ uint64_t weight(const Weight& w, uint32_t d) {
	if ((int64_t)d >= w.lim) return 0;
	const double x = (double)d, z = floor(fma(x, w.ninv, w.half)), base = fma(z, w.l, w.b - x);
	return (uint64_t)ldexp(fma(base, base, w.c), -(int)z);
}

constexpr int kSampleBlock = 1024;

// A block per row.
__global__ __launch_bounds__(kSampleBlock) void k_sample_row(SampleArgs a) {
	__shared__ unsigned long long s_hist[256], s_sum[kSampleBlock / 64];
	__shared__ int s_top, s_at;
	__shared__ uint32_t s_digit;
	__shared__ unsigned long long s_below;
	const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
	const Sampling s = a.rules[r];
	const int32_t* row = a.logits + (int64_t)r * a.ld;
	if (!sampling_ok(s, a.vocab)) {
		if (tid == 0) {
			a.tokens[r] = -2;
			if (a.mass) a.mass[2 * r] = a.mass[2 * r + 1] = 0;
		}
		return;
	}
	auto legal = [&](int i) { return !s.mask || (global_ptr(s.mask)[i >> 3] >> (i & 7) & 1); };
	if (tid == 0) {
		s_top = INT32_MIN;
		s_at = 0;
	}
	__syncthreads();
	int top = INT32_MIN;
	bool any = false;
	for (int i = tid; i < a.vocab; i += kSampleBlock)
		if (legal(i)) {
			top = max(top, row[i]);
			any = true;
		}
	if (any) {
		atomicMax(&s_top, top);
		s_at = 1;
	}
	__syncthreads();
	if (!s_at) {
		if (tid == 0) {
			a.tokens[r] = -1;
			if (a.mass) a.mass[2 * r] = a.mass[2 * r + 1] = 0;
		}
		return;
	}
	top = s_top;
	const Weight w = weight_of(s);
	const uint64_t least = share_of((uint64_t)(s.q_b * s.q_b + s.q_c), s.min_p);
	// the first ones of the order so far: (d, index) up to (dcut, icut)
	uint32_t dcut = 0xffffffffu;
	int icut = a.vocab;
	enum { COUNT, WEIGHT, KEPT };
	auto measure = [&](int what, uint32_t d) -> uint64_t {
		if (what == COUNT) return 1;
		const uint64_t x = weight(w, d);
		return what == KEPT && x < least ? 0 : x;
	};
	auto inside = [&](int i, uint32_t* d) {
		if (!legal(i)) return false;
		*d = (uint32_t)top - (uint32_t)row[i];
		return *d < dcut || (*d == dcut && i <= icut);
	};
	auto total = [&](int what) {
		uint64_t x = 0;
		uint32_t d;
		for (int i = tid; i < a.vocab; i += kSampleBlock)
			if (inside(i, &d)) x += measure(what, d);
		for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
		__syncthreads();
		if (lane == 0) s_sum[wave] = x;
		__syncthreads();
		x = 0;
		for (int i = 0; i < kSampleBlock / 64; ++i) x += s_sum[i];
		return x;
	};
	// the cut moves to the first element whose running measure reaches goal, 1 <= goal <= the total
	auto select = [&](int what, uint64_t goal) {
		uint32_t prefix = 0;
		for (int shift = 24; shift >= 0; shift -= 8) {
			__syncthreads();
			if (tid < 256) s_hist[tid] = 0;
			__syncthreads();
			uint32_t d;
			for (int i = tid; i < a.vocab; i += kSampleBlock)
				if (inside(i, &d) && (shift == 24 || d >> (shift + 8) == prefix >> (shift + 8))) atomicAdd(&s_hist[d >> shift & 255], (unsigned long long)measure(what, d));
			__syncthreads();
			if (tid == 0) {
				uint64_t run = 0;
				int b = 0;
				while (b < 255 && run + s_hist[b] < goal) run += s_hist[b++];
				s_digit = b;
				s_below = run;
			}
			__syncthreads();
			prefix |= s_digit << shift;
			goal -= s_below;
		}
		// the goal's place among the equal ones, which lie in index order
		const uint64_t each = measure(what, prefix);
		const int place = (int)((goal + each - 1) / each), per = (a.vocab + kSampleBlock - 1) / kSampleBlock;
		int n = 0;
		uint32_t d;
		const int i0 = tid * per, i1 = min(a.vocab, i0 + per);
		for (int i = i0; i < i1; ++i) n += inside(i, &d) && d == prefix;
		int x = n;
		for (int o = 1; o < 64; o *= 2) {
			const int y = __shfl_up(x, o, 64);
			x += lane >= o ? y : 0;
		}
		if (lane == 63) s_sum[wave] = x;
		__syncthreads();
		int before = x - n;
		for (int i = 0; i < wave; ++i) before += (int)s_sum[i];
		if (before < place && before + n >= place)
			for (int i = i0; i < i1; ++i)
				if (inside(i, &d) && d == prefix && ++before == place) s_at = i;
		__syncthreads();
		dcut = prefix;
		icut = s_at;
	};
	if (s.top_k > 0 && (uint64_t)s.top_k < total(COUNT)) select(COUNT, s.top_k);
	if (s.top_p < 65536) {
		const uint64_t need = share_of(total(WEIGHT), s.top_p);
		select(WEIGHT, need < 1 ? 1 : need);
	}
	const uint64_t all = total(KEPT);
	select(KEPT, random_of(all, s.random) + 1);
	if (tid == 0) {
		a.tokens[r] = icut;
		if (a.mass) {
			a.mass[2 * r] = (int64_t)weight(w, dcut);
			a.mass[2 * r + 1] = (int64_t)all;
		}
	}
}

}  // namespace sslm

namespace sslm_launch {

size_t sample_workspace(int rows, int vocab) { return up256((size_t)rows * 8); }

void sample_tokens(const SampleArgs& a, hipStream_t s) { hipLaunchKernelGGL(k_sample_row, dim3(a.rows), dim3(kSampleBlock), 0, s, a); }

}  // namespace sslm_launch

using namespace sslm_launch;

extern "C" {

size_t sslm_hip_sample_workspace(int32_t rows, int32_t vocab) {
	return rows < 1 || rows > kMaxRows || vocab < 1 || vocab > SSLM_HIP_SAMPLE_MAX_VOCAB ? 0 : sample_workspace(rows, vocab);
}

sslm_status sslm_hip_sample_tokens(const sslm_hip_sample_args* p, void* workspace, size_t workspace_bytes, void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_sample_workspace(p->rows, p->vocab);
	if (!need || !p->logits || !p->rules || !p->tokens || p->logits_ld < p->vocab || (uintptr_t)p->logits % 4) return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	static_assert(sizeof(sslm_hip_sampling) == sizeof(Sampling), "one layout");
	const SampleArgs a{p->rows, p->vocab, p->logits, p->logits_ld, (const Sampling*)p->rules, p->tokens, p->mass, workspace};
	return on_stream(stream, [&](hipStream_t s) { sample_tokens(a, s); });
}

}  // extern "C"
