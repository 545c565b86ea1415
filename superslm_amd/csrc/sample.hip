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
__device__ __forceinline__ double weight_d(const Weight& w, uint32_t d) {
	const double x = (double)d, z = floor(fma(x, w.ninv, w.half)), base = fma(z, w.l, w.b - x);
	return (int64_t)d >= w.lim ? 0.0 : floor(ldexp(fma(base, base, w.c), -(int)z));
}
__device__ __forceinline__ uint64_t weight(const Weight& w, uint32_t d) { return (uint64_t)weight_d(w, d); }

// Everything a row's sampling asks for is a border in one order, logit descending, then index ascending: the element whose
// running count (top-k), running weight (top-p) or running kept weight (the draw) reaches a goal.  Over the whole row that is a
// radix search, some passes over the vocabulary for each.  Four launches find the same borders with two passes:
//   k_sample_hist    a slice's largest logit, and how many of its logits lie in each bucket of 2^sh below it
//   k_sample_plan    a row's buckets together; from their counts and mean weights where each border must be, within a few buckets
//   k_sample_gather  the exact sums of the weights before those buckets, and the elements in them
//   k_sample_pick    the borders among these elements.  That each lies where it was expected is checked exactly, so an estimate
//                    that misses (or a list that overflows) costs the radix search over the row, not the result.
// Rows of one slice are searched in LDS by k_sample_pick alone.
constexpr int kSampleBlock = 512;
constexpr int kSampleSlice = 8192, kSampleLoads = kSampleSlice / kSampleBlock / 4;
constexpr int kBuckets = 2048, kPlanThreads = 1024;
constexpr int kSampleList = 4096;

// What the plan found: the borders' bucket ranges [a, b), 0 top-k, 1 top-p, 2 the draw (unused ones empty).
struct SamplePlan {
	int32_t top, sh;   // the row's largest logit
	int32_t state;     // 0: to be drawn from the ranges, 1: by the search over the row, -1: no legal token
	int32_t cut_k;     // whether top-k cuts, and how many of its first elements range 0 has
	uint32_t goal_k;
	uint32_t a[3], b[3];
	uint32_t count;    // elements gathered
	// sums before range 0 / 1 / 2, of the weights and of the kept ones; over the whole row where the border is none
	unsigned long long w[2], kept[3];
};

struct SampleWork {
	int64_t* smax;   // [rows][slices] a slice's largest legal logit, or none
	uint16_t* hist;  // [rows][slices][kBuckets]
	SamplePlan* plan;
	uint2* list;     // [rows][kSampleList] (distance from the largest, index)
};
constexpr int64_t kNoLogit = INT64_MIN;

// buckets of 2^sh: all that have a weight lie in the first kBuckets - 2
__device__ __forceinline__ int bucket_shift(const Sampling& s) {
	int sh = 0;
	while (((30 * s.q_ln2) >> sh) + 2 > kBuckets) ++sh;
	return sh;
}

// A thread's logits of a slice: 4 (tid + u kSampleBlock) + i, and a bit for each that is legal.
template <bool VEC>
struct SampleSlice {
	v4i x[kSampleLoads];
	uint32_t legal;
	int v0, n;
	__device__ __forceinline__ void load(const SampleArgs& a, const uint8_t* mask) {
		v0 = blockIdx.x * kSampleSlice;
		n = min(kSampleSlice, a.vocab - v0);
		const int32_t* row = a.logits + (int64_t)blockIdx.y * a.ld + v0;
		legal = 0;
#pragma unroll
		for (int u = 0; u < kSampleLoads; ++u) {
			const int j = 4 * ((int)threadIdx.x + u * kSampleBlock);
			if (VEC && j + 4 <= n) x[u] = *(const v4i*)(row + j);
			else {
#pragma unroll
				for (int i = 0; i < 4; ++i) x[u][i] = row[min(j + i, n - 1)];
			}
			uint32_t m = mask ? global_ptr(mask)[min(v0 + j, a.vocab - 1) >> 3] >> (j & 4) & 15 : 15;
			m &= j + 4 <= n ? 15u : (j < n ? (1u << (n - j)) - 1 : 0u);
			legal |= m << 4 * u;
		}
	}
	__device__ __forceinline__ bool has(int u, int i) const { return legal >> (4 * u + i) & 1; }
	__device__ __forceinline__ int index(int u, int i) const { return v0 + 4 * ((int)threadIdx.x + u * kSampleBlock) + i; }
};

template <bool VEC>
__global__ __launch_bounds__(kSampleBlock) void k_sample_hist(SampleArgs a, SampleWork w) {
	__shared__ uint32_t s_hist[kBuckets];
	__shared__ int32_t s_max[kSampleBlock / 64], s_any[kSampleBlock / 64];
	const int r = blockIdx.y, tid = threadIdx.x;
	const Sampling s = a.rules[r];
	SampleSlice<VEC> sl;
	sl.load(a, s.mask);
	if (!sampling_ok(s, a.vocab)) return;
	for (int i = tid; i < kBuckets; i += kSampleBlock) s_hist[i] = 0;
	int32_t m = INT32_MIN;
#pragma unroll
	for (int u = 0; u < kSampleLoads; ++u)
#pragma unroll
		for (int i = 0; i < 4; ++i) m = sl.has(u, i) ? max(m, sl.x[u][i]) : m;
	m = (int32_t)(wave_max32((uint32_t)m ^ 0x80000000u) ^ 0x80000000u);
	if ((tid & 63) == 0) s_max[tid >> 6] = m;
	const bool any = __any(sl.legal != 0);
	if ((tid & 63) == 0) s_any[tid >> 6] = any;
	__syncthreads();
	bool some = false;
#pragma unroll
	for (int i = 0; i < kSampleBlock / 64; ++i) {
		m = max(m, s_max[i]);
		some |= s_any[i] != 0;
	}
	const size_t at = (size_t)r * gridDim.x + blockIdx.x;
	if (tid == 0) w.smax[at] = some ? (int64_t)m : kNoLogit;
	if (!some) return;
	const int sh = bucket_shift(s), base = m >> sh;
#pragma unroll
	for (int u = 0; u < kSampleLoads; ++u)
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const uint32_t j = (uint32_t)base - (uint32_t)(sl.x[u][i] >> sh);
			if (sl.has(u, i) && j < kBuckets) atomicAdd(&s_hist[j], 1u);
		}
	__syncthreads();
	uint32_t* out = (uint32_t*)(w.hist + at * kBuckets);
	for (int i = tid; i < kBuckets / 2; i += kSampleBlock) out[i] = s_hist[2 * i] | s_hist[2 * i + 1] << 16;
}

// inclusive sums over a block's threads, and the total
template <typename T>
__device__ __forceinline__ T block_scan(T v, T* s, T* total) {
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	for (int o = 1; o < 64; o *= 2) {
		const T y = __shfl_up(v, o, 64);
		v += lane >= o ? y : (T)0;
	}
	__syncthreads();
	if (lane == 63) s[wave] = v;
	__syncthreads();
	T before = 0, all = 0;
	for (int i = 0; i < (int)blockDim.x / 64; ++i) {
		before += i < wave ? s[i] : (T)0;
		all += s[i];
	}
	*total = all;
	return before + v;
}

// A block per row, two neighbouring buckets a thread.  A bucket's weight is estimated by its count times the weight of its middle; that
// is off by a few standard deviations of places spread evenly over the buckets, so a border is looked for six of them around.
__global__ __launch_bounds__(kPlanThreads) void k_sample_plan(SampleArgs a, SampleWork w, int slices) {
	__shared__ int s_i[kPlanThreads / 64], s_a[3], s_b[3];
	__shared__ double s_d[kPlanThreads / 64];
	__shared__ long long s_top;
	const int r = blockIdx.x, tid = threadIdx.x;
	const Sampling s = a.rules[r];
	if (!sampling_ok(s, a.vocab)) return;
	if (tid == 0) s_top = kNoLogit;
	__syncthreads();
	for (int i = tid; i < slices; i += kPlanThreads) atomicMax(&s_top, (long long)w.smax[(size_t)r * slices + i]);
	if (tid < 3) {
		s_a[tid] = kBuckets;
		s_b[tid] = kBuckets;
	}
	__syncthreads();
	SamplePlan p{};
	p.state = -1;
	if (s_top != kNoLogit) {
		p.state = 0;
		p.top = (int32_t)s_top;
		p.sh = bucket_shift(s);
		const int rb = p.top >> p.sh;
		int c[2] = {0, 0};
		for (int i = 0; i < slices; ++i) {
			const int64_t m = w.smax[(size_t)r * slices + i];
			if (m == kNoLogit) continue;
			const uint32_t off = (uint32_t)rb - (uint32_t)((int32_t)m >> p.sh);  // the slice's first bucket
			const uint16_t* h = w.hist + ((size_t)r * slices + i) * kBuckets;
#pragma unroll
			for (int k = 0; k < 2; ++k) {
				const uint32_t j = 2 * tid + k;
				if (j >= off) c[k] += h[j - off];
			}
		}
		const Weight wt = weight_of(s);
		const double least = (double)share_of((uint64_t)(s.q_b * s.q_b + s.q_c), s.min_p);
		// a bucket's estimate, kept estimate and variance
		double e[2], k[2], var = 0.0, doubt = 0.0;
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			const int64_t low = ((int64_t)rb - (2 * tid + i)) * ((int64_t)1 << p.sh);  // its least logit
			const int64_t d1 = p.top - low, d0 = i64max(0, d1 - (((int64_t)1 << p.sh) - 1));
			const double w0 = (double)weight(wt, (uint32_t)i64min(d0, 0xffffffffll)), w1 = (double)weight(wt, (uint32_t)i64min(d1, 0xffffffffll));
			const double mid = 0.5 * (w0 + w1), n = (double)c[i];
			e[i] = n * mid;
			k[i] = mid >= least ? n * mid : 0.0;
			if (w0 >= least && w1 < least) doubt += n * w0;
			var += n * (w0 - w1) * (w0 - w1) * (1.0 / 12);
		}
		int all_c;
		double all_e, all_k, all_v, all_x;
		const int run_c = block_scan(c[0] + c[1], s_i, &all_c);
		const double run_e = block_scan(e[0] + e[1], s_d, &all_e), run_k = block_scan(k[0] + k[1], s_d, &all_k);
		block_scan(var, s_d, &all_v);
		block_scan(doubt, s_d, &all_x);
		// one past bucket i of this thread's
		const int pc[2] = {run_c - c[1], run_c};
		const double pe[2] = {run_e - e[1], run_e}, pk[2] = {run_k - k[1], run_k};
		__shared__ double s_sum, s_kept;
		__shared__ uint32_t s_goal;
		// top-k: exactly its bucket; the estimates up to its border
		const bool cut_k = s.top_k > 0 && s.top_k < all_c;
		if (tid == 0) {
			s_sum = all_e;
			s_kept = all_k;
			s_goal = 0;
		}
		__syncthreads();
		if (cut_k)
#pragma unroll
			for (int i = 0; i < 2; ++i)
				if (pc[i] >= s.top_k && pc[i] - c[i] < s.top_k) {
					const double part = (double)(s.top_k - (pc[i] - c[i])) / (double)c[i];
					s_a[0] = 2 * tid + i;
					s_b[0] = 2 * tid + i + 1;
					s_goal = s.top_k - (pc[i] - c[i]);
					s_sum = pe[i] - e[i] + part * e[i];
					s_kept = pk[i] - k[i] + part * k[i];
				}
		__syncthreads();
		const int end = s_b[0];  // nothing is taken past it
		const double slack = 6.0 * sqrt(all_v) + 1e-9 * all_e;
		double kept = s_kept;
		auto range = [&](int which, const double (&run)[2], const double (&one)[2], double goal, double off) {
			if (tid == 0 && goal - off <= 0.0) s_a[which] = 0;
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				const int j = 2 * tid + i;
				if (run[i] >= goal - off && run[i] - one[i] < goal - off) atomicMin(&s_a[which], max(0, j - 1));
				if (run[i] >= goal + off && run[i] - one[i] < goal + off) atomicMin(&s_b[which], j + 2);
			}
		};
		if (s.top_p < 65536) {
			const double goal = s_sum * s.top_p * (1.0 / 65536);
			range(1, pe, e, goal, slack);
			__syncthreads();
			s_kept = all_k;
			__syncthreads();
			// the kept weight up to there
#pragma unroll
			for (int i = 0; i < 2; ++i)
				if (pe[i] >= goal && pe[i] - e[i] < goal) s_kept = pk[i] - k[i] + (e[i] > 0.0 ? (goal - (pe[i] - e[i])) / e[i] : 0.0) * k[i];
			__syncthreads();
			kept = fmin(kept, s_kept);
		}
		range(2, pk, k, kept * s.random * 0x1p-32, slack + all_x);
		__syncthreads();
		p.cut_k = cut_k;
		p.goal_k = s_goal;
#pragma unroll
		for (int i = 0; i < 3; ++i) {
			p.a[i] = min(s_a[i], end - 1);
			p.b[i] = max(min(s_b[i], end), (int)p.a[i]);
		}
		if (!cut_k) p.a[0] = p.b[0] = kBuckets;
		if (s.top_p >= 65536) p.a[1] = p.b[1] = kBuckets;
		// how much would be gathered
		int n = 0;
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			const uint32_t j = 2 * tid + i;
			bool in = false;
#pragma unroll
			for (int x = 0; x < 3; ++x) in |= j >= p.a[x] && j < p.b[x];
			n += in ? c[i] : 0;
		}
		int sum;
		block_scan(n, s_i, &sum);
		if (sum > kSampleList) p.state = 1;
	}
	if (tid == 0) w.plan[r] = p;
}

template <bool VEC>
__global__ __launch_bounds__(kSampleBlock) void k_sample_gather(SampleArgs a, SampleWork w) {
	__shared__ unsigned long long s_sum[5];
	const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
	const Sampling s = a.rules[r];
	SampleSlice<VEC> sl;
	sl.load(a, s.mask);
	if (!sampling_ok(s, a.vocab)) return;
	const SamplePlan& p = w.plan[r];
	if (p.state != 0) return;
	const int32_t top = p.top, sh = p.sh, rb = top >> sh;
	const uint32_t a0 = p.a[0], a1 = p.a[1], a2 = p.a[2], b0 = p.b[0], b1 = p.b[1], b2 = p.b[2];
	// the sums that the borders need: 0, 1 weights before ranges 0 and 1; 2, 3, 4 kept weights before 0, 1 and 2
	const bool by_p = s.top_p < 65536;
	const uint32_t upto[5] = {by_p ? a0 : 0, by_p ? a1 : 0, by_p ? 0 : a0, by_p ? a1 : 0, a2};
	uint32_t most = 0;
#pragma unroll
	for (int i = 0; i < 5; ++i) most = max(most, upto[i]);
	if (tid < 5) s_sum[tid] = 0;
	__syncthreads();
	const Weight wt = weight_of(s);
	const uint64_t w0 = (uint64_t)(s.q_b * s.q_b + s.q_c);
	const double least = (double)share_of(w0, s.min_p);
	double acc[5] = {};
#pragma unroll
	for (int u = 0; u < kSampleLoads; ++u)
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const uint32_t j = (uint32_t)rb - (uint32_t)(sl.x[u][i] >> sh);
			const bool has = sl.has(u, i);
			if (__any(has && j < most)) {
				const double x = weight_d(wt, (uint32_t)top - (uint32_t)sl.x[u][i]), y = x >= least ? x : 0.0;
#pragma unroll
				for (int k = 0; k < 5; ++k) acc[k] += has && j < upto[k] ? (k < 2 ? x : y) : 0.0;  // 16 values of 2^47
			}
			const bool in = has && ((j >= a0 && j < b0) || (j >= a1 && j < b1) || (j >= a2 && j < b2));
			const uint64_t who = __ballot(in);
			if (who) {
				uint32_t at = 0;
				if (lane == __builtin_ctzll(who)) at = atomicAdd(&w.plan[r].count, (uint32_t)__popcll(who));
				at = __builtin_amdgcn_readlane(at, __builtin_ctzll(who)) + __popcll(who & ((1ull << lane) - 1));
				if (in && at < kSampleList) w.list[(size_t)r * kSampleList + at] = uint2{(uint32_t)top - (uint32_t)sl.x[u][i], (uint32_t)sl.index(u, i)};
			}
		}
#pragma unroll
	for (int k = 0; k < 5; ++k) {
		if (!upto[k]) continue;
		int64_t x = (int64_t)acc[k];
		x = row16_sum(x);
		x += __shfl_xor(x, 16, 64);
		x += __shfl_xor(x, 32, 64);
		if (lane == 0 && x) atomicAdd(&s_sum[k], (unsigned long long)x);
	}
	__syncthreads();
	if (tid < 5 && s_sum[tid]) atomicAdd(tid < 2 ? &w.plan[r].w[tid] : &w.plan[r].kept[tid - 2], s_sum[tid]);
}

struct BorderShared {
	unsigned long long m[256], below, key;
	uint32_t c[256], digit, one, found;
	unsigned long long sum[kSampleBlock / 64];
};

// The element whose running measure reaches `goal` among those that get(i, d, index) admits of `n`, by radix over the key
// (d - d0, index), d - d0 below 2^bits: a byte a pass until one element is left.  False when there is none.
template <typename G, typename M>
__device__ __forceinline__ bool find_border(int n, G&& get, M&& measure, uint64_t goal, uint32_t d0, int bits, BorderShared& s, uint32_t* dcut, uint32_t* icut) {
	const int tid = threadIdx.x;
	uint64_t prefix = 0;
	int shift = 24 + (bits + 7) / 8 * 8;
	for (uint32_t one = 0; shift > 0 && !one;) {
		shift -= 8;
		__syncthreads();
		for (int i = tid; i < 256; i += kSampleBlock) {
			s.m[i] = 0;
			s.c[i] = 0;
		}
		__syncthreads();
		for (int i = tid; i < n; i += kSampleBlock) {
			uint32_t d, index;
			if (!get(i, &d, &index)) continue;
			const uint64_t key = (uint64_t)(d - d0) << 24 | index;
			if ((key ^ prefix) >> (shift + 8)) continue;
			const int b = (int)(key >> shift & 255);
			atomicAdd(&s.m[b], (unsigned long long)measure(d));
			atomicAdd(&s.c[b], 1u);
		}
		__syncthreads();
		if (tid < 64) {
			uint64_t m[4], x = 0;
#pragma unroll
			for (int i = 0; i < 4; ++i) x += m[i] = s.m[4 * tid + i];
			const uint64_t own = x;
			for (int o = 1; o < 64; o *= 2) {
				const uint64_t y = __shfl_up(x, o, 64);
				x += tid >= o ? y : 0;
			}
			const uint64_t hit = __ballot(x >= goal);
			if (hit && tid == __builtin_ctzll(hit)) {
				uint64_t run = x - own;
				int i = 0;
				while (i < 3 && run + m[i] < goal) run += m[i++];
				s.digit = 4 * tid + i;
				s.below = run;
				s.one = s.c[4 * tid + i] == 1;
			}
			if (tid == 0) s.found = hit != 0;
		}
		__syncthreads();
		if (!s.found) return false;
		prefix |= (uint64_t)s.digit << shift;
		goal -= s.below;
		one = s.one;
	}
	for (int i = tid; i < n; i += kSampleBlock) {
		uint32_t d, index;
		if (!get(i, &d, &index)) continue;
		const uint64_t key = (uint64_t)(d - d0) << 24 | index;
		if (!((key ^ prefix) >> shift)) s.key = key;
	}
	__syncthreads();
	*dcut = (uint32_t)(s.key >> 24) + d0;
	*icut = (uint32_t)(s.key & 0xffffff);
	__syncthreads();
	return true;
}

template <typename G, typename M>
__device__ __forceinline__ uint64_t sum_of(int n, G&& get, M&& measure, BorderShared& s) {
	uint64_t x = 0;
	for (int i = threadIdx.x; i < n; i += kSampleBlock) {
		uint32_t d, index;
		if (get(i, &d, &index)) x += measure(d);
	}
	for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
	__syncthreads();
	if ((threadIdx.x & 63) == 0) s.sum[threadIdx.x >> 6] = x;
	__syncthreads();
	x = 0;
	for (int i = 0; i < kSampleBlock / 64; ++i) x += s.sum[i];
	return x;
}

// A block per row.  slices > 1: the gathered elements, or the row itself where they do not do; one slice: the row in LDS.
__global__ __launch_bounds__(kSampleBlock) void k_sample_pick(SampleArgs a, SampleWork w, int slices) {
	__shared__ uint32_t s_d[kSampleSlice];  // distances, then (of a list) the indexes
	__shared__ BorderShared sh;
	__shared__ int s_top, s_any;
	const int r = blockIdx.x, tid = threadIdx.x;
	const Sampling s = a.rules[r];
	const int32_t* row = a.logits + (int64_t)r * a.ld;
	if (!sampling_ok(s, a.vocab)) {
		if (tid == 0) {
			a.tokens[r] = -2;
			if (a.mass) a.mass[2 * r] = a.mass[2 * r + 1] = 0;
		}
		return;
	}
	const Weight wt = weight_of(s);
	const uint64_t least = share_of((uint64_t)(s.q_b * s.q_b + s.q_c), s.min_p);
	const bool by_p = s.top_p < 65536;
	auto weights = [&](uint32_t d) { return weight(wt, d); };
	auto kepts = [&](uint32_t d) {
		const uint64_t x = weight(wt, d);
		return x < least ? (uint64_t)0 : x;
	};
	auto ones = [&](uint32_t) { return (uint64_t)1; };
	uint32_t dcut = 0xffffffffu, icut = 0xffffffu;
	uint64_t all = 0;
	bool done = false;
	SamplePlan p{};
	if (slices > 1) p = w.plan[r];
	if (slices > 1 && p.state == 0 && p.count <= kSampleList) {
		const int n = (int)p.count, rb = p.top >> p.sh;
		uint32_t *d_of = s_d, *i_of = s_d + kSampleList;
		for (int i = tid; i < n; i += kSampleBlock) {
			const uint2 x = w.list[(size_t)r * kSampleList + i];
			d_of[i] = x.x;
			i_of[i] = x.y;
		}
		__syncthreads();
		auto within = [&](int which) {
			return [&, which](int i, uint32_t* d, uint32_t* index) {
				*d = d_of[i];
				*index = i_of[i];
				const uint32_t j = (uint32_t)rb - (uint32_t)((int32_t)((uint32_t)p.top - *d) >> p.sh);
				return j >= p.a[which] && j < p.b[which] && (*d < dcut || (*d == dcut && *index <= icut));
			};
		};
		// the smallest d of a bucket, and the bits of a range
		auto first = [&](int which) { return (uint32_t)i64max(0, (int64_t)p.top - (((int64_t)rb - p.a[which] + 1) * ((int64_t)1 << p.sh) - 1)); };
		auto bits = [&](int which) { return 32 - __builtin_clz(((p.b[which] - p.a[which]) << p.sh) | 1); };
		uint64_t total = p.w[0], kept = p.kept[0];
		bool ok = true;
		if (p.cut_k) {
			ok = find_border(n, within(0), ones, p.goal_k, first(0), bits(0), sh, &dcut, &icut);
			if (ok && by_p) total += sum_of(n, within(0), weights, sh);
			if (ok && !by_p) kept += sum_of(n, within(0), kepts, sh);
		}
		if (ok && by_p) {
			uint64_t need = share_of(total, s.top_p);
			need = need < 1 ? 1 : need;
			ok = need > p.w[1] && find_border(n, within(1), weights, need - p.w[1], first(1), bits(1), sh, &dcut, &icut);
			if (ok) kept = p.kept[1] + sum_of(n, within(1), kepts, sh);
		}
		if (ok) {
			const uint64_t goal = random_of(kept, s.random) + 1;
			all = kept;
			ok = goal > p.kept[2] && find_border(n, within(2), kepts, goal - p.kept[2], first(2), bits(2), sh, &dcut, &icut);
		}
		done = ok;
		__syncthreads();
	}
	if (!done) {
		// over the row itself
		const bool in_lds = slices == 1;
		if (tid == 0) {
			s_top = INT32_MIN;
			s_any = 0;
		}
		__syncthreads();
		auto legal = [&](int i) { return !s.mask || (global_ptr(s.mask)[i >> 3] >> (i & 7) & 1); };
		int top = INT32_MIN;
		bool any = false;
		for (int i = tid; i < a.vocab; i += kSampleBlock)
			if (legal(i)) {
				top = max(top, row[i]);
				any = true;
			}
		if (any) {
			atomicMax(&s_top, top);
			s_any = 1;
		}
		__syncthreads();
		if (!s_any) {
			if (tid == 0) {
				a.tokens[r] = -1;
				if (a.mass) a.mass[2 * r] = a.mass[2 * r + 1] = 0;
			}
			return;
		}
		top = s_top;
		// only what has a weight counts: the others come last in the order
		if (in_lds) {
			for (int i = tid; i < a.vocab; i += kSampleBlock) {
				const uint32_t d = (uint32_t)top - (uint32_t)row[i];
				s_d[i] = legal(i) && (int64_t)d < wt.lim ? d : 0xffffffffu;
			}
			__syncthreads();
		}
		dcut = 0xffffffffu;
		icut = 0xffffffu;
		auto get = [&](int i, uint32_t* d, uint32_t* index) {
			*d = in_lds ? s_d[i] : (legal(i) ? (uint32_t)top - (uint32_t)row[i] : 0xffffffffu);
			*index = i;
			return (int64_t)*d < wt.lim && (*d < dcut || (*d == dcut && *index <= icut));
		};
		const int bits = 64 - __builtin_clzll((uint64_t)wt.lim);
		if (s.top_k > 0 && (uint64_t)s.top_k < sum_of(a.vocab, get, ones, sh)) find_border(a.vocab, get, ones, s.top_k, 0, bits, sh, &dcut, &icut);
		if (by_p) {
			const uint64_t need = share_of(sum_of(a.vocab, get, weights, sh), s.top_p);
			find_border(a.vocab, get, weights, need < 1 ? 1 : need, 0, bits, sh, &dcut, &icut);
		}
		all = sum_of(a.vocab, get, kepts, sh);
		find_border(a.vocab, get, kepts, random_of(all, s.random) + 1, 0, bits, sh, &dcut, &icut);
	}
	if (tid == 0) {
		a.tokens[r] = (int32_t)icut;
		if (a.mass) {
			a.mass[2 * r] = (int64_t)weight(wt, dcut);
			a.mass[2 * r + 1] = (int64_t)all;
		}
	}
}

}  // namespace sslm

namespace sslm_launch {

static int sample_slices(int vocab) { return (vocab + kSampleSlice - 1) / kSampleSlice; }

static size_t sample_work(int rows, int vocab, char* base, SampleWork* w) {
	const size_t n = (size_t)rows * sample_slices(vocab);
	size_t at = 0;
	auto take = [&](size_t bytes) {
		char* p = base + at;
		at += up256(bytes);
		return p;
	};
	const bool one = sample_slices(vocab) == 1;
	w->plan = (SamplePlan*)take(rows * sizeof(SamplePlan));
	w->smax = (int64_t*)take(one ? 0 : n * 8);
	w->hist = (uint16_t*)take(one ? 0 : n * kBuckets * 2);
	w->list = (uint2*)take(one ? 0 : (size_t)rows * kSampleList * sizeof(uint2));
	return at;
}

size_t sample_workspace(int rows, int vocab) {
	SampleWork w;
	return sample_work(rows, vocab, nullptr, &w);
}

void sample_tokens(const SampleArgs& a, hipStream_t s) {
	SampleWork w;
	sample_work(a.rows, a.vocab, (char*)a.ws, &w);
	const int slices = sample_slices(a.vocab);
	if (slices > 1) {
		const bool vec = a.ld % 4 == 0 && (uintptr_t)a.logits % 16 == 0;
		const dim3 grid(slices, a.rows), bs(kSampleBlock);
		if (vec) hipLaunchKernelGGL(k_sample_hist<true>, grid, bs, 0, s, a, w);
		else hipLaunchKernelGGL(k_sample_hist<false>, grid, bs, 0, s, a, w);
		hipLaunchKernelGGL(k_sample_plan, dim3(a.rows), dim3(kPlanThreads), 0, s, a, w, slices);
		if (vec) hipLaunchKernelGGL(k_sample_gather<true>, grid, bs, 0, s, a, w);
		else hipLaunchKernelGGL(k_sample_gather<false>, grid, bs, 0, s, a, w);
	}
	hipLaunchKernelGGL(k_sample_pick, dim3(a.rows), dim3(kSampleBlock), 0, s, a, w, slices);
}

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
