// The next token by sampling (cache_ops.h): kernels, launches and the C entry.
#include <hip/hip_runtime.h>

#include <type_traits>

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
	uint32_t lim;  // below 2^30
};
__device__ __forceinline__ Weight weight_of(const Sampling& s) {
	Weight w;
	w.l = (double)s.q_ln2;
	w.ninv = 1.0 / w.l;
	w.half = 0.5 * w.ninv;
	w.b = (double)s.q_b;
	w.c = (double)s.q_c;
	w.lim = (uint32_t)(30 * s.q_ln2);
	return w;
}
__device__ __forceinline__ double weight_below(const Weight& w, uint32_t d) {  // d < lim; past it something
	const double x = (double)d, z = ceil(fma(x, -w.ninv, -w.half)), base = fma(-z, w.l, w.b - x);
	return floor(ldexp(fma(base, base, w.c), (int)z));
}
__device__ __forceinline__ double weight_d(const Weight& w, uint32_t d) { return d >= w.lim ? 0.0 : weight_below(w, d); }
__device__ __forceinline__ uint64_t weight(const Weight& w, uint32_t d) { return (uint64_t)weight_d(w, d); }

// Everything a row's sampling asks for is a border in one order, logit descending, then index ascending: the element whose
// running count (top-k), running weight (top-p) or running kept weight (the draw) reaches a goal.  Over the whole row that is a
// radix search, some passes over the vocabulary for each.  Four launches find the same borders with two passes:
//   k_sample_hist    a slice's largest logit, and how many of its logits lie in each bucket of 2^sh below it
//   k_sample_plan    a row's buckets together; from their counts and mean weights where each border must be, within a few buckets
//   k_sample_gather  the exact sums of the weights before those buckets, and the elements in them
//   k_sample_pick    the borders among these elements.  That each lies where it was expected is checked exactly, so an estimate
//                    that misses (or a list that overflows) costs the radix search over the row, not the result.
// Rows of one slice are searched in LDS by k_sample_pick alone.  At 151936 tokens 1 row takes 4.2 + 11.0 + 6.1 + 9.2 us, the chains of
// four launches, and 128 rows 16.3 + 18.4 + 29 + 13.5: the first pass reads 79 MB at 4.9 TB/s, the second is bound by its doubles, plan and
// pick are a block's chain of scans to a row.  The search over the row takes 870 .. 980 us for 1 row and
// some 1800 for 128: what a row costs whose borders' buckets hold more than kSampleList, a bell of 151936 logits of a spread below about 1.2
// natural units.
constexpr int kSampleBlock = 512;
constexpr int kSampleSlice = 8192, kSampleLoads = kSampleSlice / kSampleBlock / 4;
constexpr int kBuckets = 2048;
constexpr int kSampleList = 4096, kSliceList = 2048;  // elements gathered of a row, of a slice of it

// What the plan found: the borders' bucket ranges [a, b), 0 top-k, 1 top-p, 2 the draw (unused ones empty).
struct SamplePlan {
	int32_t top, sh;   // the row's largest logit
	int32_t state;     // 0: to be drawn from the ranges, 1: by the search over the row, 2: by that, as the ranges missed, -1: no legal token
	int32_t cut_k;     // whether top-k cuts, and how many of its first elements range 0 has
	uint32_t goal_k;
	uint32_t a[3], b[3];
	uint32_t count;    // elements gathered
	// sums of the weights before ranges 0 and 1, of the kept ones before range 1 (0 without top-p) and range 2; over the whole row
	// where there is no such border
	unsigned long long w[2], kept[2];
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
		// every load goes out before one is waited for: quads by the row's last whole one, then what stands past it
		if (VEC && n >= 4) {
#pragma unroll
			for (int u = 0; u < kSampleLoads; ++u) x[u] = *(const v4i*)(row + min(place(u), (n & ~3) - 4));
		}
		if (!VEC || n < 4 || (n & 3)) {
#pragma unroll
			for (int u = 0; u < kSampleLoads; ++u)
				if (!VEC || place(u) + 4 > n)
#pragma unroll
					for (int i = 0; i < 4; ++i) x[u][i] = row[min(place(u) + i, n - 1)];
		}
		uint32_t m[kSampleLoads];
#pragma unroll
		for (int u = 0; u < kSampleLoads; ++u) m[u] = 0xff;
		if (mask) {
#pragma unroll
			for (int u = 0; u < kSampleLoads; ++u) m[u] = global_ptr(mask)[min(v0 + place(u), a.vocab - 1) >> 3];
		}
		legal = 0;
#pragma unroll
		for (int u = 0; u < kSampleLoads; ++u) {
			const int left = n - place(u);
			legal |= (m[u] >> (place(u) & 4) & (left >= 4 ? 15u : (left > 0 ? (1u << left) - 1 : 0u))) << 4 * u;
		}
	}
	__device__ __forceinline__ int place(int u) const { return 4 * ((int)threadIdx.x + u * kSampleBlock); }
	__device__ __forceinline__ bool has(int u, int i) const { return legal >> (4 * u + i) & 1; }
	__device__ __forceinline__ int index(int u, int i) const { return v0 + place(u) + i; }
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

// What a bucket counts for in the plan, and its sums.
struct Mass {
	int32_t c;
	double e, k, v;  // weight, kept weight, variance of the weight
};
__device__ __forceinline__ Mass operator+(const Mass& a, const Mass& b) { return Mass{a.c + b.c, a.e + b.e, a.k + b.k, a.v + b.v}; }

constexpr int kPlanThreads = 512, kPlanBuckets = kBuckets / kPlanThreads;
struct __attribute__((packed)) plan_counts {
	uint64_t v;
};

// sums up to and with each thread's, in thread order, and the total
__device__ __forceinline__ Mass mass_scan(Mass x, Mass* s, Mass* total) {
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	for (int o = 1; o < 64; o *= 2) {
		const Mass y{__shfl_up(x.c, o, 64), __shfl_up(x.e, o, 64), __shfl_up(x.k, o, 64), __shfl_up(x.v, o, 64)};
		if (lane >= o) x = x + y;
	}
	if (lane == 63) s[wave] = x;
	__syncthreads();
	Mass before{0, 0.0, 0.0, 0.0}, all{0, 0.0, 0.0, 0.0};
#pragma unroll
	for (int i = 0; i < kPlanThreads / 64; ++i) {
		if (i < wave) before = before + s[i];
		all = all + s[i];
	}
	*total = all;
	return before + x;
}

// A block per row, a few neighbouring buckets a thread.  A bucket's weight is estimated by its count times the mean of its ends',
// which is off by what places spread evenly over the bucket deviate.  A border at the share f of a sum lies where the sum P up to
// it less f of all is nothing: with the errors of what is before and behind it apart, that has the variance (1 - f)^2 V_before +
// f^2 V_behind, and the border is looked for within six deviations.
__global__ __launch_bounds__(kPlanThreads) void k_sample_plan(SampleArgs a, SampleWork w, int slices) {
	__shared__ uint32_t s_off[SSLM_HIP_SAMPLE_MAX_VOCAB / kSampleSlice];
	__shared__ Mass s_scan[kPlanThreads / 64];
	__shared__ int s_a[3], s_b[3], s_n;
	__shared__ uint32_t s_goal;
	__shared__ double s_sum, s_kept, s_var;
	__shared__ unsigned long long s_doubt, s_kept_p, s_more;  // s_kept_p, s_more: bits of doubles that are not negative
	__shared__ int s_few;
	const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
	const int64_t* smax = w.smax + (size_t)r * slices;
	int64_t best = smax[min(lane, slices - 1)];
	const Sampling s = a.rules[r];
	if (!sampling_ok(s, a.vocab)) return;
	if (tid == 0) {
		s_n = 0;
		s_goal = 0;
		s_doubt = s_more = 0;
		s_kept_p = ~0ull;
	}
	if (tid < 3) s_a[tid] = s_b[tid] = kBuckets;
	// every wave finds the row's largest logit
	for (int i = lane + 64; i < slices; i += 64) best = i64max(best, smax[i]);
	const bool some = __any(best != kNoLogit);
	const int32_t top = (int32_t)(wave_max32(best == kNoLogit ? 0u : (uint32_t)(int32_t)best ^ 0x80000000u) ^ 0x80000000u);
	const int sh = bucket_shift(s), rb = top >> sh;
	for (int i = tid; i < slices; i += kPlanThreads) {
		const int64_t m = smax[i];
		s_off[i] = m == kNoLogit ? (uint32_t)kBuckets : min((uint32_t)rb - (uint32_t)((int32_t)m >> sh), (uint32_t)kBuckets);
	}
	__syncthreads();
	SamplePlan p{};
	p.state = -1;
	if (some) {
		p.state = 0;
		p.top = top;
		p.sh = sh;
		const uint32_t j0 = kPlanBuckets * tid;
		// The thread's four buckets of each slice, whose first one is the row's s_off, in eight bytes; 7 slices' counts stay below 2^16
		// each, so that they are added as they stand.  1 and 128 rows of 151936: 10.9 and 18.5 us, 12.9 and 20.5 by atomics in LDS.
		static_assert(kPlanBuckets == 4 && 7 * kSampleSlice < 1 << 16, "counts in 16 bits");
		constexpr int kGroups = 3;
		int c[kPlanBuckets] = {};
		for (int i0 = 0; i0 < slices; i0 += 7 * kGroups) {
			uint64_t x[7 * kGroups];
			int first[7 * kGroups];
#pragma unroll
			for (int q = 0; q < 7 * kGroups; ++q) {
				const int i = min(i0 + q, slices - 1);
				first[q] = i0 + q < slices ? (int)(j0 - s_off[i]) : -kBuckets;
				x[q] = ((const plan_counts*)(w.hist + ((size_t)r * slices + i) * kBuckets + max(first[q], 0)))->v;
			}
			__builtin_amdgcn_sched_barrier(0);  // all of them before the first is waited for
#pragma unroll
			for (int g = 0; g < kGroups; ++g) {
				uint64_t sum = 0;
#pragma unroll
				for (int q = 7 * g; q < 7 * g + 7; ++q) sum += first[q] >= 0 ? x[q] : (first[q] > -4 ? x[q] << 16 * -first[q] : 0);
#pragma unroll
				for (int k = 0; k < kPlanBuckets; ++k) c[k] += (int)(sum >> 16 * k & 0xffff);
			}
		}
		const Weight wt = weight_of(s);
		const double least = (double)share_of((uint64_t)(s.q_b * s.q_b + s.q_c), s.min_p);
		Mass one[kPlanBuckets], run[kPlanBuckets], all, mine{0, 0.0, 0.0, 0.0};
		double doubt = 0.0;  // what lies in the bucket that min-p cuts
#pragma unroll
		for (int i = 0; i < kPlanBuckets; ++i) {
			const int64_t low = ((int64_t)rb - (j0 + i)) * ((int64_t)1 << p.sh);  // its least logit
			const int64_t d1 = p.top - low, d0 = i64max(0, d1 - (((int64_t)1 << p.sh) - 1));
			const double w0 = weight_d(wt, (uint32_t)i64min(d0, 0xffffffffll)), w1 = weight_d(wt, (uint32_t)i64min(d1, 0xffffffffll));
			const double mid = 0.5 * (w0 + w1), n = (double)c[i];
			one[i] = Mass{c[i], n * mid, mid >= least ? n * mid : 0.0, n * (w0 - w1) * (w0 - w1) * (1.0 / 12)};
			doubt += w0 >= least && w1 < least ? n * w0 : 0.0;
			mine = mine + one[i];
		}
		// the i-exp rises a little where one of its segments ends, so that more than one bucket may be cut: a sum of integers below 2^62
		if (s.min_p > 0 && doubt > 0.0) atomicAdd(&s_doubt, (unsigned long long)doubt);
		Mass at = mass_scan(mine, s_scan, &all);
#pragma unroll
		for (int i = kPlanBuckets - 1; i >= 0; --i) {
			run[i] = at;
			at = Mass{at.c - one[i].c, at.e - one[i].e, at.k - one[i].k, at.v - one[i].v};
		}
		if (tid == 0) {
			s_sum = all.e;
			s_kept = all.k;
			s_var = all.v;
			s_few = all.c;
		}
		__syncthreads();
		// top-k: exactly its bucket; the estimates up to its border
		const bool cut_k = s.top_k > 0 && s.top_k < all.c, by_p = s.top_p < 65536;
		if (cut_k)
#pragma unroll
			for (int i = 0; i < kPlanBuckets; ++i)
				if (run[i].c >= s.top_k && run[i].c - one[i].c < s.top_k) {
					s_goal = s.top_k - (run[i].c - one[i].c);
					s_few = run[i].c;
					const double part = (double)s_goal / (double)one[i].c;
					s_a[0] = (int)j0 + i;
					s_b[0] = (int)j0 + i + 1;
					s_sum = run[i].e - (1.0 - part) * one[i].e;
					s_kept = run[i].k - (1.0 - part) * one[i].k;
					s_var = run[i].v + one[i].e * one[i].e * 0.01;  // which of the bucket's elements these are
				}
		__syncthreads();
		const int end = s_b[0];  // nothing is taken past it
		const bool few = s_few <= kSampleList / 2;  // of few elements all are gathered
		const double sum = s_sum, kept_k = s_kept, var = s_var;
		auto range = [&](int which, bool of_kept, double goal, double whole, double more) {
			const double f = whole > 0.0 ? fmin(1.0, goal / whole) : 0.0;
			int from = kBuckets, to = kBuckets;
#pragma unroll
			for (int i = kPlanBuckets - 1; i >= 0; --i) {
				const double v = fmin(run[i].v, var), off = 6.0 * sqrt((1.0 - f) * (1.0 - f) * v + f * f * (var - v)) + 1e-9 * whole + more;
				const double at = (of_kept ? run[i].k : run[i].e) - goal;
				from = at >= -off ? max(0, (int)j0 + i - 1) : from;
				to = at >= off ? (int)j0 + i + 2 : to;
			}
			// buckets ascend with the lanes: a wave's first one is its least
			const uint64_t fs = __ballot(from < kBuckets), ts = __ballot(to < kBuckets);
			if (fs && (tid & 63) == __builtin_ctzll(fs)) atomicMin(&s_a[which], from);
			if (ts && (tid & 63) == __builtin_ctzll(ts)) atomicMin(&s_b[which], to);
		};
		double kept = kept_k;
		if (by_p) {
			const double goal = sum * s.top_p * (1.0 / 65536);
			range(1, false, goal, sum, 0.0);
#pragma unroll
			for (int i = 0; i < kPlanBuckets; ++i)  // the kept weight up to there
				if (run[i].e >= goal && run[i].e - one[i].e < goal) {
					// apart from s_kept, which waves may still be reading; rounded sums can put the border into two neighbours: the lesser weight
					// and the larger element, whichever thread comes first
					const double k = run[i].k - (1.0 - (goal - (run[i].e - one[i].e)) / one[i].e) * one[i].k;
					atomicMin(&s_kept_p, k > 0.0 ? (unsigned long long)__double_as_longlong(k) : 0ull);
					atomicMax(&s_more, (unsigned long long)__double_as_longlong(1.2 * one[i].e / (double)one[i].c));  // the run ends with a whole element
				}
			__syncthreads();
			if (s_kept_p != ~0ull) kept = fmin(kept_k, __longlong_as_double((long long)s_kept_p));
		}
		range(2, true, kept * s.random * 0x1p-32, kept_k, (double)s_doubt + __longlong_as_double((long long)s_more));
		__syncthreads();
		p.cut_k = cut_k;
		p.goal_k = s_goal;
#pragma unroll
		for (int i = 0; i < 3; ++i) {
			p.a[i] = min(s_a[i], end - 1);
			p.b[i] = max(min(s_b[i], end), (int)p.a[i]);
			if (few) {
				p.a[i] = i ? 0 : p.a[i];
				p.b[i] = end;
			}
		}
		if (!cut_k) p.a[0] = p.b[0] = kBuckets;
		if (!by_p) p.a[1] = p.b[1] = kBuckets;
		// how much would be gathered
		int n = 0;
#pragma unroll
		for (int i = 0; i < kPlanBuckets; ++i) {
			const uint32_t j = j0 + i;
			n += (j >= p.a[0] && j < p.b[0]) || (j >= p.a[1] && j < p.b[1]) || (j >= p.a[2] && j < p.b[2]) ? c[i] : 0;
		}
		n = wave_sum32(n);
		if ((tid & 63) == 0 && n) atomicAdd(&s_n, n);
		__syncthreads();
		if (s_n > kSampleList) p.state = 1;
	}
	if (tid == 0) w.plan[r] = p;
}

// x, or less than 2^-1000, which no sum of integers notices: one select instead of two
__device__ __forceinline__ double only(bool take, double x) { return __hiloint2double(take ? __double2hiint(x) : 0, __double2loint(x)); }

template <bool VEC>
__global__ __launch_bounds__(kSampleBlock) void k_sample_gather(SampleArgs a, SampleWork w) {
	__shared__ unsigned long long s_sum[5];
	__shared__ uint2 s_list[kSliceList];
	__shared__ uint32_t s_n, s_at;
	const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
	const Sampling s = a.rules[r];
	SampleSlice<VEC> sl;
	sl.load(a, s.mask);
	if (!sampling_ok(s, a.vocab)) return;
	const SamplePlan& p = w.plan[r];
	if (p.state != 0) return;
	const int32_t top = p.top, sh = p.sh, rb = top >> sh;
	// the sums that the borders need: weights before ranges 0, 1 and 2, kept ones (where min-p makes them others) before 0 or 1, and 2
	const bool by_p = s.top_p < 65536, min_p = s.min_p > 0;
	if (tid < 5) s_sum[tid] = 0;
	if (tid == 0) s_n = 0;
	__syncthreads();
	const Weight wt = weight_of(s);
	const double least = (double)share_of((uint64_t)(s.q_b * s.q_b + s.q_c), s.min_p);
	double acc0 = 0.0, acc1 = 0.0, acc2 = 0.0, acc3 = 0.0, acc4 = 0.0;  // 16 values of 2^47
	// What bounds the kernel is its instructions, so the places j < x of the buckets are the d below this, one comparison of an element for
	// each, and what is not legal is moved past them all: 128 rows of 151936 in 29 us, 33 with the buckets' numbers, every sum and
	// the legal bits looked at for each element.
	auto below = [&](uint32_t x) { return (uint32_t)i64max(0, (int64_t)top + 1 - ((int64_t)rb - x + 1) * ((int64_t)1 << sh)); };
	const uint32_t r0 = below(p.a[0]), n0 = below(p.b[0]) - r0, r1 = below(p.a[1]), n1 = below(p.b[1]) - r1, r2 = below(p.a[2]), n2 = below(p.b[2]) - r2;
	const uint32_t a0 = min(r0, wt.lim), a1 = min(r1, wt.lim), a2 = min(r2, wt.lim), first = by_p ? a1 : a0, most = max(a0, max(by_p ? a1 : 0, a2));
	if (__any(sl.legal != (1u << 4 * kSampleLoads) - 1)) {
		// what is not legal goes furthest below the largest, past every range
#pragma unroll
		for (int u = 0; u < kSampleLoads; ++u)
#pragma unroll
			for (int i = 0; i < 4; ++i) sl.x[u][i] = sl.has(u, i) ? sl.x[u][i] : (int32_t)((uint32_t)top + 1);
	}
	uint64_t who[4 * kSampleLoads];  // which lanes' elements lie in a range
	auto run = [&](auto with_top_p, auto with_min_p) {
		constexpr bool TP = decltype(with_top_p)::value, MP = decltype(with_min_p)::value;
#pragma unroll
		for (int u = 0; u < kSampleLoads; ++u)
#pragma unroll
			for (int i = 0; i < 4; ++i) {
				const uint32_t d = (uint32_t)top - (uint32_t)sl.x[u][i];
				if (__any(d < most)) {
					const double x = weight_below(wt, d);
					acc0 += only(d < a0, x);
					if constexpr (TP) acc1 += only(d < a1, x);
					if constexpr (!MP) acc2 += only(d < a2, x);
					else {
						const bool kept = x >= least;
						acc3 += only((d < first) & kept, x);
						acc4 += only((d < a2) & kept, x);
					}
				}
				who[4 * u + i] = __ballot(d - r0 < n0) | __ballot(d - r2 < n2);
				if constexpr (TP) who[4 * u + i] |= __ballot(d - r1 < n1);
			}
	};
	if (by_p && min_p) run(std::true_type{}, std::true_type{});
	else if (by_p) run(std::true_type{}, std::false_type{});
	else if (min_p) run(std::false_type{}, std::true_type{});
	else run(std::false_type{}, std::false_type{});
	uint32_t mine = 0;
#pragma unroll
	for (int k = 0; k < 4 * kSampleLoads; ++k) mine += (uint32_t)__popcll(who[k]);
	if (mine) {
		uint32_t at = 0;
		if (lane == 0) at = atomicAdd(&s_n, mine);  // the wave's places in the list
		at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
		for (int k = 0; k < 4 * kSampleLoads; ++k)
			if (who[k]) {
				const uint32_t to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(who[k] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who[k], 0));
				if ((who[k] >> lane & 1) && to < kSliceList) s_list[to] = uint2{(uint32_t)top - (uint32_t)sl.x[k / 4][k % 4], (uint32_t)sl.index(k / 4, k % 4)};
				at += (uint32_t)__popcll(who[k]);
			}
	}
	const double acc[5] = {acc0, acc1, acc2, acc3, acc4};
#pragma unroll
	for (int k = 0; k < 5; ++k) {
		if (!__any(acc[k] != 0.0)) continue;
		int64_t x = (int64_t)acc[k];
		x = row16_sum(x);
		x += __shfl_xor(x, 16, 64);
		x += __shfl_xor(x, 32, 64);
		if (lane == 0) atomicAdd(&s_sum[k], (unsigned long long)x);
	}
	__syncthreads();
	const uint32_t n = s_n;
	if (tid == 0) {
		SamplePlan& o = w.plan[r];
		// a slice with more than its share: past the row's list, whose search then runs over the row
		if (n) s_at = atomicAdd(&o.count, n <= kSliceList ? n : kSampleList + 1);
		auto add = [](unsigned long long* to, unsigned long long x) {
			if (x) atomicAdd(to, x);
		};
		add(&o.w[0], s_sum[0]);
		add(&o.w[1], s_sum[1]);
		add(&o.kept[0], min_p ? s_sum[3] : (by_p ? s_sum[1] : s_sum[0]));
		add(&o.kept[1], min_p ? s_sum[4] : s_sum[2]);
	}
	__syncthreads();
	if (n > kSliceList) return;
	for (uint32_t i = tid; i < n; i += kSampleBlock)
		if (s_at + i < kSampleList) w.list[(size_t)r * kSampleList + s_at + i] = s_list[i];
}

struct BorderShared {
	unsigned long long m[256], below, key;
	uint32_t c[256], digit, one, found;
	unsigned long long sum[kSampleBlock / 64];
};

// f(d, index) for the elements i < n that fetch(i) gives (no element: kNone), eight of a thread's on their way at a time
constexpr uint32_t kNone = 0xffffffffu;
template <typename F, typename X, typename I>
__device__ __forceinline__ void each_element(int n, F&& fetch, I&& index, X&& f) {
	for (int i0 = threadIdx.x; i0 < n; i0 += 8 * kSampleBlock) {
		uint32_t d[8];
#pragma unroll
		for (int u = 0; u < 8; ++u) d[u] = i0 + u * kSampleBlock < n ? fetch(i0 + u * kSampleBlock) : kNone;
#pragma unroll
		for (int u = 0; u < 8; ++u)
			if (d[u] != kNone) f(d[u], index(i0 + u * kSampleBlock));
	}
}

// The element whose running measure reaches `goal` among those that admit(d, index) lets in, by radix over the key
// (d - d0, index), d - d0 below 2^bits: eight bits a pass until one element is left.  False when there is none.
template <typename F, typename I, typename A, typename M>
__device__ __forceinline__ bool find_border(int n, F&& fetch, I&& index, A&& admit, M&& measure, uint64_t goal, uint32_t d0, int bits, BorderShared& s, uint32_t* dcut,
                                            uint32_t* icut) {
	const int tid = threadIdx.x;
	uint64_t prefix = 0;
	int shift = 24 + bits;
	for (uint32_t one = 0; shift > 0 && !one;) {
		const int above = shift;
		shift = max(0, shift - 8);
		__syncthreads();
		for (int i = tid; i < 256; i += kSampleBlock) {
			s.m[i] = 0;
			s.c[i] = 0;
		}
		__syncthreads();
		each_element(n, fetch, index, [&](uint32_t d, uint32_t i) {
			const uint64_t key = (uint64_t)(d - d0) << 24 | i;
			if (((key ^ prefix) >> above) || !admit(d, i)) return;
			const int b = (int)(key >> shift) & ((1 << (above - shift)) - 1);
			atomicAdd(&s.m[b], (unsigned long long)measure(d));
			atomicAdd(&s.c[b], 1u);
		});
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
	each_element(n, fetch, index, [&](uint32_t d, uint32_t i) {
		const uint64_t key = (uint64_t)(d - d0) << 24 | i;
		if (!((key ^ prefix) >> shift) && admit(d, i)) s.key = key;
	});
	__syncthreads();
	*dcut = (uint32_t)(s.key >> 24) + d0;
	*icut = (uint32_t)(s.key & 0xffffff);
	__syncthreads();
	return true;
}

template <typename F, typename I, typename A, typename M>
__device__ __forceinline__ uint64_t sum_of(int n, F&& fetch, I&& index, A&& admit, M&& measure, BorderShared& s) {
	uint64_t x = 0;
	each_element(n, fetch, index, [&](uint32_t d, uint32_t i) { x += admit(d, i) ? measure(d) : 0; });
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
		auto fetch = [&](int i) { return d_of[i]; };
		auto index = [&](int i) { return i_of[i]; };
		auto within = [&](int which) {
			const uint32_t from = p.a[which], many = p.b[which] - p.a[which];
			return [&, from, many](uint32_t d, uint32_t i) {
				const uint32_t j = (uint32_t)rb - (uint32_t)((int32_t)((uint32_t)p.top - d) >> p.sh);
				return j - from < many && (d < dcut || (d == dcut && i <= icut));
			};
		};
		// the smallest d of a bucket, and the bits of a range
		auto first = [&](int which) { return (uint32_t)i64max(0, (int64_t)p.top - (((int64_t)rb - p.a[which] + 1) * ((int64_t)1 << p.sh) - 1)); };
		auto bits = [&](int which) { return 32 - __builtin_clz(((p.b[which] - p.a[which]) << p.sh) | 1); };
		uint64_t total = p.w[0], kept = p.kept[0];
		bool ok = true;
		if (p.cut_k) {
			ok = find_border(n, fetch, index, within(0), ones, p.goal_k, first(0), bits(0), sh, &dcut, &icut);
			if (ok && by_p) total += sum_of(n, fetch, index, within(0), weights, sh);
			if (ok && !by_p) kept += sum_of(n, fetch, index, within(0), kepts, sh);
		}
		if (ok && by_p) {
			uint64_t need = share_of(total, s.top_p);
			need = need < 1 ? 1 : need;
			ok = need > p.w[1] && find_border(n, fetch, index, within(1), weights, need - p.w[1], first(1), bits(1), sh, &dcut, &icut);
			if (ok) kept += sum_of(n, fetch, index, within(1), kepts, sh);
		}
		if (ok) {
			const uint64_t goal = random_of(kept, s.random) + 1;
			all = kept;
			ok = goal > p.kept[1] && find_border(n, fetch, index, within(2), kepts, goal - p.kept[1], first(2), bits(2), sh, &dcut, &icut);
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
			if (slices > 1 && p.state == 0) w.plan[r].state = 2;  // so that tests see which rows missed
		}
		__syncthreads();
		auto legal = [&](int i) { return !s.mask || (global_ptr(s.mask)[i >> 3] >> (i & 7) & 1); };
		int top = INT32_MIN;
		bool any = false;
		for (int i0 = tid; i0 < a.vocab; i0 += 8 * kSampleBlock) {
			int32_t x[8];
			bool ok[8];
#pragma unroll
			for (int u = 0; u < 8; ++u) {
				const int i = min(i0 + u * kSampleBlock, a.vocab - 1);
				x[u] = row[i];
				ok[u] = legal(i);
			}
#pragma unroll
			for (int u = 0; u < 8; ++u) {  // a clamped one repeats the last
				top = ok[u] ? max(top, x[u]) : top;
				any |= ok[u];
			}
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
				s_d[i] = legal(i) && d < wt.lim ? d : kNone;
			}
			__syncthreads();
		}
		dcut = 0xffffffffu;
		icut = 0xffffffu;
		auto fetch = [&](int i) {
			if (in_lds) return s_d[i];
			const uint32_t d = (uint32_t)top - (uint32_t)row[i];
			return legal(i) && d < wt.lim ? d : kNone;
		};
		auto index = [&](int i) { return (uint32_t)i; };
		auto admit = [&](uint32_t d, uint32_t i) { return d < dcut || (d == dcut && i <= icut); };
		const int bits = 64 - __builtin_clzll((uint64_t)wt.lim);
		if (s.top_k > 0 && (uint64_t)s.top_k < sum_of(a.vocab, fetch, index, admit, ones, sh)) find_border(a.vocab, fetch, index, admit, ones, s.top_k, 0, bits, sh, &dcut, &icut);
		if (by_p) {
			const uint64_t need = share_of(sum_of(a.vocab, fetch, index, admit, weights, sh), s.top_p);
			find_border(a.vocab, fetch, index, admit, weights, need < 1 ? 1 : need, 0, bits, sh, &dcut, &icut);
		}
		all = sum_of(a.vocab, fetch, index, admit, kepts, sh);
		find_border(a.vocab, fetch, index, admit, kepts, random_of(all, s.random) + 1, 0, bits, sh, &dcut, &icut);
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
