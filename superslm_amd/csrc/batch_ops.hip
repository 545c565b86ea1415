// Operators of a decode step whose rows differ (batch_ops.h): kernels, launches and C entries.
#include <hip/hip_runtime.h>
#include <stdio.h>

#include "../../include/sslm_hip.h"
#include "batch_ops.h"
#include "device_util.h"

namespace sslm {

using sslm_launch::LogitRule;
using sslm_launch::LoraRef;

template <int BS>
__device__ __forceinline__ int64_t block_sum_i64(int64_t v, int64_t* slots) {
	for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
	if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
	__syncthreads();
	int64_t r = 0;
#pragma unroll
	for (int i = 0; i < BS / 64; ++i) r += slots[i];
	return r;
}

template <int BS>
__device__ __forceinline__ uint32_t block_max_u32(uint32_t v, uint32_t* slots) {
	v = wave_max32(v);
	if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = v;
	__syncthreads();
	uint32_t r = slots[0];
#pragma unroll
	for (int i = 1; i < BS / 64; ++i) r = max(r, slots[i]);
	return __builtin_amdgcn_readfirstlane(r);
}

// ------------------------------------------------------------------------------------------
// attention of rows that share prompts
// ------------------------------------------------------------------------------------------

// Where a row's positions lie: [0, start) in its prefix's block, [start, width) in its own.
struct RowSpan {
	int64_t width, start;
	const int8_t *own, *pre;
	int32_t st;
};

__device__ __forceinline__ RowSpan row_span(const sslm_launch::SharedAttnArgs& a, int r) {
	RowSpan s{a.row_width[r], 0, a.pool, a.pool, kOk};
	int p = -1;
	for (int i = 0; i < a.prefixes; ++i)
		if (a.prefix_rows[i] <= r && r < a.prefix_rows[i + 1]) p = i;
	const int blk = a.row_block[r];
	if (blk < 0 || blk >= a.blocks || s.width < 0 || s.width > a.cap) s.st = kPositionOverCap;
	else s.own += (int64_t)blk * a.block_bytes;
	if (p >= 0) {
		const int pb = a.prefix_block[p];
		const int64_t len = a.prefix_len[p];
		if (pb < 0 || pb >= a.blocks || len < 0 || len > a.cap || len > a.max_prefix) s.st = kPositionOverCap;
		else {
			s.pre += (int64_t)pb * a.block_bytes;
			s.start = len < s.width ? len : s.width;
		}
	}
	if (s.st == kOk && s.width - s.start > a.max_own) s.st = kPositionOverCap;
	if (s.st == kOk && s.width == 0) s.st = kSoftmaxRowWidthOutOfDomain;
	return s;
}

struct RowConst {
	int64_t q_ln2, q_b, q_c, ceil;
	int32_t st;
};

// The softmax constants of (row, KV head) (forward_sites.cpp:1805-1830).
__device__ __forceinline__ RowConst row_const(const sslm_launch::SharedAttnArgs& a, int r, int kvh, int64_t width) {
	RowConst c{0, 0, 0, 0, kOk};
	const Scale qs = a.q_scale[r];
	const int64_t km = a.khead_m[kvh], ke = a.khead_e[kvh];
	if (!fits_i32(qs.m) || !fits_i32(km)) {
		c.st = kCarriedScaleMantissaOutOfDomain;
		return c;
	}
	const Scale sm = combine_scale(qs, Scale{km, ke});
	if (!fits_i32(sm.m)) c.st = kCarriedScaleMantissaOutOfDomain;
	else if (iexp_scale_constants(sm.m, sm.e, a.ln2_q, a.b_q, a.ca_q, &c.q_ln2, &c.q_b, &c.q_c) != 0)
		c.st = kIExpScaleDerivationOutOfDomain;
	else c.st = check_softmax_width(c.q_b, c.q_c, width);
	if (c.st == kOk) c.ceil = softmax_ceiling(c.q_b, c.q_c);
	return c;
}

// One block per (row, query head): scores, i-exp values and Q15 probabilities recomputed from K in
// three passes over the positions, as the reference's definition has them
// (forward_sites.cpp:1791-1905).
template <int D>
__global__ __launch_bounds__(256) void k_shared_attn_row(sslm_launch::SharedAttnArgs a, int32_t* f, int32_t* hst) {
	constexpr int BS = 256;
	__shared__ __attribute__((aligned(16))) int8_t s_q[D];
	__shared__ int32_t s_p[BS], s_acc[D];
	__shared__ uint32_t s_mx[BS / 64], s_bad[BS / 64];
	__shared__ int64_t s_sum[BS / 64];
	const int h = blockIdx.x, r = blockIdx.y, i = threadIdx.x, kvh = h / (a.NH / a.NKV);
	const RowSpan sp = row_span(a, r);
	if (sp.st != kOk) {
		if (i == 0) hst[(size_t)r * a.NH + h] = sp.st;
		return;
	}
	for (int d = i; d < D; d += BS) {
		s_q[d] = a.q[((size_t)r * a.NH + h) * D + d];
		s_acc[d] = 0;
	}
	__syncthreads();
	const int64_t head = (int64_t)kvh * a.cap * D;
	auto score = [&](int64_t p) {
		const int8_t* k = (p < sp.start ? sp.pre : sp.own) + a.k_off + head + p * D;
		int32_t s = 0;
		for (int c = 0; c < D; c += 16) {
			const v4i x = load16(k + c), q = *(const v4i*)(s_q + c);
#pragma unroll
			for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_sdot4(x[j], q[j], s, false);
		}
		return s;
	};
	uint32_t mx = 0;
	for (int64_t p = i; p < sp.width; p += BS) mx = max(mx, (uint32_t)score(p) ^ 0x80000000u);
	const int32_t top = (int32_t)(block_max_u32<BS>(mx, s_mx) ^ 0x80000000u);
	const RowConst c = row_const(a, r, kvh, sp.width);
	if (c.st != kOk) {
		if (i == 0) hst[(size_t)r * a.NH + h] = c.st;
		return;
	}
	const double inv_ln2 = 1.0 / (double)c.q_ln2;
	int64_t sum = 0;
	uint32_t bad = 0;
	for (int64_t p = i; p < sp.width; p += BS) {
		const int64_t e = iexp_fast((int64_t)score(p) - top, c.q_ln2, inv_ln2, c.q_b, c.q_c, c.ceil);
		if (e < 0) bad = 1;
		else sum += e;
	}
	sum = block_sum_i64<BS>(sum, s_sum);
	if (block_max_u32<BS>(bad, s_bad)) {
		if (i == 0) hst[(size_t)r * a.NH + h] = kSoftmaxKernelRefusedAfterGateAccepted;
		return;
	}
	const int64_t den = sum > 1 ? sum : 1;
	const double inv = 1.0 / (double)den;
	int32_t acc = 0;
	const int d = i % D, part = i / D;
	for (int64_t b = 0; b < sp.width; b += BS) {
		const int64_t p = b + i;
		int64_t e = 0;
		if (p < sp.width) e = iexp_fast((int64_t)score(p) - top, c.q_ln2, inv_ln2, c.q_b, c.q_c, c.ceil);
		s_p[i] = e > 0 ? (int32_t)div_rcp(e << 15, den, inv, 32768) : 0;
		__syncthreads();
		const int n = (int)(sp.width - b < BS ? sp.width - b : BS);
		for (int j = part; j < n; j += BS / D) {
			const int64_t pj = b + j;
			acc += s_p[j] * (int32_t)((pj < sp.start ? sp.pre : sp.own) + a.v_off + head + pj * D)[d];
		}
		__syncthreads();
	}
	atomicAdd(&s_acc[d], acc);
	__syncthreads();
	const int32_t* cf = a.ctx_fold + 3 * h;
	if (i < D) f[((size_t)r * a.NH + h) * D + i] = sat_i32(apply_fold(s_acc[i], cf[0], cf[1], cf[2]));
	if (i == 0) hst[(size_t)r * a.NH + h] = kOk;
}

// The context funnel of one row (checked_chain_funnel.cpp:257-364), after the first refusing head.
template <int BS, int EPT>
__global__ __launch_bounds__(BS) void k_ctx_funnel(sslm_launch::SharedAttnArgs a, const int32_t* f, const int32_t* hst) {
	__shared__ uint32_t s_m[BS / 64];
	__shared__ int32_t s_st;
	const int r = blockIdx.x, N = a.NH * a.D;
	if (threadIdx.x == 0) {
		int32_t st = kOk;
		for (int h = a.NH - 1; h >= 0; --h) st = hst[(size_t)r * a.NH + h] != kOk ? hst[(size_t)r * a.NH + h] : st;
		s_st = st;
	}
	__syncthreads();
	if (s_st != kOk) {
		if (threadIdx.x == 0) a.status[r] = s_st;
		return;
	}
	int32_t v[EPT];
	uint32_t mx = 0;
#pragma unroll
	for (int k = 0; k < EPT; ++k) {
		const int j = (int)threadIdx.x + k * BS;
		v[k] = j < N ? f[(size_t)r * N + j] : 0;
		mx = max(mx, sat_abs_u32(v[k]));
	}
	mx = block_max_u32<BS>(mx, s_m);
	FunnelPlan plan;
	const int32_t st = funnel_plan(mx, nullptr, 0, a.site, &plan);
	if (threadIdx.x == 0) {
		a.status[r] = st;
		if (st == kOk) a.scales[r] = plan.out;
	}
	if (st != kOk) return;
#pragma unroll
	for (int k = 0; k < EPT; ++k) {
		const int j = (int)threadIdx.x + k * BS;
		if (j < N) a.codes[(size_t)r * N + j] = requant_code_f(v[k], plan.f);
	}
}

// ------------------------------------------------------------------------------------------
// a projection with an adapter of its own per row
// ------------------------------------------------------------------------------------------
constexpr int32_t kBadAdapter = -1;  // the row's status where its adapter is not one of the table's

// the row's adapter, or null; false: an index or rank outside the table's domain
__device__ __forceinline__ bool row_adapter(const sslm_launch::LoraGemmArgs& g, int t, const LoraRef** out) {
	const int i = g.row_adapter[t];
	*out = nullptr;
	if (i < 0) return true;
	if (i >= g.count || g.adapters[i].rank < 1 || g.adapters[i].rank > kMaxRank) return false;
	*out = g.adapters + i;
	return true;
}

// u = clamp(amp_fold(A x)) of a row (forward_sites.cpp:1066-1086), one wave per rank.
__global__ __launch_bounds__(256) void k_rows_u(sslm_launch::LoraGemmArgs g, int8_t* u) {
	const int t = blockIdx.x, rk = blockIdx.y * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
	const LoraRef* ad;
	if (!row_adapter(g, t, &ad) || !ad || rk >= ad->rank) return;
	const int8_t *x = g.a + (size_t)t * g.k, *w = ad->a + (size_t)rk * g.k;
	int32_t acc = 0;  // |A.x| <= 127^2 k < 2^31
	for (int c = lane * 16; c < g.k; c += 1024) {
		const v4i p = load16(x + c), q = load16(w + c);
#pragma unroll
		for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_sdot4(p[j], q[j], acc, false);
	}
	acc = wave_sum32(acc);
	if (lane == 0) {
		const int32_t* fd = ad->ufold + 3 * rk;
		u[(size_t)t * kMaxRank + rk] = (int8_t)clamp_code(apply_amp_fold((int64_t)acc, fd[0], fd[1], fd[2]));
	}
}

// Fold, adapter delta and funnel of a row of accumulators.
template <int BS, int EPT>
__global__ __launch_bounds__(BS) void k_lora_funnel(sslm_launch::LoraGemmArgs g, const int32_t* acc, const int8_t* u) {
	__shared__ uint32_t s_m[BS / 64];
	const int t = blockIdx.x;
	const LoraRef* ad;
	if (!row_adapter(g, t, &ad)) {
		if (threadIdx.x == 0) g.status[t] = kBadAdapter;
		return;
	}
	const int rank = ad ? ad->rank : 0;
	const int8_t* ur = u + (size_t)t * kMaxRank;
	int32_t v[EPT];
	uint32_t mx = 0;
#pragma unroll
	for (int k = 0; k < EPT; ++k) {
		const int j = (int)threadIdx.x + k * BS;
		v[k] = 0;
		if (j < g.n) {
			const int32_t* fd = g.fold + 3 * j;
			int64_t x = apply_fold((int64_t)acc[(size_t)t * g.n + j], fd[0], fd[1], fd[2]);
			if (ad) {
				const int8_t* b = ad->b + (size_t)j * rank;
				int32_t d = 0;  // |B.u| <= 127^2 64 < 2^31
				for (int i = 0; i < rank; ++i) d += (int32_t)b[i] * (int32_t)ur[i];
				const int32_t* df = ad->dfold + 3 * j;
				x += apply_amp_fold((int64_t)d, df[0], df[1], df[2]);
			}
			mx = max(mx, sat_abs_u32(x));
			v[k] = sat_i32(x);
		}
	}
	mx = block_max_u32<BS>(mx, s_m);
	FunnelPlan plan;
	const Scale in = g.in_scale[t];
	const int32_t st = funnel_plan(mx, &in, 1, g.site, &plan);
	if (threadIdx.x == 0) {
		g.status[t] = st;
		if (st == kOk) g.scales[t] = plan.out;
	}
	if (st != kOk) return;
#pragma unroll
	for (int k = 0; k < EPT; ++k) {
		const int j = (int)threadIdx.x + k * BS;
		if (j < g.n) g.codes[(size_t)t * g.n + j] = requant_code_f(v[k], plan.f);
	}
}

// ------------------------------------------------------------------------------------------
// the next token under each row's rules
// ------------------------------------------------------------------------------------------
constexpr int kPickSlice = 4096;  // tokens per block: counts and biases of a slice take 48 KB of LDS
constexpr int kPickBlock = 256;

__device__ __forceinline__ bool rule_ok(const LogitRule& r) {
	return r.history_len >= 0 && r.bias_count >= 0 && r.repetition_q16 >= 1 && (r.history_len == 0 || r.history) &&
	       (r.bias_count == 0 || (r.bias_ids && r.bias_values));
}

// One block per (slice of the vocabulary, row): the slice's token counts and bias sums in LDS, then
// one pass over its logits.  Keys order by logit, then by the lower index; 0 marks no legal token.
__global__ __launch_bounds__(kPickBlock) void k_pick_slice(sslm_launch::PickArgs a, unsigned long long* keys) {
	__shared__ int32_t s_cnt[kPickSlice];
	__shared__ unsigned long long s_bias[kPickSlice];
	__shared__ uint64_t s_key[kPickBlock / 64];
	const int r = blockIdx.y, v0 = blockIdx.x * kPickSlice, n = min(kPickSlice, a.vocab - v0);
	const LogitRule ru = a.rules[r];
	if (!rule_ok(ru)) return;
	const bool any = ru.history_len > 0 || ru.bias_count > 0;
	if (any) {
		for (int j = threadIdx.x; j < kPickSlice; j += kPickBlock) {
			s_cnt[j] = 0;
			s_bias[j] = 0;
		}
		__syncthreads();
		for (int i = threadIdx.x; i < ru.history_len; i += kPickBlock) {
			const int64_t j = (int64_t)ru.history[i] - v0;
			if (j >= 0 && j < n) atomicAdd(&s_cnt[j], 1);
		}
		for (int i = threadIdx.x; i < ru.bias_count; i += kPickBlock) {
			const int64_t j = (int64_t)ru.bias_ids[i] - v0;
			if (j >= 0 && j < n) atomicAdd(&s_bias[j], (unsigned long long)(int64_t)ru.bias_values[i]);
		}
		__syncthreads();
	}
	const int32_t* row = a.logits + (int64_t)r * a.ld + v0;
	uint64_t key = 0;
	for (int j = threadIdx.x; j < n; j += kPickBlock) {
		int64_t x = row[j];
		if (any) {
			const int32_t c = s_cnt[j];
			if (c > 0) {
				// (x << 16) / rho: below 2^47, so the double quotient's truncation is the integer one
				x = x > 0 ? (int64_t)((double)(x << 16) / (double)ru.repetition_q16) : (x * ru.repetition_q16) >> 16;
				x -= (int64_t)ru.presence + (int64_t)ru.frequency * c;
			}
			x += (int64_t)s_bias[j];
		}
		int32_t y = sat_i32(x);
		const int id = v0 + j;
		const bool legal = !ru.mask || ((ru.mask[id >> 3] >> (id & 7)) & 1u);
		y = legal ? y : kI32Min;
		if (a.adjusted) a.adjusted[(int64_t)r * a.adjusted_ld + id] = y;
		const uint64_t k = legal ? ((uint64_t)((uint32_t)y ^ 0x80000000u) << 32) | (0xffffffffu - (uint32_t)id) : 0;
		key = k > key ? k : key;
	}
	for (int o = 32; o > 0; o >>= 1) {
		const uint64_t w = __shfl_xor(key, o, 64);
		key = w > key ? w : key;
	}
	if ((threadIdx.x & 63) == 0) s_key[threadIdx.x >> 6] = key;
	__syncthreads();
	if (threadIdx.x == 0) {
		for (int w = 1; w < kPickBlock / 64; ++w) key = s_key[w] > key ? s_key[w] : key;
		keys[(size_t)r * gridDim.x + blockIdx.x] = key;
	}
}

__global__ __launch_bounds__(64) void k_pick_final(sslm_launch::PickArgs a, const unsigned long long* keys, int slices) {
	const int r = blockIdx.x;
	const LogitRule ru = a.rules[r];
	if (!rule_ok(ru)) {
		if (threadIdx.x == 0) a.tokens[r] = -2;
		return;
	}
	uint64_t key = 0;
	for (int i = threadIdx.x; i < slices; i += 64) key = max(key, (uint64_t)keys[(size_t)r * slices + i]);
	for (int o = 32; o > 0; o >>= 1) {
		const uint64_t w = __shfl_xor(key, o, 64);
		key = w > key ? w : key;
	}
	if (threadIdx.x == 0) a.tokens[r] = key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1;
}

}  // namespace sslm

// ------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------
namespace sslm_launch {

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

bool shared_attn_ok(int rows, int NH, int NKV, int D) {
	return rows >= 1 && NKV >= 1 && NH >= NKV && NH % NKV == 0 && (D == 32 || D == 64 || D == 128 || D == 256) &&
	       (int64_t)NH * D <= kFunnelMaxN;
}

size_t shared_attn_workspace(int rows, int NH, int NKV, int D, int prefixes, int64_t max_prefix, int64_t max_own) {
	return up256((size_t)rows * NH * D * 4) + up256((size_t)rows * NH * 4);
}

void shared_attn(const SharedAttnArgs& a, hipStream_t s) {
	int32_t* f = (int32_t*)a.ws;
	int32_t* hst = (int32_t*)((char*)a.ws + up256((size_t)a.rows * a.NH * a.D * 4));
	const dim3 grid(a.NH, a.rows);
	switch (a.D) {
		case 32: hipLaunchKernelGGL(k_shared_attn_row<32>, grid, dim3(256), 0, s, a, f, hst); break;
		case 64: hipLaunchKernelGGL(k_shared_attn_row<64>, grid, dim3(256), 0, s, a, f, hst); break;
		case 128: hipLaunchKernelGGL(k_shared_attn_row<128>, grid, dim3(256), 0, s, a, f, hst); break;
		default: hipLaunchKernelGGL(k_shared_attn_row<256>, grid, dim3(256), 0, s, a, f, hst); break;
	}
	hipLaunchKernelGGL((k_ctx_funnel<1024, 8>), dim3(a.rows), dim3(1024), 0, s, a, f, hst);
}

size_t lora_gemm_workspace(int m, int n, int k) { return up256((size_t)m * n * 4) + up256((size_t)m * kMaxRank); }

void lora_gemm(const LoraGemmArgs& g, hipStream_t s) {
	int32_t* acc = (int32_t*)g.ws;
	int8_t* u = (int8_t*)g.ws + up256((size_t)g.m * g.n * 4);
	GemmArgs ga{};
	ga.a = g.a;
	ga.w = g.w;
	ga.M = g.m;
	ga.N = g.n;
	ga.K = g.k;
	ga.lda = g.k;
	ga.epi.raw_out = acc;
	gemm(ga, s);
	hipLaunchKernelGGL(k_rows_u, dim3(g.m, kMaxRank / 4), dim3(256), 0, s, g, u);
	hipLaunchKernelGGL((k_lora_funnel<1024, 8>), dim3(g.m), dim3(1024), 0, s, g, acc, u);
}

static int pick_slices(int vocab) { return (vocab + kPickSlice - 1) / kPickSlice; }

size_t pick_workspace(int rows, int vocab) { return up256((size_t)rows * pick_slices(vocab) * 8); }

void pick_tokens(const PickArgs& a, hipStream_t s) {
	const int slices = pick_slices(a.vocab);
	unsigned long long* keys = (unsigned long long*)a.ws;
	hipLaunchKernelGGL(k_pick_slice, dim3(slices, a.rows), dim3(kPickBlock), 0, s, a, keys);
	hipLaunchKernelGGL(k_pick_final, dim3(a.rows), dim3(64), 0, s, a, keys, slices);
}

}  // namespace sslm_launch

// ------------------------------------------------------------------------------------------
// C entries
// ------------------------------------------------------------------------------------------
namespace {

using namespace sslm_launch;

constexpr int kMaxRows = 65535;  // a grid's y extent

// A launch on the caller's stream: the stream belongs to the current device, and nothing throws
// past the boundary.
template <typename F>
sslm_status on_stream(void* stream, F&& launch) {
	int cur = -1;
	hipDevice_t of = -1;
	if (hipGetDevice(&cur) != hipSuccess) return SSLM_INVALID_ARGUMENT;
	if (stream && (hipStreamGetDevice((hipStream_t)stream, &of) != hipSuccess || of != cur)) return SSLM_INVALID_ARGUMENT;
	(void)hipGetLastError();  // an error left by an unrelated earlier call is not this call's
	try {
		launch((hipStream_t)stream);
	} catch (const LaunchRefused& e) {
		fprintf(stderr, "sslm_hip: launch refused (%s)\n", e.what);
		return SSLM_HIP_LAUNCH_FAILED;
	} catch (...) {
		return SSLM_HIP_LAUNCH_FAILED;
	}
	return hipGetLastError() == hipSuccess ? SSLM_OK : SSLM_HIP_LAUNCH_FAILED;
}

bool workspace_ok(const void* ws, size_t have, size_t need, sslm_status* st) {
	*st = !ws ? SSLM_INVALID_ARGUMENT : (((uintptr_t)ws % 256) ? SSLM_MISALIGNED_BUFFER : SSLM_BUFFER_TOO_SMALL);
	return ws && (uintptr_t)ws % 256 == 0 && have >= need;
}

}  // namespace

extern "C" {

size_t sslm_hip_shared_attention_workspace(int32_t rows, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                           int32_t prefixes, int64_t max_prefix, int64_t max_own) {
	if (!shared_attn_ok(rows, heads, kv_heads, head_dim) || rows > kMaxRows || prefixes < 0 || prefixes > rows ||
	    max_prefix < 0 || max_own < 0 || max_prefix > SSLM_HIP_ATTENTION_MAX_WIDTH || max_own > SSLM_HIP_ATTENTION_MAX_WIDTH)
		return 0;
	return shared_attn_workspace(rows, heads, kv_heads, head_dim, prefixes, max_prefix, max_own);
}

sslm_status sslm_hip_shared_attention(const sslm_hip_shared_attention_args* p, void* workspace, size_t workspace_bytes,
                                      void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_shared_attention_workspace(p->rows, p->heads, p->kv_heads, p->head_dim, p->prefixes,
	                                                        p->max_prefix, p->max_own);
	if (!need || !p->kv_pool || !p->q || !p->q_scale || !p->khead_m || !p->khead_e || !p->ctx_fold || !p->row_block ||
	    !p->row_width || !p->codes || !p->scales || !p->status)
		return SSLM_INVALID_ARGUMENT;
	if (p->prefixes > 0 && (!p->prefix_rows || !p->prefix_block || !p->prefix_len)) return SSLM_INVALID_ARGUMENT;
	const int64_t half = (int64_t)p->kv_heads * p->cap * p->head_dim;
	if (p->blocks < 1 || p->cap < 1 || p->cap > SSLM_HIP_ATTENTION_MAX_WIDTH || p->k_offset < 0 || p->v_offset < 0 ||
	    p->block_bytes < half || p->k_offset > p->block_bytes - half || p->v_offset > p->block_bytes - half ||
	    p->block_bytes % 16 || p->k_offset % 16 || p->v_offset % 16 || (uintptr_t)p->kv_pool % 16 || (uintptr_t)p->q % 16)
		return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	SharedAttnArgs a{};
	a.rows = p->rows;
	a.NH = p->heads;
	a.NKV = p->kv_heads;
	a.D = p->head_dim;
	a.prefixes = p->prefixes;
	a.blocks = p->blocks;
	a.max_prefix = p->max_prefix;
	a.max_own = p->max_own;
	a.pool = p->kv_pool;
	a.block_bytes = p->block_bytes;
	a.k_off = p->k_offset;
	a.v_off = p->v_offset;
	a.cap = p->cap;
	a.q = p->q;
	a.q_scale = (const Scale*)p->q_scale;
	a.khead_m = p->khead_m;
	a.khead_e = p->khead_e;
	a.ln2_q = p->ln2_q;
	a.b_q = p->b_q;
	a.ca_q = p->ca_q;
	a.ctx_fold = p->ctx_fold;
	a.site = Scale{p->site_m, p->site_e};
	a.row_block = p->row_block;
	a.row_width = p->row_width;
	a.prefix_rows = p->prefix_rows;
	a.prefix_block = p->prefix_block;
	a.prefix_len = p->prefix_len;
	a.codes = p->codes;
	a.scales = (Scale*)p->scales;
	a.status = p->status;
	a.ws = workspace;
	return on_stream(stream, [&](hipStream_t s) { shared_attn(a, s); });
}

size_t sslm_hip_gemm_lora_workspace(int32_t m, int32_t n, int32_t k) {
	if (m < 1 || m > SSLM_HIP_GEMM_LORA_MAX_M || n < 16 || n % 16 || n > kFunnelMaxN || k < 16 || k % 16 ||
	    k > SSLM_HIP_GEMM_LORA_MAX_K)
		return 0;
	return lora_gemm_workspace(m, n, k);
}

sslm_status sslm_hip_gemm_lora_requant(const sslm_hip_gemm_lora_args* p, void* workspace, size_t workspace_bytes,
                                       void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_gemm_lora_workspace(p->m, p->n, p->k);
	if (!need || !p->a || !p->w || !p->fold || !p->in_scale || !p->row_adapter || p->adapter_count < 0 ||
	    (p->adapter_count > 0 && !p->adapters) || !p->codes || !p->scales || !p->status || (uintptr_t)p->a % 16 ||
	    (uintptr_t)p->w % 16)
		return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	static_assert(sizeof(sslm_hip_lora) == sizeof(LoraRef), "one layout");
	LoraGemmArgs g{};
	g.m = p->m;
	g.n = p->n;
	g.k = p->k;
	g.count = p->adapter_count;
	g.a = p->a;
	g.w = p->w;
	g.fold = p->fold;
	g.in_scale = (const Scale*)p->in_scale;
	g.site = Scale{p->site_m, p->site_e};
	g.adapters = (const LoraRef*)p->adapters;
	g.row_adapter = p->row_adapter;
	g.codes = p->codes;
	g.scales = (Scale*)p->scales;
	g.status = p->status;
	g.ws = workspace;
	return on_stream(stream, [&](hipStream_t s) { lora_gemm(g, s); });
}

size_t sslm_hip_pick_workspace(int32_t rows, int32_t vocab) {
	return rows < 1 || rows > kMaxRows || vocab < 1 ? 0 : pick_workspace(rows, vocab);
}

sslm_status sslm_hip_pick_tokens(const sslm_hip_pick_args* p, void* workspace, size_t workspace_bytes, void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_pick_workspace(p->rows, p->vocab);
	if (!need || !p->logits || !p->rules || !p->tokens || p->logits_ld < p->vocab ||
	    (p->adjusted && p->adjusted_ld < p->vocab) || (uintptr_t)p->logits % 4 || (uintptr_t)p->adjusted % 4)
		return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	static_assert(sizeof(sslm_hip_logit_rule) == sizeof(LogitRule), "one layout");
	PickArgs a{};
	a.rows = p->rows;
	a.vocab = p->vocab;
	a.logits = p->logits;
	a.ld = p->logits_ld;
	a.adjusted_ld = p->adjusted_ld;
	a.rules = (const LogitRule*)p->rules;
	a.adjusted = p->adjusted;
	a.tokens = p->tokens;
	a.ws = workspace;
	return on_stream(stream, [&](hipStream_t s) { pick_tokens(a, s); });
}

}  // extern "C"
