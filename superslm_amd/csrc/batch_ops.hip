// Operators of a decode step whose rows differ (batch_ops.h): kernels, launches and C entries.
#include <hip/hip_runtime.h>
#include <stdio.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/sslm_hip.h"
#include "batch_ops.h"
#include "device_util.h"

namespace sslm {

using sslm_launch::LogitRule;

// A pointer that was read from memory is generic to the compiler, whose flat loads count as LDS operations
// too: each wait for LDS would then be one for every load in flight.  All of these point to global memory.
template <typename T>
__device__ __forceinline__ const __attribute__((address_space(1))) T* global_ptr(const T* p) {
	return (const __attribute__((address_space(1))) T*)p;
}
__device__ __forceinline__ v4i global16(const int8_t* p) { return *global_ptr((const v4i*)p); }

struct __attribute__((packed)) unaligned16 {
	v4i v;
};
struct __attribute__((packed)) unaligned4 {
	int32_t v;
};

// ------------------------------------------------------------------------------------------
// attention of rows that share prompts
// ------------------------------------------------------------------------------------------

// Where a row's positions lie: [0, start) in its prefix's block, [start, width) in its own.
struct RowSpan {
	int64_t width, start;
	const int8_t *own, *pre;
	int32_t st, pad;
};

// All lanes of the wave call it for one row.  The tables are read a lane to a prefix, so that the row's
// span costs two round trips whatever the number of prefixes; prefix_rows has to be a division of the
// rows, ascending from at least 0 to at most `rows`.
__device__ __forceinline__ RowSpan row_span(const sslm_launch::SharedAttnArgs& a, int r) {
	RowSpan s{a.row_width[r], 0, a.pool, a.pool, kOk, 0};
	const int blk = a.row_block[r], lane = threadIdx.x & 63;
	bool bad = false;
	int pb = 0;
	int64_t len = -1;
	for (int i0 = 0; i0 < a.prefixes; i0 += 64) {
		const int i = min(i0 + lane, a.prefixes - 1);
		const int x = a.prefix_rows[i], y = a.prefix_rows[i + 1], b = a.prefix_block[i];
		const int64_t l = a.prefix_len[i];
		bad |= x < 0 || y < x || y > a.rows;
		const uint64_t hit = __ballot(x <= r && r < y && i0 + lane < a.prefixes);
		if (hit) {
			const int at = __builtin_ctzll(hit);
			pb = __builtin_amdgcn_readlane(b, at);
			len = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)l >> 32), at) << 32 |
			                (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)l, at));
			if (pb < 0 || pb >= a.blocks || len < 0 || len > a.cap || len > a.max_prefix) s.st = kPositionOverCap;
			else {
				s.pre = a.pool + (int64_t)pb * a.block_bytes;
				s.start = len < s.width ? len : s.width;
			}
		}
	}
	if (__any(bad) || blk < 0 || blk >= a.blocks || s.width < 0 || s.width > a.cap) s.st = kPositionOverCap;
	else s.own += (int64_t)blk * a.block_bytes;
	if (s.st == kOk && s.width - s.start > a.max_own) s.st = kPositionOverCap;
	if (s.st == kOk && s.width == 0) s.st = kSoftmaxRowWidthOutOfDomain;
	return s;
}

struct RowConst {
	int64_t q_ln2, q_b, q_c, ceil;
	int32_t st;
};

// The softmax constants of (row, KV head) (forward_sites.cpp:1805-1830): the general form.
__device__ __forceinline__ RowConst row_const_general(Scale sm, int64_t ln2_q, int64_t b_q, int64_t ca_q, int64_t width) {
	RowConst c{0, 0, 0, 0, kOk};
	if (iexp_scale_constants(sm.m, sm.e, ln2_q, b_q, ca_q, &c.q_ln2, &c.q_b, &c.q_c) != 0) c.st = kIExpScaleDerivationOutOfDomain;
	else c.st = check_softmax_width(c.q_b, c.q_c, width);
	if (c.st == kOk) c.ceil = softmax_ceiling(c.q_b, c.q_c);
	return c;
}

// The same in 64 bits where it fits (iexp_scale_constants' products below 2^63 and 2^126, its shifts in
// [1, 63], check_softmax_width's q_b below 2^24): some forty scalar instructions in the row's chain of
// latencies instead of several hundred.
struct RowScales {
	Scale q;
	int64_t km, ke;
};
__device__ __forceinline__ RowScales row_scales(const sslm_launch::SharedAttnArgs& a, int r, int kvh) {
	return RowScales{a.q_scale[r], a.khead_m[kvh], a.khead_e[kvh]};
}
__device__ __forceinline__ RowConst row_const(const sslm_launch::SharedAttnArgs& a, const RowScales& rs, int64_t width) {
	RowConst c{0, 0, 0, 0, kOk};
	const Scale qs = rs.q;
	const int64_t km = rs.km, ke = rs.ke;
	if (!fits_i32(qs.m) || !fits_i32(km)) {
		c.st = kCarriedScaleMantissaOutOfDomain;
		return c;
	}
	const Scale sm = combine_scale(qs, Scale{km, ke});
	if (!fits_i32(sm.m)) {
		c.st = kCarriedScaleMantissaOutOfDomain;
		return c;
	}
	const int64_t lim = (int64_t)1 << 30;
	// 92 + e and 154 + 2 e in [1, 63] (e <= -46 already gives the latter's bound, e >= -76 its least)
	if (sm.m >= lim && a.ln2_q > 0 && a.ln2_q < lim && a.b_q > 0 && a.b_q < 2 * lim && a.ca_q > 0 && a.ca_q < lim && sm.e >= -76 && sm.e <= -46) {
		const uint64_t rc = (uint64_t)reciprocal_norm(sm.m);  // in (2^31, 2^32]
		const uint64_t ca = (uint64_t)a.ca_q * rc, lo = ca * rc, hi = __umul64hi(ca, rc);
		const int sh = (int)(92 + sm.e), sc = (int)(154 + 2 * sm.e);  // sc even, in [2, 62]
		const uint64_t b = (uint64_t)a.b_q * rc >> sh;
		if ((hi >> sc) == 0 && b < ((uint64_t)1 << 24)) {
			const uint64_t qc = hi << (64 - sc) | lo >> sc, m = b * b + qc;
			if (qc < ((uint64_t)1 << 62) && m >= 1) {
				c.q_ln2 = (int64_t)((uint64_t)a.ln2_q * rc >> sh);
				c.q_b = (int64_t)b;
				c.q_c = (int64_t)qc;
				const bool wide = m > (uint64_t)kSoftmaxMaxSafe || width <= 0 || __umul64hi(m, (uint64_t)width) != 0 || (int64_t)(m * (uint64_t)width) < 0;
				c.st = wide ? kSoftmaxRowWidthOutOfDomain : kOk;
				c.ceil = wide ? 0 : (int64_t)m;
				return c;
			}
		}
	}
	return row_const_general(sm, a.ln2_q, a.b_q, a.ca_q, width);
}

// The layout of one call's launches.  The unit of work is a wave with a tile of 16 query rows and a
// range of positions, a "plane": shared planes cut a prefix into sb positions each and their tiles hold
// the query heads of one KV head of 16 / G neighbouring rows (G heads share a KV head), and the tiles of a block's
// four waves share each K or V row that it loads; own planes cut a row's own positions, their tiles hold the row's G heads.
// The softmax's maximum and sum run over the whole row and every probability is rounded by itself, so no
// rescaling of partial results is exact: three launches -- maxima, sums, P.V -- recompute the scores,
// which cost 8 MFMAs a step of 64 positions at D = 128 where the i-exp of the step's scores costs some
// hundreds of vector instructions, and integer sums join the planes exactly in any order.
// 96 rows of 28 heads over 4 KV heads of 128, 4096 shared positions and 16 .. 384 own: maxima 9.4 us, sums 15.7,
// P.V 25.4, join 5.9.  Bound by the vector instructions of i-exp and probability (issued back to back they take 3.0,
// 7.8 and 12.2 us) at the two waves a SIMD that P.V's registers allow, and by each launch's chain of loads.
struct SaPlan {
	int tb;          // blocks of kSaWaves tiles of shared rows: at least those of every prefix together
	int shared, sb;  // shared planes and the positions of one (a multiple of 64)
	int owned, ob;   // own planes and the positions of one
	int ht;          // tiles of a row's own heads
	int shared_blocks;
};

// (row, KV head): the softmax constants and whether the row is computed at all
struct SaConst {
	int64_t q_ln2, q_b, q_c, ceil;
	int32_t st, pad;
};

struct SaWork {
	RowSpan* span;  // [rows], written with cst by k_sa_max
	SaConst* cst;   // [rows, NKV]
	int32_t* pmax;  // [planes][rows NH]
	int64_t* psum;  // [planes][rows NH]; negative: an i-exp value was refused
	int32_t* part;  // [planes][rows][NH D]
	int32_t* hst;   // [rows, NH] refusals of the softmax
};

constexpr int kSaWaves = 4;

// What a wave works on; the fields that differ by lane belong to query row ri = lane & 15 of its tile.
struct SaJob {
	const int8_t *k, *v;  // the KV head's position 0
	int64_t p0, p1;       // positions of the plane (p1: also the end of what may be read)
	int plane, kvh;
	int r, h;             // by lane: row and query head (r < 0: none)
	int row;              // an own plane's row
	int64_t start, width; // by lane: where the row's own positions begin, and its width
	bool owned, first;    // an own plane; the row's first
};

__device__ __forceinline__ int64_t i64min(int64_t a, int64_t b) { return a < b ? a : b; }

// A wave of the shared planes: false, for its whole block, when there is nothing to do.  A block's waves have
// neighbouring tiles of one prefix and the same positions; a wave past the last tile has no live lane.
__device__ __forceinline__ bool sa_shared_job(const sslm_launch::SharedAttnArgs& a, const SaPlan& pl, SaJob* j) {
	const int blk = blockIdx.x;
	// blocks go to the XCDs in turn: a (KV head, plane)'s tiles stay on one, whose L2 then holds its K/V
	const int grp = (blk / 8 / pl.tb) * 8 + blk % 8;
	int b = (blk / 8) % pl.tb;
	if (grp >= a.NKV * pl.shared) return false;
	j->plane = grp / a.NKV;
	j->kvh = grp % a.NKV;
	const int G = a.NH / a.NKV;
	int p = 0, r0 = 0, r1 = 0;
	for (;; ++p) {  // the block's prefix
		if (p >= a.prefixes) return false;
		r0 = max(0, min(a.prefix_rows[p], a.rows));
		r1 = max(r0, min(a.prefix_rows[p + 1], a.rows));
		const int n = ((r1 - r0) * G + 16 * kSaWaves - 1) / (16 * kSaWaves);
		if (b < n) break;
		b -= n;
	}
	const int tile = b * kSaWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int pb = a.prefix_block[p];
	const int64_t len = a.prefix_len[p];
	j->p0 = (int64_t)j->plane * pl.sb;
	if (pb < 0 || pb >= a.blocks || len < 0 || len > a.cap || len > a.max_prefix || j->p0 >= len) return false;
	j->p1 = i64min(len, j->p0 + pl.sb);
	const int8_t* head = a.pool + (int64_t)pb * a.block_bytes + (int64_t)j->kvh * a.cap * a.D;
	j->k = head + a.k_off;
	j->v = head + a.v_off;
	const int i = tile * 16 + (threadIdx.x & 15);
	const bool live = i < (r1 - r0) * G;
	j->r = live ? r0 + i / G : -1;
	j->h = j->kvh * G + (live ? i % G : 0);
	j->width = live ? a.row_width[j->r] : 0;
	j->start = i64min(len, j->width);
	j->owned = j->first = false;
	return true;
}

// A wave of the own planes (number `w` of them): its row, and the rest once the row's span is known.
__device__ __forceinline__ bool sa_own_row(const sslm_launch::SharedAttnArgs& a, const SaPlan& pl, SaJob* j) {
	const int w = ((int)blockIdx.x - pl.shared_blocks) * kSaWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	if (w >= a.rows * a.NKV * pl.ht * pl.owned) return false;
	const int G = a.NH / a.NKV, plane = w % pl.owned, t = w / pl.owned % pl.ht;
	j->kvh = w / pl.owned / pl.ht % a.NKV;
	const int r = w / pl.owned / pl.ht / a.NKV, i = t * 16 + (threadIdx.x & 15);
	j->owned = true;
	j->first = plane == 0;
	j->plane = pl.shared + plane;
	j->row = r;
	j->r = i < G ? r : -1;
	j->h = j->kvh * G + (i < G ? i : 0);
	return true;
}
__device__ __forceinline__ void sa_own_span(const sslm_launch::SharedAttnArgs& a, const SaPlan& pl, const RowSpan& sp, SaJob* j) {
	j->start = sp.start;
	j->width = sp.width;
	j->p0 = sp.start + (int64_t)(j->plane - pl.shared) * pl.ob;
	j->p1 = i64min(sp.width, j->p0 + pl.ob);
	const int8_t* head = sp.own + (int64_t)j->kvh * a.cap * a.D;
	j->k = head + a.k_off;
	j->v = head + a.v_off;
}

// the wave's query rows as an MFMA operand: lane (ri, g) holds bytes 64 c + 16 g .. + 16 of row ri
template <int D, int NC>
__device__ __forceinline__ void sa_load_q(const sslm_launch::SharedAttnArgs& a, const SaJob& j, v4i (&q)[NC]) {
	const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
	for (int c = 0; c < NC; ++c) {
		const int off = c * 64 + g * 16;
		q[c] = j.r >= 0 && off < D ? load16(a.q + ((size_t)j.r * a.NH + j.h) * D + off) : v4i{0, 0, 0, 0};
	}
}

// K or V rows of 64 positions on their way through LDS (32 D bytes of the wave's own, half the rows at a
// time).  An MFMA operand has a row per lane, which as a global load touches 64 lines an instruction; loaded
// D / 16 lanes to a row and turned in LDS it touches D / 2 (the maxima of 96 rows over 4096 positions: 20 us
// with direct loads, whatever the waves and the loads in flight).  LDS operations of one wave take effect in
// order, so no barrier but the compiler's stands between them.
template <int D>
struct SaRows {
	static constexpr int PER = D / 16;
	v4i r[PER];
	// where 16-byte chunk `ch` of row `row` lies: chunks change places by row, so that one chunk of
	// neighbouring rows covers all banks
	static __device__ __forceinline__ int at(int row, int ch) { return row * D + ((ch ^ (row & (PER - 1))) << 4); }
	// row(p): position p's row; positions past `last` repeat it
	template <typename F>
	__device__ __forceinline__ void load(int64_t p, int64_t last, F&& row) {
		const int lane = threadIdx.x & 63;
#pragma unroll
		for (int u = 0; u < PER; ++u) {
			const int i = lane + 64 * u;
			r[u] = global16(row(i64min(p + i / PER, last)) + i % PER * 16);
		}
	}
	// rows 32 h .. 32 h + 31 into LDS
	__device__ __forceinline__ void stage(int8_t* lds, int h) const {
		const int lane = threadIdx.x & 63;
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
		for (int u = 0; u < PER / 2; ++u) {
			const int c = lane + 64 * u;
			*(v4i*)(lds + at(c / PER, c % PER)) = r[h * (PER / 2) + u];
		}
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		__builtin_amdgcn_wave_barrier();
	}
	// As K: the scores of query operand q, added to s.  Lane (ri, g) gets those of query row ri at positions
	// 16 t + 4 g + v.
	template <int NC>
	__device__ __forceinline__ void scores(int8_t* lds, const v4i (&q)[NC], v4i (&s)[4]) const {
		const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4;
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			stage(lds, h);
#pragma unroll
			for (int t = 2 * h; t < 2 * h + 2; ++t) {
#pragma unroll
				for (int c = 0; c < NC; ++c) {
					const int ch = c * 4 + g;  // q is zero past D
					const v4i k = *(const v4i*)(lds + at((t & 1) * 16 + ri, D < 64 ? ch & (PER - 1) : ch));
					s[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q[c], s[t], 0, 0, 0);
				}
			}
		}
	}
	// As V: context += P V by the byte-transposing LDS read, which gives lane (ri, g) dim 16 dt + ri of the
	// positions in sa_pack's order.  Lane (ri, g) of acc[dt][part] holds dims 16 dt + 4 g .. + 3 of query row ri.
	__device__ __forceinline__ void multiply(int8_t* lds, const v4i& lo, const v4i& nhi, v4i (&acc)[D / 16][2]) const {
		const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4, i = ri >> 1, row = (i >> 2) * 16 + g * 4 + (i & 3);
		v2i half[2][D / 16];
#pragma unroll
		for (int h = 0; h < 2; ++h) {
			stage(lds, h);
#pragma unroll
			for (int dt = 0; dt < D / 16; ++dt)
				half[h][dt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(lds + at(row, dt) + 8 * (ri & 1)));
		}
#pragma unroll
		for (int dt = 0; dt < D / 16; ++dt) {
			const v4i b = v4i{half[0][dt].x, half[0][dt].y, half[1][dt].x, half[1][dt].y};
			acc[dt][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, lo, acc[dt][0], 0, 0, 0);
			acc[dt][1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, nhi, acc[dt][1], 0, 0, 0);
		}
	}
};

// The same from 64 rows that a whole block staged.
template <int D, int NC>
__device__ __forceinline__ void sa_block_scores(const int8_t* lds, const v4i (&q)[NC], v4i (&s)[4]) {
	const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4;
#pragma unroll
	for (int t = 0; t < 4; ++t) {
		s[t] = v4i{0, 0, 0, 0};
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			const int ch = c * 4 + g;
			const v4i k = *(const v4i*)(lds + SaRows<D>::at(t * 16 + ri, D < 64 ? ch & (D / 16 - 1) : ch));
			s[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q[c], s[t], 0, 0, 0);
		}
	}
}
template <int D>
__device__ __forceinline__ void sa_block_multiply(const int8_t* lds, const v4i& lo, const v4i& nhi, v4i (&acc)[D / 16][2]) {
	const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4, i = ri >> 1, row = (i >> 2) * 16 + g * 4 + (i & 3);
#pragma unroll
	for (int dt = 0; dt < D / 16; ++dt) {
		const int8_t* from = lds + SaRows<D>::at(row, dt) + 8 * (ri & 1);  // rows 32 apart change places alike
		const v2i x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)from);
		const v2i y = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(from + 32 * D));
		const v4i b = v4i{x.x, x.y, y.x, y.y};
		acc[dt][0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, lo, acc[dt][0], 0, 0, 0);
		acc[dt][1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, nhi, acc[dt][1], 0, 0, 0);
	}
}

// The i-exp of one query row in doubles, each value exact: with y = q_b - x for a score x below the
// maximum (x <= 30 q_ln2 by the clip), z = floor(x / q_ln2) = floor((x + 1/2) / q_ln2), whose argument is at
// least 1 / (2 q_ln2) from an integer and estimated within (q_b + 30 q_ln2) 2^-51 / q_ln2 of its value;
// base = y + z q_ln2, and base^2 + q_c <= q_b^2 + q_c <= 2^47 by the softmax gate.  `fast` rows have
// 0 <= q_b, q_ln2 <= 2 q_b + 1 (then base^2 <= q_b^2, so no value leaves the domain) and a sum
// below 2^53, exact in doubles.  Eleven instructions a value; the integer form takes some forty.
struct SaExp {
	double ninv, c0, l, qc;
	int32_t add, ymin;
};
__device__ __forceinline__ bool sa_fast(const SaConst& c, int64_t width) {
	return c.q_b >= 0 && c.q_ln2 >= 1 && c.ceil >= 1 && c.q_ln2 <= 2 * c.q_b + 1 && (double)c.ceil * (double)width < 0x1p53;
}
__device__ __forceinline__ SaExp sa_exp_of(const SaConst& c, int32_t top) {
	SaExp e;
	e.l = (double)c.q_ln2;
	e.ninv = -1.0 / e.l;
	e.c0 = -((double)c.q_b + 0.5) * e.ninv;
	e.qc = (double)c.q_c;
	e.add = (int32_t)c.q_b - top;
	e.ymin = (int32_t)(c.q_b - 30 * c.q_ln2);
	return e;
}
__device__ __forceinline__ double sa_exp(const SaExp& e, int32_t score) {
	const double y = (double)max(score + e.add, e.ymin);
	const double z = floor(fma(y, e.ninv, e.c0));
	const double base = fma(z, e.l, y);
	return floor(ldexp(fma(base, base, e.qc), -(int)z));
}

// The wave's rows joined over their planes; a lane's row is read by the lanes ri, ri + 16, ri + 32, ri + 48,
// kSaJoin planes each in flight.
constexpr int kSaJoin = 8;
__device__ __forceinline__ int sa_plane_count(const SaPlan& pl, const SaJob& j, int* shared) {
	const int64_t own = j.width - j.start;
	*shared = (int)((j.start + pl.sb - 1) / pl.sb);
	return *shared + (int)((own + pl.ob - 1) / pl.ob);
}
__device__ __forceinline__ int32_t sa_row_max(const sslm_launch::SharedAttnArgs& a, const SaPlan& pl, const SaWork& w, const SaJob& j, bool live) {
	int sh, m = INT32_MIN;
	const int n = live ? sa_plane_count(pl, j, &sh) : 0;
	const int32_t* at = w.pmax + (size_t)(live ? j.r : 0) * a.NH + j.h;
	for (int i = (threadIdx.x & 63) >> 4; i < n; i += 4 * kSaJoin) {
		int32_t x[kSaJoin];
#pragma unroll
		for (int e = 0; e < kSaJoin; ++e) {
			const int k = min(i + 4 * e, n - 1);
			x[e] = at[(size_t)(k < sh ? k : pl.shared + k - sh) * a.rows * a.NH];
		}
#pragma unroll
		for (int e = 0; e < kSaJoin; ++e) m = max(m, x[e]);  // the last plane may count twice
	}
	m = max(m, __shfl_xor(m, 16, 64));
	return max(m, __shfl_xor(m, 32, 64));
}
// negative: refused
__device__ __forceinline__ int64_t sa_row_sum(const sslm_launch::SharedAttnArgs& a, const SaPlan& pl, const SaWork& w, const SaJob& j, bool live) {
	int sh, bad = 0;
	int64_t m = 0;
	const int n = live ? sa_plane_count(pl, j, &sh) : 0;
	const int64_t* at = w.psum + (size_t)(live ? j.r : 0) * a.NH + j.h;
	for (int i = (threadIdx.x & 63) >> 4; i < n; i += 4 * kSaJoin) {
		int64_t x[kSaJoin];
#pragma unroll
		for (int e = 0; e < kSaJoin; ++e) {
			const int k = min(i + 4 * e, n - 1);
			x[e] = at[(size_t)(k < sh ? k : pl.shared + k - sh) * a.rows * a.NH];
		}
#pragma unroll
		for (int e = 0; e < kSaJoin; ++e)
			if (i + 4 * e < n) {
				bad |= x[e] < 0;
				m += x[e] < 0 ? 0 : x[e];
			}
	}
	for (int o = 16; o < 64; o *= 2) {
		m += __shfl_xor(m, o, 64);
		bad |= __shfl_xor(bad, o, 64);
	}
	return bad ? -1 : m;
}

// Steps of 64 positions over an own plane: `step(p, scores, multiply)`, where multiply(lo, nhi, acc) adds P V (WITH_V).
// The next step's K rows are in flight meanwhile.  LDS: the wave's 32 D bytes.
template <int D, bool WITH_V, int NC, typename F>
__device__ __forceinline__ void sa_own_steps(const SaJob& j, int8_t* lds, const v4i (&q)[NC], F&& step) {
	SaRows<D> k, v;
	v4i s[4];
	const int64_t last = j.p1 - 1;
	auto krow = [&](int64_t p) { return j.k + p * D; };
	auto vrow = [&](int64_t p) { return j.v + p * D; };
	k.load(j.p0, last, krow);
	for (int64_t p = j.p0; p < j.p1; p += 64) {
		s[0] = s[1] = s[2] = s[3] = v4i{0, 0, 0, 0};
		if (WITH_V) v.load(p, last, vrow);
		k.scores(lds, q, s);
		k.load(p + 64, last, krow);
		__builtin_amdgcn_sched_barrier(0);
		step(p, s, [&](const v4i& lo, const v4i& nhi, v4i (&acc)[D / 16][2]) { v.multiply(lds, lo, nhi, acc); });
	}
}

// The same over a shared plane, whose rows all waves of the block use: each thread loads its share of a step's
// rows, AHEAD steps ahead, and stages it into one of two buffers, so a step costs one barrier (buffer b was
// last read before the previous one).  All waves of the block have to come here by the same branch (sa_vote).
// Sums of 96 rows over 4096: 15.8 us, 18.4 with each wave staging its own.  LDS: 64 D bytes a buffer, K's two and then V's two.
template <int D, bool WITH_V, int NC, typename F>
__device__ __forceinline__ void sa_block_steps(const SaJob& j, int8_t* lds, const v4i (&q)[NC], F&& step) {
	constexpr int BS = 64 * kSaWaves, CH = 4 * D, PT = (CH + BS - 1) / BS, PER = D / 16, AHEAD = D <= 128 ? 2 : 1;
	const int64_t last = j.p1 - 1;
	v4i kr[AHEAD][PT], vr[AHEAD][PT], s[4];
	auto load = [&](int64_t p, v4i (&k)[PT], v4i (&v)[PT]) {
#pragma unroll
		for (int u = 0; u < PT; ++u) {
			const int c = min((int)threadIdx.x + u * BS, CH - 1);
			const int64_t at = i64min(p + c / PER, last) * D + c % PER * 16;
			k[u] = global16(j.k + at);
			if (WITH_V) v[u] = global16(j.v + at);
		}
	};
#pragma unroll
	for (int i = 0; i < AHEAD; ++i) load(j.p0 + 64 * i, kr[i], vr[i]);
	int b = 0;
	for (int64_t p0 = j.p0; p0 < j.p1; p0 += 64 * AHEAD) {
#pragma unroll
		for (int i = 0; i < AHEAD; ++i) {
			const int64_t p = p0 + 64 * i;
			if (i && p >= j.p1) break;
			int8_t *kb = lds + b * 64 * D, *vb = lds + (2 + b) * 64 * D;
#pragma unroll
			for (int u = 0; u < PT; ++u) {
				const int c = (int)threadIdx.x + u * BS;
				if (CH % BS == 0 || c < CH) {
					*(v4i*)(kb + SaRows<D>::at(c / PER, c % PER)) = kr[i][u];
					if (WITH_V) *(v4i*)(vb + SaRows<D>::at(c / PER, c % PER)) = vr[i][u];
				}
			}
			load(p + 64 * AHEAD, kr[i], vr[i]);
			__syncthreads();
			sa_block_scores<D>(kb, q, s);
			step(p, s, [&](const v4i& lo, const v4i& nhi, v4i (&acc)[D / 16][2]) { sa_block_multiply<D>(vb, lo, nhi, acc); });
			b ^= 1;
		}
	}
}

// `step` over the wave's plane.
template <int D, bool WITH_V, int NC, typename F>
__device__ __forceinline__ void sa_steps(const SaJob& j, int8_t* lds, const v4i (&q)[NC], F&& step) {
	if (j.owned) sa_own_steps<D, WITH_V>(j, lds + (threadIdx.x >> 6) * 32 * D, q, step);
	else sa_block_steps<D, WITH_V>(j, lds, q, step);
}

// Which bits some live row of a shared plane's block, or of an own plane's wave, has set: what every wave of it then
// branches on alike.  The block's waves meet in the second buffer of K, which none writes before the first step's barrier.
template <int D>
__device__ __forceinline__ int sa_vote(const SaJob& j, int bits, int8_t* lds) {
	int* s_vote = (int*)(lds + 64 * D);
	const int wave = threadIdx.x >> 6;
	int all = (__any(bits & 1) ? 1 : 0) | (__any(bits & 2) ? 2 : 0);
	if (!j.owned) {
		if ((threadIdx.x & 63) == 0) s_vote[wave] = all;
		__syncthreads();
		all = 0;
#pragma unroll
		for (int i = 0; i < kSaWaves; ++i) all |= s_vote[i];
	}
	return __builtin_amdgcn_readfirstlane(all);
}

// How many of the step's positions, counted from the lane's first (4 g), its row has.
__device__ __forceinline__ int sa_left(int64_t p, int64_t end) { return (int)i64min(end - p, 64) - ((threadIdx.x & 63) >> 4) * 4; }

template <int D>
__global__ __launch_bounds__(64 * kSaWaves) void k_sa_max(sslm_launch::SharedAttnArgs a, SaPlan pl, SaWork w) {
	constexpr int NC = (D + 63) / 64;
	__shared__ __attribute__((aligned(16))) int8_t lds[2 * 64 * D];  // also kSaWaves 32 D
	const int lane = threadIdx.x & 63, g = lane >> 4;
	SaJob j;
	RowSpan sp;
	RowScales rs;
	if ((int)blockIdx.x < pl.shared_blocks) {
		if (!sa_shared_job(a, pl, &j)) return;
	} else {
		if (!sa_own_row(a, pl, &j)) return;
		rs = row_scales(a, j.row, j.kvh);
		sp = row_span(a, j.row);
		sa_own_span(a, pl, sp, &j);
	}
	const int64_t end = j.owned ? j.p1 : i64min(j.p1, j.start);  // by lane
	if (j.p0 < j.p1 && (!j.owned || sp.st == kOk)) {
		v4i q[NC];
		sa_load_q<D>(a, j, q);
		int32_t m = INT32_MIN;
		sa_steps<D, false>(j, lds, q, [&](int64_t p, v4i (&s)[4], auto&&) {
			const int left = sa_left(p, end);
#pragma unroll
			for (int t = 0; t < 4; ++t)
#pragma unroll
				for (int v = 0; v < 4; ++v) m = max(m, t * 16 + v < left ? s[t][v] : INT32_MIN);
		});
		m = max(m, __shfl_xor(m, 16, 64));
		m = max(m, __shfl_xor(m, 32, 64));
		if (g == 0 && j.r >= 0) w.pmax[(size_t)j.plane * a.rows * a.NH + (size_t)j.r * a.NH + j.h] = m;
	}
	if (!j.owned || !j.first) return;
	SaConst c{0, 0, 0, 0, sp.st, 0};
	if (c.st == kOk) {
		const RowConst rc = row_const(a, rs, sp.width);
		c = SaConst{rc.q_ln2, rc.q_b, rc.q_c, rc.ceil, rc.st, 0};
	}
	if (lane == 0) {
		w.cst[(size_t)j.row * a.NKV + j.kvh] = c;
		w.span[j.row] = sp;
	}
}

// A wave's job in the launches after k_sa_max.
__device__ __forceinline__ bool sa_job(const sslm_launch::SharedAttnArgs& a, const SaPlan& pl, const SaWork& w, SaJob* j) {
	if ((int)blockIdx.x < pl.shared_blocks) return sa_shared_job(a, pl, j);
	if (!sa_own_row(a, pl, j)) return false;
	const RowSpan sp = w.span[j->row];
	if (sp.st != kOk) return false;
	sa_own_span(a, pl, sp, j);
	return true;
}

template <int D>
__global__ __launch_bounds__(64 * kSaWaves, D <= 128 ? 4 : 2) void k_sa_sum(sslm_launch::SharedAttnArgs a, SaPlan pl, SaWork w) {
	constexpr int NC = (D + 63) / 64;
	__shared__ __attribute__((aligned(16))) int8_t lds[2 * 64 * D];  // also kSaWaves 32 D
	const int g = (threadIdx.x & 63) >> 4;
	SaJob j;
	if (!sa_job(a, pl, w, &j) || j.p0 >= j.p1) return;  // alike for the waves of a shared plane's block
	v4i q[NC];
	sa_load_q<D>(a, j, q);
	const SaConst c = w.cst[(size_t)max(j.r, 0) * a.NKV + j.kvh];
	const bool live = j.r >= 0 && c.st == kOk;  // by lane
	const int32_t top = sa_row_max(a, pl, w, j, live);
	const int64_t end = !live ? 0 : (j.owned ? j.p1 : i64min(j.p1, j.start));
	int64_t sum = 0;
	int bad = 0;
	if (!sa_vote<D>(j, live && !sa_fast(c, j.width), lds)) {
		const SaExp e = sa_exp_of(live ? c : SaConst{1, 1, 0, 1, 0, 0}, top);
		double acc = 0.0;
		sa_steps<D, false>(j, lds, q, [&](int64_t p, v4i (&s)[4], auto&&) {
			const int left = sa_left(p, end);
#pragma unroll
			for (int t = 0; t < 4; ++t)
#pragma unroll
				for (int v = 0; v < 4; ++v) {
					const double x = sa_exp(e, s[t][v]);
					acc += t * 16 + v < left ? x : 0.0;
				}
		});
		sum = (int64_t)acc;
	} else {
		const double inv = 1.0 / (double)c.q_ln2;
		sa_steps<D, false>(j, lds, q, [&](int64_t p, v4i (&s)[4], auto&&) {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				if (p + (i >> 2) * 16 + g * 4 + (i & 3) >= end) continue;
				const int64_t x = iexp_fast_cold((int64_t)s[i >> 2][i & 3] - top, c.q_ln2, inv, c.q_b, c.q_c, c.ceil);
				bad |= x < 0;
				sum += x < 0 ? 0 : x;
			}
		});
	}
	for (int o = 16; o < 64; o *= 2) {
		sum += __shfl_xor(sum, o, 64);
		bad |= __shfl_xor(bad, o, 64);
	}
	if (g == 0 && live) w.psum[(size_t)j.plane * a.rows * a.NH + (size_t)j.r * a.NH + j.h] = bad ? -1 : sum;
}

// The Q15 probability floor(2^15 e / d) in doubles, d the row's sum: for d < 2^36 the truncation of
// (2^15 e + 1/2) / d, which is at least 2^-37 from an integer and estimated within 2^-37; else an estimate
// from below, off by less than one, and the exact remainder (a multiple of 2^-15 below 2^38).
struct SaProb {
	double c1, c2, d;  // small sums: 2^15 / d, 1 / (2 d); else the estimate's factor, unused, d / 2^15
};
__device__ __forceinline__ SaProb sa_prob_of(double d, bool small) {
	SaProb p;
	p.d = d * 0x1p-15;
	p.c1 = small ? 32768.0 / d : (1.0 - 0x1p-50) / p.d;
	p.c2 = 0.5 / d;
	return p;
}
template <bool SMALL>
__device__ __forceinline__ int32_t sa_prob(const SaProb& p, double e) {
	if constexpr (SMALL) return (int32_t)fma(e, p.c1, p.c2);
	const double q = floor(e * p.c1);
	return (int32_t)q + (fma(-q, p.d, e) >= p.d ? 1 : 0);
}

// Probabilities p of 64 positions as two int8 MFMA operands with p = 256 hi + lo: lo is p's low byte taken
// as signed, -hi = floor((127 - p) / 256) in [-128, 0] (hi itself reaches 128).  Byte 4 t + v of lane
// (ri, g) is position 16 t + 4 g + v: the products sum over positions, so the scores' own order serves.
__device__ __forceinline__ void sa_pack(const int32_t (&p)[16], v4i* lo, v4i* nhi) {
#pragma unroll
	for (int t = 0; t < 4; ++t) {
		const uint32_t a = __builtin_amdgcn_perm(p[4 * t + 1], p[4 * t], 0x0c0c0400), b = __builtin_amdgcn_perm(p[4 * t + 3], p[4 * t + 2], 0x0c0c0400);
		(*lo)[t] = (int)(a | b << 16);
		const uint32_t c = __builtin_amdgcn_perm(127 - p[4 * t + 1], 127 - p[4 * t], 0x0c0c0501),
		               d = __builtin_amdgcn_perm(127 - p[4 * t + 3], 127 - p[4 * t + 2], 0x0c0c0501);
		(*nhi)[t] = (int)(c | d << 16);
	}
}

template <int D>
__global__ __launch_bounds__(64 * kSaWaves, D <= 128 ? 2 : 1) void k_sa_pv(sslm_launch::SharedAttnArgs a, SaPlan pl, SaWork w) {
	constexpr int NC = (D + 63) / 64, DT = D / 16;
	__shared__ __attribute__((aligned(16))) int8_t lds[4 * 64 * D];
	const int g = (threadIdx.x & 63) >> 4;
	SaJob j;
	if (!sa_job(a, pl, w, &j)) return;
	const SaConst c = w.cst[(size_t)max(j.r, 0) * a.NKV + j.kvh];
	bool live = j.r >= 0 && c.st == kOk;  // by lane
	const int32_t top = sa_row_max(a, pl, w, j, live);
	const int64_t sum = sa_row_sum(a, pl, w, j, live);
	if (j.first && g == 0 && live) w.hst[(size_t)j.r * a.NH + j.h] = sum < 0 ? kSoftmaxKernelRefusedAfterGateAccepted : kOk;
	if (j.p0 >= j.p1) return;
	live = live && sum >= 0;
	const int64_t den = live && sum > 1 ? sum : 1;
	const int64_t end = !live ? 0 : (j.owned ? j.p1 : i64min(j.p1, j.start));
	v4i q[NC], acc[DT][2], lo, nhi;
	sa_load_q<D>(a, j, q);
#pragma unroll
	for (int d = 0; d < DT; ++d) acc[d][0] = acc[d][1] = v4i{0, 0, 0, 0};
	int32_t pr[16];
	const int form = sa_vote<D>(j, (live && !sa_fast(c, j.width) ? 1 : 0) | (den >= ((int64_t)1 << 36) ? 2 : 0), lds);
	if (!(form & 1)) {
		const SaExp e = sa_exp_of(live ? c : SaConst{1, 1, 0, 1, 0, 0}, top);
		auto run = [&](auto small) {
			constexpr bool SMALL = decltype(small)::value;
			const SaProb pb = sa_prob_of((double)den, SMALL);
			sa_steps<D, true>(j, lds, q, [&](int64_t p, v4i (&s)[4], auto&& multiply) {
				const int left = sa_left(p, end);
#pragma unroll
				for (int i = 0; i < 16; ++i) {
					const int32_t x = sa_prob<SMALL>(pb, sa_exp(e, s[i >> 2][i & 3]));
					pr[i] = (i >> 2) * 16 + (i & 3) < left ? x : 0;
				}
				sa_pack(pr, &lo, &nhi);
				multiply(lo, nhi, acc);
			});
		};
		if (!(form & 2)) run(std::true_type{});
		else run(std::false_type{});
	} else {
		const double inv = 1.0 / (double)c.q_ln2, dinv = 1.0 / (double)den;
		sa_steps<D, true>(j, lds, q, [&](int64_t p, v4i (&s)[4], auto&& multiply) {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				pr[i] = 0;
				if (p + (i >> 2) * 16 + g * 4 + (i & 3) >= end) continue;
				const int64_t x = iexp_fast_cold((int64_t)s[i >> 2][i & 3] - top, c.q_ln2, inv, c.q_b, c.q_c, c.ceil);
				pr[i] = (int32_t)div_rcp_cold(x << 15, den, dinv, 32768);
			}
			sa_pack(pr, &lo, &nhi);
			multiply(lo, nhi, acc);
		});
	}
	if (j.r < 0) return;
	int32_t* out = w.part + ((size_t)j.plane * a.rows + j.r) * a.NH * D + (size_t)j.h * D + 4 * g;
#pragma unroll
	for (int d = 0; d < DT; ++d) *(v4i*)(out + 16 * d) = acc[d][0] - 256 * acc[d][1];
}

// The status of row r, from one thread.  In a model's step (a.tok) a slot's first refusal stays.
__device__ __forceinline__ void sa_status(const sslm_launch::SharedAttnArgs& a, int r, int32_t st) {
	if (!a.tok) a.status[r] = st;
	else set_status(a.status, a.tok[r].slot, a.layer, st);
}
__device__ __forceinline__ bool sa_refused(const sslm_launch::SharedAttnArgs& a, int r) { return a.tok && a.status[a.tok[r].slot] != 0; }

// The fold of this thread's units of four dims, read ahead: unit u's head is the same for all four.
template <int BS, int U>
__device__ __forceinline__ void sa_folds(const sslm_launch::SharedAttnArgs& a, FoldConsts (&fc)[U]) {
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int32_t* cf = a.ctx_fold + 3 * (4 * min((int)threadIdx.x + u * BS, a.NH * a.D / 4 - 1) / a.D);
		fc[u] = fold_consts(cf[0], cf[1], cf[2]);
	}
}

// The fold and funnel of one row's context (checked_chain_funnel.cpp:257-364), U units of four dims per
// thread, unless `first`, the smallest (head << 8) | status of a refusing head, is there.
template <int BS, int U>
__device__ __forceinline__ void sa_finish(const sslm_launch::SharedAttnArgs& a, int r, v4i (&v)[U], const FoldConsts (&fc)[U],
                                          uint32_t first, bool refused, uint32_t* s_red) {
	const int N = a.NH * a.D;
	uint32_t mx = 0;
#pragma unroll
	for (int u = 0; u < U; ++u) {  // a clamped unit repeats the last one
#pragma unroll
		for (int x = 0; x < 4; ++x) {
			v[u][x] = fold_bounded(v[u][x], fc[u]);  // |context| <= 2^15 128
			mx = max(mx, (uint32_t)(v[u][x] < 0 ? -v[u][x] : v[u][x]));
		}
	}
	mx = wave_max32(mx);
	first = ~wave_max32(~first);
	if ((threadIdx.x & 63) == 0) {
		s_red[threadIdx.x >> 6] = mx;
		s_red[BS / 64 + (threadIdx.x >> 6)] = first;
	}
	__syncthreads();
#pragma unroll
	for (int i = 0; i < BS / 64; ++i) {
		mx = max(mx, s_red[i]);
		first = min(first, s_red[BS / 64 + i]);
	}
	if (refused) return;
	if (first != 0xffffffffu) {
		if (threadIdx.x == 0) sa_status(a, r, (int32_t)(first & 0xff));
		return;
	}
	FunnelPlan plan;
	const int32_t st = funnel_plan(__builtin_amdgcn_readfirstlane(mx), nullptr, 0, a.site, &plan);
	if (threadIdx.x == 0) {
		sa_status(a, r, st);
		if (st == kOk) a.scales[r] = plan.out;
	}
	if (st != kOk) return;
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int i = (int)threadIdx.x + u * BS;
		if (4 * i < N) {
			uint32_t o = 0;
#pragma unroll
			for (int x = 0; x < 4; ++x) o |= (uint32_t)(uint8_t)requant_code_f(v[u][x], plan.f) << 8 * x;
			((unaligned4*)(a.codes + (size_t)r * N + 4 * i))->v = (int32_t)o;
		}
	}
}

// The planes' contexts joined and finished, a block per row.
template <int BS, int U>
__global__ __launch_bounds__(BS) void k_sa_out(sslm_launch::SharedAttnArgs a, SaPlan pl, SaWork w) {
	__shared__ uint32_t s_red[2 * BS / 64];
	const int r = blockIdx.x, N = a.NH * a.D, G = a.NH / a.NKV;
	const RowSpan sp = w.span[r];
	// read before this row's own status is written: by one thread, after the block's reduction
	const bool refused = sa_refused(a, r);
	// the first refusing head, heads of one KV head sharing its constants' status
	uint32_t first = 0xffffffffu;
	for (int h = threadIdx.x; h < a.NH; h += BS) {
		const int32_t st = w.cst[(size_t)r * a.NKV + h / G].st;
		const int32_t x = st != kOk ? st : w.hst[(size_t)r * a.NH + h];
		if (x != kOk) first = min(first, (uint32_t)h << 8 | (uint32_t)x);
	}
	const int sh = (int)((sp.start + pl.sb - 1) / pl.sb);
	const int n = sp.st != kOk ? 0 : sh + (int)((sp.width - sp.start + pl.ob - 1) / pl.ob);
	FoldConsts fc[U];
	sa_folds<BS>(a, fc);
	v4i v[U];
	const int32_t* at[U];
#pragma unroll
	for (int u = 0; u < U; ++u) {
		v[u] = v4i{0, 0, 0, 0};
		at[u] = w.part + (size_t)r * N + 4 * min((int)threadIdx.x + u * BS, N / 4 - 1);
	}
	constexpr int PK = 8 / U;  // planes in flight
	for (int k = 0; k < n; k += PK) {
		v4i x[PK][U];
#pragma unroll
		for (int e = 0; e < PK; ++e) {
			const int p = min(k + e, n - 1);
			const size_t off = (size_t)(p < sh ? p : pl.shared + p - sh) * a.rows * N;
#pragma unroll
			for (int u = 0; u < U; ++u) x[e][u] = *(const v4i*)(at[u] + off);
		}
#pragma unroll
		for (int e = 0; e < PK; ++e)
#pragma unroll
			for (int u = 0; u < U; ++u) v[u] += k + e < n ? x[e][u] : v4i{0, 0, 0, 0};
	}
	sa_finish<BS>(a, r, v, fc, first, refused, s_red);
}

// The whole of a short row in one launch: a block per row, its eight waves cut over the KV heads and
// then over the positions, NS steps to a wave whose scores stay in registers; maxima, sums and contexts are
// joined in LDS.  A step is F times 64 positions: where G <= 8 heads would leave half of a tile's columns
// empty, columns 8 .. 15 hold the same heads at the next 64 positions (F = 2), by adding the products of
// the second 64 with a query operand that is zero in the other half; the i-exp, which bounds the
// kernel, then works on full waves.  K and V are read once per row here, from L2 for the prefix's.
// 2 rows of 97 .. 105 positions 11.3 us, 16 of up to 609 18.4 (12 heads over 2 KV heads of 128); in the launches by
// planes 18.8 and 24.1 of kernel time alone.  The chain of one wave's stages bounds it: span, constants, scores, maxima,
// sums, probabilities and products, funnel.
constexpr int kSaRowWaves = 8, kSaRowSteps = 2, kSaRowN = 4096;
template <int D, int F, int NS>
__global__ __launch_bounds__(64 * kSaRowWaves, 2) void k_sa_row(sslm_launch::SharedAttnArgs a) {
	constexpr int NC = (D + 63) / 64, DT = D / 16, NW = kSaRowWaves, BS = 64 * NW, U = kSaRowN / 4 / BS, GP = 16 / F;
	constexpr bool KEEP = NS == 1;  // the i-exp values kept in registers between the sums and the probabilities
	__shared__ __attribute__((aligned(16))) int8_t s_kv[NW][32 * D];
	__shared__ __attribute__((aligned(16))) int32_t s_ctx[kSaRowN];
	__shared__ int32_t s_max[NW][16];
	__shared__ int64_t s_sum[NW][16];
	__shared__ uint32_t s_first, s_red[2 * NW];
	const int r = blockIdx.x, lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4, col = ri % GP, part = ri / GP;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), per = NW / a.NKV, kvh = wave / per, sub = wave % per;
	const int G = a.NH / a.NKV;
	int8_t* lds = s_kv[wave];
	const RowScales rs = row_scales(a, r, kvh);
	const bool refused = sa_refused(a, r);  // before this row's own status is written
	const RowSpan sp = row_span(a, r);
	if (sp.st != kOk) {
		if (threadIdx.x == 0) sa_status(a, r, sp.st);
		return;
	}
	const int64_t head = (int64_t)kvh * a.cap * D, last = sp.width - 1;
	auto krow = [&](int64_t p) { return (p < sp.start ? sp.pre : sp.own) + a.k_off + head + p * D; };
	auto vrow = [&](int64_t p) { return (p < sp.start ? sp.pre : sp.own) + a.v_off + head + p * D; };
	auto base = [&](int n) { return (int64_t)(sub + n * per) * (64 * F); };  // step n's first position
	auto at = [&](int n, int i) { return base(n) + part * 64 + (i >> 2) * 16 + g * 4 + (i & 3); };  // score i's, by lane
	SaJob j{};
	j.r = col < G ? r : -1;
	j.h = kvh * G + (col < G ? col : 0);
	// 64-position blocks of K (V) in flight: a wave alone waits a memory round trip for each that is not
	constexpr int NB = NS * F, AK = NB < 2 ? NB : 2, AV = 1;
	auto block = [&](int b) { return base(b / F) + b % F * 64; };
	SaRows<D> kr[AK], vr[AV];
#pragma unroll
	for (int b = 0; b < AK; ++b) kr[b].load(block(b), last, krow);
	v4i q[F][NC], s[NS][4];
	sa_load_q<D>(a, j, q[0]);
	if constexpr (F == 2) {
#pragma unroll
		for (int c = 0; c < NC; ++c) {
			q[1][c] = part == 1 ? q[0][c] : v4i{0, 0, 0, 0};
			q[0][c] = part == 0 ? q[0][c] : v4i{0, 0, 0, 0};
		}
	}
	FoldConsts fc[U];
	sa_folds<BS>(a, fc);
	if (threadIdx.x == 0) s_first = 0xffffffffu;
	for (int i = threadIdx.x; i < a.NH * D / 4; i += BS) ((v4i*)s_ctx)[i] = v4i{0, 0, 0, 0};
	const RowConst rc = row_const(a, rs, sp.width);
	const SaConst c{rc.q_ln2, rc.q_b, rc.q_c, rc.ceil, rc.st, 0};
	int32_t m = INT32_MIN;
#pragma unroll
	for (int n = 0; n < NS; ++n) {
		if (base(n) > last) break;
		s[n][0] = s[n][1] = s[n][2] = s[n][3] = v4i{0, 0, 0, 0};
#pragma unroll
		for (int f = 0; f < F; ++f) {
			const int b = n * F + f;
			kr[b % AK].scores(lds, q[f], s[n]);
			if (b + AK < NB) kr[b % AK].load(block(b + AK), last, krow);
		}
#pragma unroll
		for (int i = 0; i < 16; ++i) m = max(m, at(n, i) <= last ? s[n][i >> 2][i & 3] : INT32_MIN);
	}
#pragma unroll
	for (int b = 0; b < AV; ++b) vr[b].load(block(b), last, vrow);  // in flight through the softmax
	if (F == 2) m = max(m, __shfl_xor(m, 8, 64));
	m = max(m, __shfl_xor(m, 16, 64));
	m = max(m, __shfl_xor(m, 32, 64));
	if (lane < GP) s_max[wave][lane] = m;
	__syncthreads();
	int32_t top = INT32_MIN;
	for (int i = 0; i < per; ++i) top = max(top, s_max[kvh * per + i][col]);
	const bool ok = c.st == kOk, fast = ok && sa_fast(c, sp.width);
	if (!ok && sub == 0 && lane == 0) atomicMin(&s_first, (uint32_t)(kvh * G) << 8 | (uint32_t)c.st);
	const SaExp e = sa_exp_of(fast ? c : SaConst{1, 1, 0, 1, 0, 0}, top);
	const double inv = fast ? 0.0 : 1.0 / (double)c.q_ln2;
	int64_t sum = 0;
	int bad = 0;
	double ev[KEEP ? NS : 1][16];
	if (fast) {
		double acc = 0.0;
#pragma unroll
		for (int n = 0; n < NS; ++n) {
			if (base(n) > last) break;
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				const double x = at(n, i) <= last ? sa_exp(e, s[n][i >> 2][i & 3]) : 0.0;
				acc += x;
				if (KEEP) ev[n][i] = x;
			}
		}
		sum = (int64_t)acc;
	} else if (ok) {
#pragma unroll
		for (int n = 0; n < NS; ++n) {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				if (at(n, i) > last) continue;
				const int64_t x = iexp_fast_cold((int64_t)s[n][i >> 2][i & 3] - top, c.q_ln2, inv, c.q_b, c.q_c, c.ceil);
				bad |= x < 0;
				sum += x < 0 ? 0 : x;
			}
		}
	}
	for (int o = GP; o < 64; o *= 2) {
		sum += __shfl_xor(sum, o, 64);
		bad |= __shfl_xor(bad, o, 64);
	}
	if (lane < GP) s_sum[wave][lane] = sum;
	if (lane < G && bad) atomicMin(&s_first, (uint32_t)(kvh * G + lane) << 8 | (uint32_t)kSoftmaxKernelRefusedAfterGateAccepted);
	__syncthreads();
	sum = 0;
	for (int i = 0; i < per; ++i) sum += s_sum[kvh * per + i][col];
	const int64_t den = sum > 1 ? sum : 1;
	v4i acc[DT][2], lo, nhi;
#pragma unroll
	for (int d = 0; d < DT; ++d) acc[d][0] = acc[d][1] = v4i{0, 0, 0, 0};
	const bool small = fast && !__any(den >= ((int64_t)1 << 36));
	const SaProb pb = sa_prob_of((double)den, small);
	const double dinv = 1.0 / (double)den;
#pragma unroll
	for (int n = 0; n < NS; ++n) {
		if (base(n) > last || s_first != 0xffffffffu) break;
		int32_t pr[16];
		auto value = [&](int i) { return KEEP ? ev[KEEP ? n : 0][i] : (at(n, i) <= last ? sa_exp(e, s[n][i >> 2][i & 3]) : 0.0); };
		if (small) {
#pragma unroll
			for (int i = 0; i < 16; ++i) pr[i] = sa_prob<true>(pb, value(i));
		} else if (fast) {
#pragma unroll
			for (int i = 0; i < 16; ++i) pr[i] = sa_prob<false>(pb, value(i));
		} else {
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				pr[i] = 0;
				if (at(n, i) > last) continue;
				const int64_t x = iexp_fast_cold((int64_t)s[n][i >> 2][i & 3] - top, c.q_ln2, inv, c.q_b, c.q_c, c.ceil);
				pr[i] = (int32_t)div_rcp_cold(x << 15, den, dinv, 32768);
			}
		}
		sa_pack(pr, &lo, &nhi);
#pragma unroll
		for (int f = 0; f < F; ++f) {
			const v4i z{0, 0, 0, 0};
			const int b = n * F + f;
			vr[b % AV].multiply(lds, F == 1 || part == f ? lo : z, F == 1 || part == f ? nhi : z, acc);
			if (b + AV < NB) vr[b % AV].load(block(b + AV), last, vrow);
		}
	}
	// dims change places within a head by its row, so that a tile's additions meet different banks
	if (col < G) {
		int32_t* ctx = s_ctx + j.h * D;
#pragma unroll
		for (int d = 0; d < DT; ++d)
#pragma unroll
			for (int x = 0; x < 4; ++x) atomicAdd(ctx + (((16 * d + 4 * g) ^ (col * 4 & (D - 1))) + x), acc[d][0][x] - 256 * acc[d][1][x]);
	}
	__syncthreads();
	v4i v[U];
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int i = min((int)threadIdx.x + u * BS, a.NH * D / 4 - 1), h = 4 * i / D;
		v[u] = *(const v4i*)(s_ctx + h * D + ((4 * i % D) ^ (h % G * 4 & (D - 1))));
	}
	sa_finish<BS>(a, r, v, fc, s_first, refused, s_red);
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
	if (i >= g.count) return false;
	const LoraRef& r = g.adapters[i];
	if (r.rank < 1 || r.rank > kMaxRank || !r.a || (uintptr_t)r.a % 16 || !r.ufold || !r.b || !r.dfold) return false;
	*out = g.adapters + i;
	return true;
}

constexpr int kUChunks = 5;

// u = clamp(amp_fold(A x)) of a row (forward_sites.cpp:1066-1086), one wave per rank `rk`.
__device__ __forceinline__ void row_u(const LoraRef& ad, const int8_t* x, int k, int rk, int8_t* u) {
	if (rk >= ad.rank) return;
	const int lane = threadIdx.x & 63;
	const int8_t* w = ad.a + (size_t)rk * k;
	int32_t acc = 0;  // |A.x| <= 128^2 k <= 2^29
	for (int c0 = lane * 16; c0 < k; c0 += 1024 * kUChunks) {  // kUChunks loads of each in flight
		v4i p[kUChunks], q[kUChunks];
#pragma unroll
		for (int i = 0; i < kUChunks; ++i) {
			const int c = min(c0 + 1024 * i, k - 16);
			p[i] = load16(x + c);
			q[i] = global16(w + c);
		}
		__builtin_amdgcn_sched_barrier(0);
#pragma unroll
		for (int i = 0; i < kUChunks; ++i) {
			if (c0 + 1024 * i >= k) p[i] = v4i{0, 0, 0, 0};
#pragma unroll
			for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_sdot4(p[i][j], q[i][j], acc, false);
		}
	}
	acc = wave_sum32(acc);
	if (lane == 0) {
		const auto* fd = global_ptr(ad.ufold + 3 * rk);
		u[rk] = (int8_t)clamp_code(apply_amp_fold((int64_t)acc, fd[0], fd[1], fd[2]));
	}
}

__device__ __forceinline__ void rows_u(const sslm_launch::LoraGemmArgs& g, int t, int rk, int8_t* u) {
	const LoraRef* ad;
	if (!row_adapter(g, t, &ad) || !ad) return;
	row_u(*ad, g.a + (size_t)t * g.k, g.k, rk, u + (size_t)t * kMaxRank);
}

__global__ __launch_bounds__(256) void k_rows_u(sslm_launch::LoraGemmArgs g, int8_t* u) {
	rows_u(g, blockIdx.x, blockIdx.y * 4 + (threadIdx.x >> 6), u);
}

__global__ __launch_bounds__(256) void k_refs_u(sslm_launch::RowsUArgs a) {
	const int t = blockIdx.x, p = blockIdx.z;
	const LoraRef ad = a.refs[p][t];
	if (ad.a) row_u(ad, a.x + (size_t)t * a.K, a.K, blockIdx.y * 4 + (threadIdx.x >> 6), a.u[p] + (size_t)t * kMaxRank);
}

__global__ __launch_bounds__(64) void k_lora_table(const LoraRef* const* rows, int M, int i0, LoraRef* out, int ld) {
	const int t = blockIdx.y * 64 + threadIdx.x, i = i0 + blockIdx.x;
	if (t < M) out[(size_t)i * ld + t] = rows[t] ? rows[t][i] : LoraRef{};
}

// The products of up to 64 rows and their adapters' u in one launch, neither waiting for the other.
// A block holds 16 columns and one plane's share of K, cut over its four waves; each lane streams 16
// bytes of its column's weights per 64-byte chunk (KC loads in flight, the weights being what has to be
// read) against MB MFMA tiles of 16 rows, whose codes come from L2.  The waves' int32 sums are
// joined in LDS and stored as plane blockIdx / tiles of [planes][m][n].  Blocks past the products' do
// rows_u: 16 of them per row, four ranks each.  Bound by the chain of loads of a wave's share: 4 x 1536 x 1536 4.0 us,
// 32 x 4864 x 896 5.7, 64 x 1536 x 8960 15.3 (28 MB: 13.8 of weights, 13.5 of the A of the 41 adapters
// that 64 rows drawn from 64 have on average, 0.5 of codes); as the decode GEMV and a launch of
// k_rows_u 7.6, 9.6 and 29.5.
template <int MB, int KC>
__global__ __launch_bounds__(256) void k_lora_proj(sslm_launch::LoraGemmArgs g, int planes, int32_t* part, int8_t* u) {
	__shared__ v4i s_acc[3][MB][64];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ri = lane & 15, gr = lane >> 4, tiles = g.n / 16;
	if ((int)blockIdx.x >= tiles * planes) {
		const int b = blockIdx.x - tiles * planes;
		rows_u(g, b >> 4, (b & 15) * 4 + wave, u);
		return;
	}
	const int tile = blockIdx.x % tiles, plane = blockIdx.x / tiles, chunks = (g.k + 63) / 64;
	const int per = (chunks + planes * 4 - 1) / (planes * 4), c0 = (plane * 4 + wave) * per, c1 = min(chunks, c0 + per);
	const int8_t* w = g.w + (size_t)(tile * 16 + ri) * g.k + gr * 16;
	const int8_t* x[MB];
#pragma unroll
	for (int i = 0; i < MB; ++i) x[i] = g.a + (size_t)min(i * 16 + ri, g.m - 1) * g.k + gr * 16;
	v4i acc[MB];
#pragma unroll
	for (int i = 0; i < MB; ++i) acc[i] = v4i{0, 0, 0, 0};
	for (int c = c0; c < c1; c += KC) {
		v4i wf[KC], xf[MB][KC];
#pragma unroll
		for (int e = 0; e < KC; ++e) {
			// past the range or K: row 0's bytes, taken as zero on the weights' side
			const bool in = c + e < c1 && (c + e) * 64 + gr * 16 < g.k;
			const int off = in ? (c + e) * 64 : -gr * 16;
			wf[e] = load16(w + off);
#pragma unroll
			for (int i = 0; i < MB; ++i) xf[i][e] = load16(x[i] + off);
		}
		__builtin_amdgcn_sched_barrier(0);  // every load issued before the first is waited for
#pragma unroll
		for (int e = 0; e < KC; ++e)
			if (c + e >= c1 || (c + e) * 64 + gr * 16 >= g.k) wf[e] = v4i{0, 0, 0, 0};
#pragma unroll
		for (int e = 0; e < KC; ++e)
#pragma unroll
			for (int i = 0; i < MB; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[e], xf[i][e], acc[i], 0, 0, 0);
	}
	if (wave) {
#pragma unroll
		for (int i = 0; i < MB; ++i) s_acc[wave - 1][i][lane] = acc[i];
	}
	__syncthreads();
	if (wave) return;
	// lane (ri, gr): columns 16 tile + 4 gr .. + 3 of row 16 i + ri
#pragma unroll
	for (int i = 0; i < MB; ++i) {
		const v4i o = acc[i] + s_acc[0][i][lane] + s_acc[1][i][lane] + s_acc[2][i][lane];
		const int t = i * 16 + ri;
		if (t < g.m) *(v4i*)(part + ((size_t)plane * g.m + t) * g.n + tile * 16 + gr * 4) = o;
	}
}

// A row's u as dot operands of the rows of B, which are taken in pieces of w bytes (16, or 4 where the rank is
// below 16) from the 4 bytes that hold a row's first one: a 16-byte load that is not 4-byte aligned takes
// about twice as long.  A row whose first byte is the f-th of its four spans lora_span bytes from there,
// piece q lies at byte lora_piece of them, and copy f of u has zeros where a piece holds other rows' bytes or
// those of an earlier piece.  n rank is a multiple of 16, so nothing past B is read.
__device__ __forceinline__ int lora_span(int rank, int f) { return (f + rank + 3) & ~3; }
__device__ __forceinline__ int lora_piece(int q, int rank, int f, int w) { return min(w * q, lora_span(rank, f) - w); }
constexpr int kLoraU = 80;  // bytes of a copy: a span of 68 in 16-byte pieces

// A column's folded accumulator plus its adapter's apply_amp_fold(d), |d| <= 128 127 64 < 2^20.  There the
// doubling high multiplication cannot saturate and keeps |x| < 2^20, so that for exponents in [-10, 31] the
// rounding shift is fold_bounded's and a left shift stays below 2^30: with |folded| <= 2^29 the sum needs no
// 64 bits and no saturation.  Other exponents take the general form.
__device__ __forceinline__ int32_t lora_add(int32_t folded, int32_t d, const int32_t (&df)[3], uint32_t* mag) {
	const int e = df[2];
	if ((uint32_t)(e + 10) > 41u) {
		const int64_t x = (int64_t)folded + apply_amp_fold((int64_t)d, df[0], df[1], e);
		*mag = sat_abs_u32(x);
		return sat_i32(x);
	}
	const int32_t hi = (int32_t)(((int64_t)d * df[1] + ((int64_t)1 << 30)) >> 31);
	const int right = max(e, 0);
	const int32_t half = (int32_t)((1u << right) >> 1), neg = e > 0 ? hi >> 31 : 0;
	const int32_t amp = ((hi + half + neg) >> right) << max(-e, 0);
	const int32_t x = folded + (df[0] != 0 ? d : amp);
	*mag = (uint32_t)abs(x);
	return x;
}

// Fold, adapter delta and funnel (forward_sites.cpp:1114-1154) of a row of accumulators (the sum of PL planes).
// Every load of a thread's EPT columns is issued from a clamped index before the first is used (taken column
// by column they cost a round trip each); two pieces of B in flight take more registers and are slower.
// 512 rows of 8192: 10.9 us without adapters, 18.6 at rank 16, 24.8 at rank 32, bound by the B rows and
// folds from L2, some 300 KB a row.
template <int BS, int EPT, int PL>
__global__ __launch_bounds__(BS) void k_lora_funnel(sslm_launch::LoraGemmArgs g, const int32_t* part, const int8_t* u) {
	__shared__ __attribute__((aligned(16))) int8_t s_u[4][kLoraU];
	__shared__ uint32_t s_m[BS / 64];
	const int t = blockIdx.x;
	auto col = [&](int k) { return min((int)threadIdx.x + k * BS, g.n - 1); };
	int32_t v[EPT], fd[EPT][3], pv[PL][EPT];
#pragma unroll
	for (int k = 0; k < EPT; ++k)
#pragma unroll
		for (int i = 0; i < 3; ++i) fd[k][i] = g.fold[3 * col(k) + i];
	const int32_t* at = part + (size_t)t * g.n;
#pragma unroll
	for (int p = 0; p < PL; ++p)
#pragma unroll
		for (int k = 0; k < EPT; ++k) pv[p][k] = at[(size_t)p * g.m * g.n + col(k)];
	const LoraRef* ad;
	const bool ok = row_adapter(g, t, &ad);
	const LoraRef ref = ok && ad ? *ad : LoraRef{};
	const int rank = ref.rank;
	if (rank > 0) {
		const int w = rank >= 16 ? 16 : 4, last = rank % 4 ? 4 : 1;
		for (int x = threadIdx.x; x < last * kLoraU; x += BS) {
			const int f = x / kLoraU, q = x % kLoraU / w, p = lora_piece(q, rank, f, w) + x % w, i = p - f;
			s_u[f][x % kLoraU] = p >= w * q && i >= 0 && i < rank ? u[(size_t)t * kMaxRank + i] : (int8_t)0;
		}
	}
#pragma unroll
	for (int k = 0; k < EPT; ++k) {
		v[k] = pv[0][k];
#pragma unroll
		for (int p = 1; p < PL; ++p) v[k] += pv[p][k];
		v[k] = fold_bounded(v[k], fold_consts(fd[k][0], fd[k][1], fd[k][2]));  // |acc| <= 128^2 k <= 2^29
	}
	__builtin_amdgcn_sched_barrier(0);  // the folds' registers are B's from here on
	uint32_t mx = 0;
	if (rank > 0) {
		int32_t d[EPT] = {}, df[EPT][3];  // |B.u| <= 128 127 64 < 2^31
#pragma unroll
		for (int k = 0; k < EPT; ++k)
#pragma unroll
			for (int i = 0; i < 3; ++i) df[k][i] = global_ptr(ref.dfold)[3 * col(k) + i];
		const int span = lora_span(rank, rank % 4 ? 3 : 0);
		__syncthreads();
		if (rank >= 16) {
			for (int q = 0; 16 * q < span; ++q) {
				v4i x[EPT];
#pragma unroll
				for (int k = 0; k < EPT; ++k) {
					const int off = col(k) * rank;
					x[k] = global_ptr((const unaligned16*)(ref.b + (uint32_t)((off & ~3) + lora_piece(q, rank, off & 3, 16))))->v;
				}
#pragma unroll
				for (int k = 0; k < EPT; ++k) {
					const v4i y = *(const v4i*)(s_u[col(k) * rank & 3] + 16 * q);
#pragma unroll
					for (int i = 0; i < 4; ++i) d[k] = __builtin_amdgcn_sdot4(x[k][i], y[i], d[k], false);
				}
			}
		} else {
			for (int q = 0; 4 * q < span; ++q) {
				int32_t x[EPT];
#pragma unroll
				for (int k = 0; k < EPT; ++k) {
					const int off = col(k) * rank;
					x[k] = global_ptr((const unaligned4*)(ref.b + (uint32_t)((off & ~3) + lora_piece(q, rank, off & 3, 4))))->v;
				}
#pragma unroll
				for (int k = 0; k < EPT; ++k) d[k] = __builtin_amdgcn_sdot4(x[k], *(const int32_t*)(s_u[col(k) * rank & 3] + 4 * q), d[k], false);
			}
		}
#pragma unroll
		for (int k = 0; k < EPT; ++k) {
			uint32_t mag;
			v[k] = lora_add(v[k], d[k], df[k], &mag);
			mx = max(mx, mag);  // a clamped column repeats the last one
		}
	} else {
#pragma unroll
		for (int k = 0; k < EPT; ++k) mx = max(mx, sat_abs_u32(v[k]));
	}
	mx = wave_max32(mx);
	if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = mx;
	__syncthreads();
	if (!ok) {
		if (threadIdx.x == 0) g.status[t] = kBadAdapter;
		return;
	}
	uint32_t m = s_m[0];
#pragma unroll
	for (int i = 1; i < BS / 64; ++i) m = max(m, s_m[i]);
	FunnelPlan plan;
	const Scale in = g.in_scale[t];
	const int32_t st = funnel_plan(__builtin_amdgcn_readfirstlane(m), &in, 1, g.site, &plan);
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
constexpr int kPickSlice = 4096;  // tokens per block: a slice's counts and biases take 48 KB of LDS, three blocks to a CU
constexpr int kPickBlock = 512;

__device__ __forceinline__ bool rule_ok(const LogitRule& r) {
	return r.history_len >= 0 && r.bias_count >= 0 && r.repetition_q16 >= 1 && (r.history_len == 0 || r.history) &&
	       (r.bias_count == 0 || (r.bias_ids && r.bias_values));
}

// A row's token from its best (logit, index) keys: they order by logit, then by the lower index, and 0 marks
// no legal token.
__device__ __forceinline__ int32_t pick_of(uint64_t key) { return key ? (int32_t)(0xffffffffu - (uint32_t)key) : -1; }

// One block per (slice of the vocabulary, row).  Histories and biases touch few of a slice's tokens, so the
// rules' 64-bit arithmetic and its division run over those alone: counts, bias sums and a bit per touched token
// are gathered in LDS while the logits are in flight, and a thread takes its touched tokens one by one.  Bound by
// the logits' traffic: a thread's are 16-byte loads and stores (VEC: rows 16-byte aligned), the row's history
// (read by every slice of it, from L2) four loads at a time.  16 rows of 151936 7.4 us, 128 with histories of 3000
// 40.9 (154 MB: 3.8 TB/s; 47.3 with the arithmetic over every token).  With one slice to a row the block writes
// the token itself.
template <bool VEC>
__global__ __launch_bounds__(kPickBlock) void k_pick_slice(sslm_launch::PickArgs a, unsigned long long* keys) {
	__shared__ __attribute__((aligned(16))) int32_t s_cnt[kPickSlice];
	__shared__ __attribute__((aligned(16))) unsigned long long s_bias[kPickSlice];
	__shared__ uint32_t s_bits[kPickSlice / 32];
	__shared__ uint64_t s_key[kPickBlock / 64];
	constexpr int U = kPickSlice / kPickBlock / 4;
	const int r = blockIdx.y, v0 = blockIdx.x * kPickSlice, n = min(kPickSlice, a.vocab - v0);
	const int32_t* row = a.logits + (int64_t)r * a.ld + v0;
	v4i x[U];
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int j = 4 * ((int)threadIdx.x + u * kPickBlock);
		if (VEC && j + 4 <= n) x[u] = *(const v4i*)(row + j);
		else {
#pragma unroll
			for (int i = 0; i < 4; ++i) x[u][i] = row[min(j + i, n - 1)];
		}
	}
	const LogitRule ru = a.rules[r];
	if (!rule_ok(ru)) {
		if (gridDim.x == 1 && threadIdx.x == 0) a.tokens[r] = -2;
		return;
	}
	const bool seen = ru.history_len > 0, biased = ru.bias_count > 0;
	uint32_t legal[U];  // bit i: token 4 i of the group
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int id = v0 + 4 * ((int)threadIdx.x + u * kPickBlock);
		legal[u] = ru.mask ? global_ptr(ru.mask)[min(id, a.vocab - 1) >> 3] >> (id & 4) : 15u;
	}
	if (seen || biased) {
		const int tid = threadIdx.x;
		int32_t h[4], id = -1, bv = 0;
		auto ids = [&](int64_t i) {
#pragma unroll
			for (int e = 0; e < 4; ++e) h[e] = global_ptr(ru.history)[i64min(i + e * kPickBlock, ru.history_len - 1)];
		};
		auto bias = [&](int64_t i) {
			id = global_ptr(ru.bias_ids)[i64min(i, ru.bias_count - 1)];
			bv = global_ptr(ru.bias_values)[i64min(i, ru.bias_count - 1)];
		};
		if (seen) ids(tid);  // the first ones in flight while LDS is cleared
		if (biased) bias(tid);
		if (tid < kPickSlice / 32) s_bits[tid] = 0;
		for (int i = tid; seen && i < kPickSlice / 4; i += kPickBlock) ((v4i*)s_cnt)[i] = v4i{0, 0, 0, 0};
		for (int i = tid; biased && i < kPickSlice / 2; i += kPickBlock) ((v4i*)s_bias)[i] = v4i{0, 0, 0, 0};
		__syncthreads();
		for (int64_t i = tid; i < ru.history_len; i += 4 * kPickBlock) {
			if (i != tid) ids(i);
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				const int64_t j = (int64_t)h[e] - v0;
				if (i + e * kPickBlock >= ru.history_len || j < 0 || j >= n) continue;
				atomicAdd(&s_cnt[j], 1);
				atomicOr(&s_bits[j >> 5], 1u << (j & 31));
			}
		}
		for (int64_t i = tid; i < ru.bias_count; i += kPickBlock) {
			if (i != tid) bias(i);
			const int64_t j = (int64_t)id - v0;
			if (j < 0 || j >= n) continue;
			atomicAdd(&s_bias[j], (unsigned long long)(int64_t)bv);
			atomicOr(&s_bits[j >> 5], 1u << (j & 31));
		}
		__syncthreads();
#pragma unroll
		for (int u = 0; u < U; ++u) {
			const int j = 4 * (tid + u * kPickBlock);
			for (uint32_t b = s_bits[j >> 5] >> (j & 31) & 15; b; b &= b - 1) {
				const int i = __builtin_ctz(b), c = seen ? s_cnt[j + i] : 0;
				int64_t w = i < 2 ? (i == 0 ? x[u][0] : x[u][1]) : (i == 2 ? x[u][2] : x[u][3]);
				if (c > 0) {
					// (w << 16) / rho: below 2^47, so the double quotient's truncation is the integer one
					w = w > 0 ? (int64_t)((double)(w << 16) / (double)ru.repetition_q16) : (w * ru.repetition_q16) >> 16;
					w -= (int64_t)ru.presence + (int64_t)ru.frequency * c;
				}
				if (biased) w += (int64_t)s_bias[j + i];
#pragma unroll
				for (int e = 0; e < 4; ++e) x[u][e] = i == e ? sat_i32(w) : x[u][e];
			}
		}
	}
	int32_t best = 0;
	int at = -1;
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int j = 4 * ((int)threadIdx.x + u * kPickBlock);
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			int32_t y = x[u][i];
			const bool ok = (legal[u] >> i & 1) != 0;
			y = ok ? y : kI32Min;
			x[u][i] = y;
			if (ok && j + i < n && (at < 0 || y > best)) {
				best = y;
				at = v0 + j + i;
			}
		}
		if (a.adjusted) {
			int32_t* out = a.adjusted + (int64_t)r * a.adjusted_ld + v0;
			if (VEC && j + 4 <= n) __builtin_nontemporal_store(x[u], (v4i*)(out + j));  // nothing here reads it: 8.1 -> 7.4 us at 16 rows
			else {
#pragma unroll
				for (int i = 0; i < 4; ++i)
					if (j + i < n) out[j + i] = x[u][i];
			}
		}
	}
	uint64_t key = at < 0 ? 0 : ((uint64_t)((uint32_t)best ^ 0x80000000u) << 32) | (0xffffffffu - (uint32_t)at);
	for (int o = 32; o > 0; o >>= 1) {
		const uint64_t w = __shfl_xor(key, o, 64);
		key = w > key ? w : key;
	}
	if ((threadIdx.x & 63) == 0) s_key[threadIdx.x >> 6] = key;
	__syncthreads();
	if (threadIdx.x == 0) {
		for (int w = 1; w < kPickBlock / 64; ++w) key = s_key[w] > key ? s_key[w] : key;
		if (gridDim.x == 1) a.tokens[r] = pick_of(key);
		else keys[(size_t)r * gridDim.x + blockIdx.x] = key;
	}
}

__global__ __launch_bounds__(64) void k_append_tokens(int32_t* const* at, const int32_t* token, int n) {
	const int i = blockIdx.x * 64 + threadIdx.x;
	if (i < n && at[i]) *at[i] = token[i];
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
	if (threadIdx.x == 0) a.tokens[r] = pick_of(key);
}

}  // namespace sslm

// ------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------
namespace sslm_launch {

constexpr int kSaTargetWaves = 1536;

static size_t up256(size_t n) { return (n + 255) / 256 * 256; }

bool shared_attn_ok(int rows, int NH, int NKV, int D) {
	return rows >= 1 && NKV >= 1 && NH >= NKV && NH % NKV == 0 && (D == 32 || D == 64 || D == 128 || D == 256) &&
	       (int64_t)NH * D <= kFunnelMaxN;
}

// The most planes of so many steps: they are cut in time and joined by every later launch, and the sum of both is
// least at a count that grows with the root of the steps.  The four launches, so and in as many planes as fill the
// chip: one row of 8 heads over 8000 positions of 128 27.6 and 34.4 us, 2 rows of 12 over 96000 71 and 198.
static int64_t sa_most_planes(int64_t steps) { return std::min<int64_t>(steps, std::max<int64_t>(1, (int64_t)std::sqrt(16.0 * (double)steps))); }

// Planes: enough waves for the chip's 1024 SIMDs, a plane at least one step of 64 positions.  The three launches
// of 96 rows over 4096 positions at kSaTargetWaves 1024, 1536 and 2048: 60, 52 and 59 us.
static SaPlan sa_plan(int rows, int NH, int NKV, int prefixes, int64_t max_prefix, int64_t max_own) {
	SaPlan p{};
	const int G = NH / NKV;
	p.tb = prefixes > 0 && max_prefix > 0 ? rows * G / (16 * kSaWaves) + prefixes : 0;
	const int64_t steps = (max_prefix + 63) / 64, jobs = std::min<int64_t>((int64_t)p.tb * kSaWaves, (int64_t)rows * G / 16 + prefixes) * NKV;
	if (jobs > 0) {
		const int64_t want = std::min<int64_t>(sa_most_planes(steps), std::max<int64_t>(1, (kSaTargetWaves + jobs - 1) / jobs));
		p.sb = (int)((steps + want - 1) / want) * 64;
		p.shared = (int)((max_prefix + p.sb - 1) / p.sb);
	} else {
		p.sb = 64;
	}
	p.ht = (G + 15) / 16;
	const int64_t osteps = std::max<int64_t>(1, (max_own + 63) / 64), ojobs = (int64_t)rows * NKV * p.ht;
	const int64_t owant = std::min<int64_t>(sa_most_planes(osteps), std::max<int64_t>(1, (kSaTargetWaves + ojobs - 1) / ojobs));
	p.ob = (int)((osteps + owant - 1) / owant) * 64;
	p.owned = (int)std::max<int64_t>(1, (max_own + p.ob - 1) / p.ob);
	p.shared_blocks = (NKV * p.shared + 7) / 8 * 8 * p.tb;
	return p;
}

static int64_t sa_blocks(const SaPlan& p, int rows, int NKV) {
	return p.shared_blocks + ((int64_t)rows * NKV * p.ht * p.owned + kSaWaves - 1) / kSaWaves;
}

static size_t sa_work(const SaPlan& p, int rows, int NH, int NKV, int D, char* base, SaWork* w) {
	size_t at = 0;
	auto take = [&](size_t n) {
		char* x = base + at;
		at += up256(n);
		return x;
	};
	const size_t planes = p.shared + p.owned, r = (size_t)rows * NH;
	w->span = (RowSpan*)take((size_t)rows * sizeof(RowSpan));
	w->cst = (SaConst*)take((size_t)rows * NKV * sizeof(SaConst));
	w->pmax = (int32_t*)take(planes * r * 4);
	w->psum = (int64_t*)take(planes * r * 8);
	w->hst = (int32_t*)take(r * 4);
	w->part = (int32_t*)take(planes * r * D * 4);
	return at;
}

// Steps of a wave of k_sa_row, 0 where it does not take the call: more heads, dims or steps than its registers
// hold (a third step spills), the times on either side at the kernel.
static int sa_row_steps(int NH, int NKV, int D, int prefixes, int64_t max_prefix, int64_t max_own) {
	const int G = NH / NKV;
	if (NKV > kSaRowWaves || kSaRowWaves % NKV || G > 16 || NH * D > kSaRowN || D > 128) return 0;
	const int64_t step = G <= 8 ? 128 : 64, steps = ((prefixes > 0 ? max_prefix : 0) + max_own + step - 1) / step;
	const int64_t per = kSaRowWaves / NKV, n = std::max<int64_t>(1, (steps + per - 1) / per);
	return n > kSaRowSteps ? 0 : (int)n;
}

size_t shared_attn_workspace(int rows, int NH, int NKV, int D, int prefixes, int64_t max_prefix, int64_t max_own) {
	SaWork w;
	const SaPlan p = sa_plan(rows, NH, NKV, prefixes, max_prefix, max_own);
	if (sa_blocks(p, rows, NKV) * 64 * kSaWaves > UINT32_MAX) return 0;  // a grid's most threads
	return sa_work(p, rows, NH, NKV, D, nullptr, &w);
}

// Steps of four layers, shared against not, in ms: shapes as heads / KV heads x dims, `n of p` rows with a prompt of p and
// 16 or 32 positions of their own, `beside n of p` one row with a prompt of 20 beside n rows of p without one.
//
// The launches by planes cut all rows over the whole chip: their time hardly grows with the prompts, but with the
// rows' own positions for each CU.  The other attention takes a block per (row, KV head), or per query head, over
// its row alone: its time is the longest row's, once more where the blocks pass the CUs.
//
// Up to one block per (row, KV head) for each CU: where the longest row is ahead of the own positions for each CU by
// kSharedPositions (kSharedPositions64 for less than 128 dims, whose rows the other form passes over faster; a quarter
// more for one row, whose fused layers end), and where it is that long and a block per query head would run.
//   28/4x128: 8 of 1000 0.69 / 0.63, 2 of 2600 0.683 / 0.689, 8 of 4000 0.71 / 0.78, one of 2600 0.687 / 0.651, of 3200 0.690 /
//   0.686, of 3700 0.69 / 0.71; beside 7 of 3000 0.71 / 0.73, 15 of 3000 0.76 / 0.73, 31 of 3000 0.89 / 0.81, 31 of 4400
//   0.95 / 0.88, 39 of 3000 0.97 / 0.91, 39 of 3600 (per head) 1.00 / 1.41.
//   12/2x128: 2 of 2600 0.45 / 0.48, 8 of 2000 0.448 / 0.461, of 8000 0.48 / 0.82; beside 15 of 3000 0.47 / 0.53,
//   47 of 3000 0.62 / 0.59, 63 of 4000 0.73 / 0.67, 127 of 6000 (per head) 1.16 / 2.01.
//   32/8x64: one of 3300 0.408 / 0.375, 2 of 2700 0.406 / 0.379, of 3300 0.405 / 0.401, 8 of 2700 0.420 / 0.425.
//   16/4x256: 2 of 2700 0.56 / 0.69.
// Past it: blocks per query head of at least four to a KV head, up to 128 dims, cost more than the planes whatever
// the lengths once there are kSharedHeadDims for each CU; else the planes have to save kSharedSaved positions for each CU.
//   28/4x128: 65 of 32 0.624 / 0.644, 128 of 32 0.69 / 0.75; beside 64 of 300 0.68 / 0.68, 95 of 4400 1.57 / 2.21.
//   32/8x64: 65 of 32 0.53 / 0.50, 100 of 32 0.57 / 0.58; beside 64 of 300 0.56 / 0.54, 127 of 300 0.65 / 0.69.
//   32/8x128: 33 of 300 0.63 / 0.60, of 1000 0.666 / 0.669, 64 of 1000 0.71 / 0.73; beside 63 of 1000 0.84 / 0.70.
//   16/8x128: 100 of 32 0.57 / 0.54, of 1000 0.62 / 0.78; beside 99 of 1000 0.85 / 0.76.
//   16/4x256: 65 of 32 0.76 / 0.69, 100 of 300 0.851 / 0.859; beside 127 of 300 0.95 / 0.90.
constexpr int64_t kSharedPositions = 2600, kSharedPositions64 = 3400, kSharedHeadDims = 800, kSharedSaved = 1000;
bool shared_attn_pays(const SharedUnit& u, int cus) {
	if ((int64_t)u.rows * u.NKV > cus) {
		if (u.per_head && u.D <= 128 && u.NH >= 4 * u.NKV && (int64_t)u.rows * u.NH * u.D >= kSharedHeadDims * cus) return true;
		return (u.adopted - u.own) * u.NKV / cus >= kSharedSaved;
	}
	const int64_t least = u.D < 128 ? kSharedPositions64 : kSharedPositions;
	if (u.width < (u.rows == 1 ? least + least / 4 : least)) return false;
	return u.per_head || u.width - u.own * u.NKV / cus >= least;
}

template <int D, int F>
static void sa_row_launch(const SharedAttnArgs& a, int steps, hipStream_t s) {
	const dim3 grid(a.rows), block(64 * kSaRowWaves);
	if (steps == 1) hipLaunchKernelGGL((k_sa_row<D, F, 1>), grid, block, 0, s, a);
	else hipLaunchKernelGGL((k_sa_row<D, F, kSaRowSteps>), grid, block, 0, s, a);
}

// Each launch takes lengths and blocks from what the one before wrote: false when one fails, and none follows it.
template <int D>
static bool sa_launch(const SharedAttnArgs& a, const SaPlan& p, const SaWork& w, hipStream_t s) {
	const dim3 grid((uint32_t)sa_blocks(p, a.rows, a.NKV)), block(64 * kSaWaves);
	hipLaunchKernelGGL(k_sa_max<D>, grid, block, 0, s, a, p, w);
	if (hipPeekAtLastError() != hipSuccess) return false;
	hipLaunchKernelGGL(k_sa_sum<D>, grid, block, 0, s, a, p, w);
	if (hipPeekAtLastError() != hipSuccess) return false;
	hipLaunchKernelGGL(k_sa_pv<D>, grid, block, 0, s, a, p, w);
	return hipPeekAtLastError() == hipSuccess;
}

void shared_attn(const SharedAttnArgs& a, hipStream_t s) {
	if (const int n = sa_row_steps(a.NH, a.NKV, a.D, a.prefixes, a.max_prefix, a.max_own)) {
		const bool two = a.NH / a.NKV <= 8;
		if (a.D == 32) two ? sa_row_launch<32, 2>(a, n, s) : sa_row_launch<32, 1>(a, n, s);
		else if (a.D == 64) two ? sa_row_launch<64, 2>(a, n, s) : sa_row_launch<64, 1>(a, n, s);
		else two ? sa_row_launch<128, 2>(a, n, s) : sa_row_launch<128, 1>(a, n, s);
		return;
	}
	const SaPlan p = sa_plan(a.rows, a.NH, a.NKV, a.prefixes, a.max_prefix, a.max_own);
	SaWork w;
	sa_work(p, a.rows, a.NH, a.NKV, a.D, (char*)a.ws, &w);
	bool ok = false;
	switch (a.D) {
		case 32: ok = sa_launch<32>(a, p, w, s); break;
		case 64: ok = sa_launch<64>(a, p, w, s); break;
		case 128: ok = sa_launch<128>(a, p, w, s); break;
		default: ok = sa_launch<256>(a, p, w, s); break;
	}
	if (!ok) return;  // the caller reads the error
	const int units = a.NH * a.D / 4;
	if (units <= 512) hipLaunchKernelGGL((k_sa_out<512, 1>), dim3(a.rows), dim3(512), 0, s, a, p, w);
	else if (units <= 1024) hipLaunchKernelGGL((k_sa_out<512, 2>), dim3(a.rows), dim3(512), 0, s, a, p, w);
	else hipLaunchKernelGGL((k_sa_out<512, 4>), dim3(a.rows), dim3(512), 0, s, a, p, w);
}

// Planes of k_lora_proj (a power of two): a wave's share of K at most ten chunks of 64 bytes, where that
// takes more than one plane (their sums are read back by the funnel).  64 x 1536 x 8960: 15.3 us in the four planes
// that ten chunks give, 16.2 in eight, 24.5 in one.
static int lora_planes(int k) {
	int p = 1;
	while (p < 8 && (k + 63) / 64 > 40 * p) p *= 2;
	return p;
}
constexpr int kLoraProjRows = 64;  // rows k_lora_proj takes; past them the prefill GEMM and k_rows_u

size_t lora_gemm_workspace(int m, int n, int k) {
	const int planes = m <= kLoraProjRows ? lora_planes(k) : 1;
	return up256((size_t)planes * m * n * 4) + up256((size_t)m * kMaxRank);
}

template <int BS, int EPT>
static void lora_funnel(const LoraGemmArgs& g, int planes, const int32_t* part, const int8_t* u, hipStream_t s) {
	const dim3 grid(g.m), block(BS);
	switch (planes) {
		case 1: hipLaunchKernelGGL((k_lora_funnel<BS, EPT, 1>), grid, block, 0, s, g, part, u); break;
		case 2: hipLaunchKernelGGL((k_lora_funnel<BS, EPT, 2>), grid, block, 0, s, g, part, u); break;
		case 4: hipLaunchKernelGGL((k_lora_funnel<BS, EPT, 4>), grid, block, 0, s, g, part, u); break;
		default: hipLaunchKernelGGL((k_lora_funnel<BS, EPT, 8>), grid, block, 0, s, g, part, u); break;
	}
}

void lora_gemm(const LoraGemmArgs& g, hipStream_t s) {
	const int planes = g.m <= kLoraProjRows ? lora_planes(g.k) : 1;
	int32_t* part = (int32_t*)g.ws;
	int8_t* u = (int8_t*)g.ws + up256((size_t)planes * g.m * g.n * 4);
	if (g.m <= kLoraProjRows) {
		const dim3 grid(g.n / 16 * planes + (g.count > 0 ? g.m * (kMaxRank / 4) : 0));
		auto proj = [&](auto mb) {
			// loads in flight against waves per SIMD: 3 chunks of 64 rows' codes take as many registers as
			// let u's waves in (64 x 1536 x 8960 with 64 adapters: 15.0 us, 17.8 at 10 chunks)
			constexpr int MB = decltype(mb)::value, KC = MB == 4 ? 3 : 4;
			hipLaunchKernelGGL((k_lora_proj<MB, KC>), grid, dim3(256), 0, s, g, planes, part, u);
		};
		if (g.m <= 16) proj(std::integral_constant<int, 1>{});
		else if (g.m <= 32) proj(std::integral_constant<int, 2>{});
		else proj(std::integral_constant<int, 4>{});
	} else {
		GemmArgs ga{};
		ga.a = g.a;
		ga.w = g.w;
		ga.M = g.m;
		ga.N = g.n;
		ga.K = g.k;
		ga.lda = g.k;
		ga.epi.raw_out = part;
		gemm(ga, s);
		if (g.count > 0) hipLaunchKernelGGL(k_rows_u, dim3(g.m, kMaxRank / 4), dim3(256), 0, s, g, u);
	}
	if (g.n <= 2048) lora_funnel<512, 4>(g, planes, part, u, s);
	else if (g.n <= 5120) lora_funnel<1024, 5>(g, planes, part, u, s);
	else lora_funnel<1024, 8>(g, planes, part, u, s);
}

void lora_table(const LoraRef* const* rows, int M, int l0, int l1, LoraRef* out, int ld, hipStream_t s) {
	hipLaunchKernelGGL(k_lora_table, dim3((l1 - l0) * 7, (M + 63) / 64), dim3(64), 0, s, rows, M, l0 * 7, out, ld);
}

void rows_u(const RowsUArgs& a, hipStream_t s) {
	hipLaunchKernelGGL(k_refs_u, dim3(a.M, kMaxRank / 4, a.nproj), dim3(256), 0, s, a);
}

static int pick_slices(int vocab) { return (int)(((int64_t)vocab + kPickSlice - 1) / kPickSlice); }

void append_tokens(int32_t* const* at, const int32_t* token, int n, hipStream_t s) {
	hipLaunchKernelGGL(k_append_tokens, dim3((n + 63) / 64), dim3(64), 0, s, at, token, n);
}

size_t pick_workspace(int rows, int vocab) { return up256((size_t)rows * pick_slices(vocab) * 8); }

void pick_tokens(const PickArgs& a, hipStream_t s) {
	const int slices = pick_slices(a.vocab);
	unsigned long long* keys = (unsigned long long*)a.ws;
	const bool vec = a.ld % 4 == 0 && (uintptr_t)a.logits % 16 == 0 && (!a.adjusted || (a.adjusted_ld % 4 == 0 && (uintptr_t)a.adjusted % 16 == 0));
	if (vec) hipLaunchKernelGGL(k_pick_slice<true>, dim3(slices, a.rows), dim3(kPickBlock), 0, s, a, keys);
	else hipLaunchKernelGGL(k_pick_slice<false>, dim3(slices, a.rows), dim3(kPickBlock), 0, s, a, keys);
	if (slices > 1) hipLaunchKernelGGL(k_pick_final, dim3(a.rows), dim3(64), 0, s, a, keys, slices);
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
