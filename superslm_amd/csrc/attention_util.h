// What the attention kernels of batch_ops.hip and cache_ops.hip share: loads of pointers read from memory, the
// softmax's constants of a row, its i-exp and probabilities in doubles, K and V rows through LDS.
#pragma once

#include "device_util.h"

namespace sslm {

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

__device__ __forceinline__ int64_t i64min(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t i64max(int64_t a, int64_t b) { return a < b ? b : a; }

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
__device__ __forceinline__ RowConst row_const(const RowScales& rs, int64_t ln2_q, int64_t b_q, int64_t ca_q, int64_t width) {
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
	if (sm.m >= lim && ln2_q > 0 && ln2_q < lim && b_q > 0 && b_q < 2 * lim && ca_q > 0 && ca_q < lim && sm.e >= -76 && sm.e <= -46) {
		const uint64_t rc = (uint64_t)reciprocal_norm(sm.m);  // in (2^31, 2^32]
		const uint64_t ca = (uint64_t)ca_q * rc, lo = ca * rc, hi = __umul64hi(ca, rc);
		const int sh = (int)(92 + sm.e), sc = (int)(154 + 2 * sm.e);  // sc even, in [2, 62]
		const uint64_t b = (uint64_t)b_q * rc >> sh;
		if ((hi >> sc) == 0 && b < ((uint64_t)1 << 24)) {
			const uint64_t qc = hi << (64 - sc) | lo >> sc, m = b * b + qc;
			if (qc < ((uint64_t)1 << 62) && m >= 1) {
				c.q_ln2 = (int64_t)((uint64_t)ln2_q * rc >> sh);
				c.q_b = (int64_t)b;
				c.q_c = (int64_t)qc;
				const bool wide = m > (uint64_t)kSoftmaxMaxSafe || width <= 0 || __umul64hi(m, (uint64_t)width) != 0 || (int64_t)(m * (uint64_t)width) < 0;
				c.st = wide ? kSoftmaxRowWidthOutOfDomain : kOk;
				c.ceil = wide ? 0 : (int64_t)m;
				return c;
			}
		}
	}
	return row_const_general(sm, ln2_q, b_q, ca_q, width);
}

// (row, KV head): the softmax constants and whether the row is computed at all
struct SaConst {
	int64_t q_ln2, q_b, q_c, ceil;
	int32_t st, pad;
};

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
	// at(u): this lane's chunk u, byte 16 (i % PER) of row i / PER, i = lane + 64 u
	template <typename F>
	__device__ __forceinline__ void load_at(F&& at) {
#pragma unroll
		for (int u = 0; u < PER; ++u) r[u] = at(u);
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
		const v4i x[2] = {lo, nhi};
		multiply(lds, x, acc);
	}
	template <int NP>
	__device__ __forceinline__ void multiply(int8_t* lds, const v4i (&x)[NP], v4i (&acc)[D / 16][NP]) const {
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
#pragma unroll
			for (int i = 0; i < NP; ++i) acc[dt][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b, x[i], acc[dt][i], 0, 0, 0);
		}
	}
};

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

// The same for p up to 2^23 (a probability times 2^e, e <= 8) as three operands, p = x[0] - 256 x[1] - 65536 x[2]: p's
// low byte taken as signed, and n = floor((127 - p) / 256) in [-2^15, 0] as its own signed low byte and the rest in [-128, 0].
__device__ __forceinline__ void sa_pack3_word(int32_t p0, int32_t p1, int32_t p2, int32_t p3, uint32_t (&x)[3]) {
	const int32_t n0 = 127 - p0, n1 = 127 - p1, n2 = 127 - p2, n3 = 127 - p3;
	x[0] = __builtin_amdgcn_perm(p1, p0, 0x0c0c0400) | __builtin_amdgcn_perm(p3, p2, 0x0c0c0400) << 16;
	x[1] = __builtin_amdgcn_perm(n1, n0, 0x0c0c0501) | __builtin_amdgcn_perm(n3, n2, 0x0c0c0501) << 16;
	x[2] = __builtin_amdgcn_perm(n1 + 32768, n0 + 32768, 0x0c0c0602) | __builtin_amdgcn_perm(n3 + 32768, n2 + 32768, 0x0c0c0602) << 16;
}
__device__ __forceinline__ void sa_pack3(const int32_t (&p)[16], v4i (&x)[3]) {
#pragma unroll
	for (int t = 0; t < 4; ++t) {
		uint32_t y[3];
		sa_pack3_word(p[4 * t], p[4 * t + 1], p[4 * t + 2], p[4 * t + 3], y);
#pragma unroll
		for (int n = 0; n < 3; ++n) x[n][t] = (int)y[n];
	}
}

}  // namespace sslm
