// A cache in pages (cache_ops.h): kernels, launches and C entries.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/sslm_hip.h"
#include "attention_util.h"
#include "cache_ops.h"
#include "entry_util.h"

namespace sslm {

using sslm_launch::CacheAttnArgs;
using sslm_launch::CacheStoreArgs;
using sslm_launch::kMaxShift;
using sslm_launch::kMaxUnits;
using sslm_launch::PageCompactArgs;
using sslm_launch::Pages;
using sslm_launch::PageUpdateArgs;

__device__ __forceinline__ int64_t pages_for(int64_t positions, int lp) { return (positions + ((int64_t)1 << lp) - 1) >> lp; }

// ------------------------------------------------------------------------------------------
// pages change hands
// ------------------------------------------------------------------------------------------
constexpr int kPlanBlock = 1024;

// The sum of v over the threads before this one; *total: over all.  s: kPlanBlock / 64 words.
template <typename T>
__device__ __forceinline__ T block_before(T v, T* total, T* s) {
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	T x = v;
	for (int o = 1; o < 64; o *= 2) {
		const T y = __shfl_up(x, o, 64);
		x += lane >= o ? y : 0;
	}
	__syncthreads();
	if (lane == 63) s[wave] = x;
	__syncthreads();
	T before = 0, all = 0;
#pragma unroll
	for (int i = 0; i < kPlanBlock / 64; ++i) {
		before += i < wave ? s[i] : 0;
		all += s[i];
	}
	*total = all;
	return before + x - v;
}

// What a plan leaves for the launch that carries it out.
struct PlanWork {
	int32_t* state;   // [0]: whether there is anything to do, [1]: pages to copy
	// [rows] a row's first free page in `free`, the page it gets a copy of or -1, its pages that stay, all of its pages: keep and room
	// themselves may be the buffer that new_lengths goes to
	v4i* row;
	int32_t* free;    // [pages] free pages in the order they are given out (compaction: the holes)
	int32_t *from, *to;  // pages to copy
	int32_t* old;     // [rows, table_ld] the tables as they were, where the new ones take their place
};

__global__ __launch_bounds__(256) void k_table_copy(const int32_t* from, int32_t* to, int64_t n) {
	for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = from[i];
}

// One block: bitmaps of the pages that rows hold (seen), hold more than once (multi), and hold without writing
// into them or keep from outside (fixed), in LDS; then who gets a copy, how many pages each row takes, and the free
// pages in ascending order.  Bound by its chain of loads (a row's numbers, its source's length, the tables) and of block sums:
// 6.2 us for 4 rows and 114 pages, 9.2 for 128 rows of 16 pages; a block per row would need its answers joined by further launches.
constexpr int kLowSlots = 2048;
constexpr int kWrites = 1 << 30;  // beside a row's number of kept pages: it writes into the last of them
__global__ __launch_bounds__(kPlanBlock) void k_update_plan(PageUpdateArgs a, const int32_t* tables, PlanWork w) {
	extern __shared__ uint32_t lds[];
	__shared__ int64_t s_scan[kPlanBlock / 64];
	__shared__ int s_bad, s_most, s_low[kLowSlots];  // s_low: the lowest row that writes into a page of the slot
	const int tid = threadIdx.x, words = (a.pages + 31) / 32;
	uint32_t *seen = lds, *multi = seen + words, *fixed = multi + words;
	int32_t *s_src = (int32_t*)(fixed + words), *s_kept = s_src + a.rows, *s_tail = s_kept + a.rows;
	const int64_t cap = (int64_t)a.table_ld << a.lp;
	if (tid == 0) {
		s_bad = a.rows;
		s_most = 0;
	}
	for (int i = tid; i < 3 * words; i += kPlanBlock) lds[i] = 0;
	for (int i = tid; i < kLowSlots; i += kPlanBlock) s_low[i] = a.rows;
	__syncthreads();
	for (int r = tid; r < a.rows; r += kPlanBlock) {
		const int s = a.source[r];
		const int64_t keep = a.keep[r], room = a.room[r], len = s >= 0 && s < a.rows ? a.lengths[s] : 0;
		const bool ok = s >= -1 && s < a.rows && len >= 0 && len <= cap && keep >= 0 && keep <= len && room >= keep && room <= cap;
		if (!ok) atomicMin(&s_bad, r);
		const int kept = ok ? (int)pages_for(keep, a.lp) : 0;
		const bool writes = ok && (keep & (((int64_t)1 << a.lp) - 1)) && room > keep;
		s_src[r] = s;
		s_kept[r] = kept | (writes ? kWrites : 0);
		if (kept) atomicMax(&s_most, kept);
	}
	if (a.held)
		for (int p = tid; p < a.pages; p += kPlanBlock)
			if (a.held[p]) atomicOr(&fixed[p >> 5], 1u << (p & 31));
	__syncthreads();
	const uint32_t most = s_most;
	const uint64_t cells = (uint64_t)a.rows * most;
	for (uint64_t c0 = tid; c0 < cells; c0 += 4 * kPlanBlock) {
		int r[4], i[4], p[4];
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			const uint64_t c = c0 + u * kPlanBlock;
			r[u] = cells >> 32 ? (int)(c / most) : (int)((uint32_t)c / most);
			i[u] = (int)(c - (uint64_t)r[u] * most);
			const bool in = c < cells && i[u] < (s_kept[min(r[u], a.rows - 1)] & ~kWrites);
			p[u] = in ? tables[(int64_t)s_src[r[u]] * a.table_ld + i[u]] : 0;
			r[u] = in ? r[u] : -1;
		}
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			if (r[u] < 0) continue;
			if (p[u] < 0 || p[u] >= a.pages) {
				atomicMin(&s_bad, r[u]);
				continue;
			}
			const uint32_t bit = 1u << (p[u] & 31);
			if (atomicOr(&seen[p[u] >> 5], bit) & bit) atomicOr(&multi[p[u] >> 5], bit);
			if (i[u] == (s_kept[r[u]] ^ kWrites) - 1) s_tail[r[u]] = p[u];
			else atomicOr(&fixed[p[u] >> 5], bit);
		}
	}
	__syncthreads();
	if (s_bad < a.rows) {
		if (tid == 0) {
			a.result[0] = SSLM_INVALID_ARGUMENT;
			a.result[1] = a.result[2] = 0;
			a.result[3] = s_bad;
			w.state[0] = 0;
		}
		return;
	}
	// pages that only rows which write into them hold stay with the lowest of these
	auto slot = [](int p) { return (int)((uint32_t)p * 2654435761u >> 21); };
	auto contested = [&](int r) {
		const int p = s_tail[r];
		const uint32_t bit = 1u << (p & 31);
		return (multi[p >> 5] & bit) && !(fixed[p >> 5] & bit);
	};
	for (int r = tid; r < a.rows; r += kPlanBlock)
		if ((s_kept[r] & kWrites) && contested(r)) atomicMin(&s_low[slot(s_tail[r])], r);
	__syncthreads();
	int64_t wants = 0, copies = 0;
	for (int r0 = 0; r0 < a.rows; r0 += kPlanBlock) {
		const int r = r0 + tid;
		int64_t n = 0;
		int t = -1, kept = 0, need = 0;
		if (r < a.rows) {
			if (s_kept[r] & kWrites) {
				const int p = s_tail[r];
				bool copy = fixed[p >> 5] >> (p & 31) & 1;
				if (contested(r)) {
					const int low = s_low[slot(p)];
					copy = low != r && s_tail[low] == p;
					for (int q = low; low != r && !copy && q < r; ++q) copy = (s_kept[q] & kWrites) && s_tail[q] == p;  // another page's slot
				}
				if (copy) t = p;
			}
			kept = s_kept[r] & ~kWrites;
			need = (int)pages_for(a.room[r], a.lp);
			n = need - kept + (t >= 0);
		}
		int64_t all;  // pages below 2^40, copies above
		const int64_t before = block_before<int64_t>(n + ((int64_t)(t >= 0) << 40), &all, s_scan), mine = (before >> 40) + copies;
		if (r < a.rows) {
			const int off = (int)min((before & (((int64_t)1 << 40) - 1)) + wants, (int64_t)INT32_MAX);
			w.row[r] = v4i{off, t, kept, need};
			if (t >= 0) {
				w.from[mine] = t;
				w.to[mine] = off;  // its place among the free pages
			}
		}
		wants += all & (((int64_t)1 << 40) - 1);
		copies += all >> 40;
	}
	// free pages: neither seen nor held; a thread's are those of neighbouring words
	const int per = (words + kPlanBlock - 1) / kPlanBlock;
	auto free_bits = [&](int i) {
		const uint32_t valid = a.pages - 32 * i >= 32 ? ~0u : (1u << (a.pages - 32 * i)) - 1;
		return ~(seen[i] | fixed[i]) & valid;
	};
	int64_t mine = 0, total;
	for (int i = tid * per; i < min(words, (tid + 1) * per); ++i) mine += __popc(free_bits(i));
	int64_t at = block_before<int64_t>(mine, &total, s_scan);
	const bool ok = wants <= total;
	if (ok)
		for (int i = tid * per; i < min(words, (tid + 1) * per) && at < wants; ++i)
			for (uint32_t b = free_bits(i); b && at < wants; b &= b - 1) w.free[at++] = 32 * i + __builtin_ctz(b);
	if (tid == 0) {
		a.result[0] = ok ? SSLM_OK : SSLM_KV_POOL_EXHAUSTED;
		a.result[1] = (int32_t)i64max(total - wants, INT32_MIN);
		a.result[2] = ok ? (int32_t)copies : 0;
		a.result[3] = -1;
		w.state[0] = ok;
		w.state[1] = ok ? (int32_t)copies : 0;
	}
}

// Pages from one place of the pool to another, 16 KB to a block and step: no page is both read and written.  Bound by HBM: 283 MB
// (read + written) in 60 us, 4.7 TB/s (47 where the caches still hold some of them); a handful of pages is a launch's 4 us.
constexpr int kCopyChunk = 16384;
template <typename F>
__device__ __forceinline__ void copy_pages(int8_t* pool, int64_t page_bytes, int n, F&& pair) {
	const int chunks = (int)((page_bytes + kCopyChunk - 1) / kCopyChunk);
	for (int64_t i = blockIdx.x; i < (int64_t)n * chunks; i += gridDim.x) {
		const int c = (int)(i / chunks);
		const int64_t at = (i - (int64_t)c * chunks) * kCopyChunk;
		int from, to;
		pair(c, &from, &to);
		const int8_t* src = pool + from * page_bytes + at;
		int8_t* dst = pool + to * page_bytes + at;
		const int left = (int)i64min(page_bytes - at, kCopyChunk) / 16;
		v4i x[kCopyChunk / 4096];
#pragma unroll
		for (int u = 0; u < kCopyChunk / 4096; ++u) x[u] = load16(src + 16 * min((int)threadIdx.x + 256 * u, left - 1));
#pragma unroll
		for (int u = 0; u < kCopyChunk / 4096; ++u)
			if ((int)threadIdx.x + 256 * u < left) *(v4i*)(dst + 16 * (threadIdx.x + 256 * u)) = x[u];
	}
}

__global__ __launch_bounds__(256) void k_update_apply(PageUpdateArgs a, const int32_t* tables, PlanWork w) {
	if (!w.state[0]) return;
	const int64_t cells = (int64_t)a.rows * a.table_ld;
	for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < cells; c += (int64_t)gridDim.x * 256) {
		const int r = (int)(c / a.table_ld), i = (int)(c - (int64_t)r * a.table_ld);
		const v4i row = w.row[r];
		const int off = row.x, kept = row.z, need = row.w;
		const bool copied = row.y >= 0;
		int p = -1;
		if (i < kept) p = copied && i == kept - 1 ? w.free[off] : tables[(int64_t)a.source[r] * a.table_ld + i];
		else if (i < need) p = w.free[off + copied + i - kept];
		a.new_tables[c] = p;
		if (i == 0) a.new_lengths[r] = a.room[r];
	}
	copy_pages(a.pool, a.page_bytes, w.state[1], [&](int c, int* from, int* to) {
		*from = w.from[c];
		*to = w.free[w.to[c]];
	});
}

// One block: the pages in use and those held as bitmaps; the boundary before which the movable ones come to lie;
// the holes before it and the movers after it, both in ascending order.  The same chain as the update's plan: 6.6 us for 6 rows,
// 9.7 for 100 rows and 800 pages.
__global__ __launch_bounds__(kPlanBlock) void k_compact_plan(PageCompactArgs a, PlanWork w) {
	extern __shared__ uint32_t lds[];
	__shared__ int64_t s_scan[kPlanBlock / 64];
	__shared__ int s_bad, s_most, s_edge, s_top;
	const int tid = threadIdx.x, words = (a.pages + 31) / 32;
	uint32_t *live = lds, *held = live + words;
	int32_t *rank = (int32_t*)(held + words), *s_len = rank + words;  // s_len: a row's pages
	const int64_t cap = (int64_t)a.table_ld << a.lp;
	if (tid == 0) {
		s_bad = a.rows;
		s_most = 0;
		s_edge = a.pages;
		s_top = 0;
	}
	for (int i = tid; i < 2 * words; i += kPlanBlock) lds[i] = 0;
	__syncthreads();
	for (int r = tid; r < a.rows; r += kPlanBlock) {
		const int64_t len = a.lengths[r];
		const bool ok = len >= 0 && len <= cap;
		if (!ok) atomicMin(&s_bad, r);
		s_len[r] = ok ? (int)pages_for(len, a.lp) : 0;
		if (ok && len) atomicMax(&s_most, s_len[r]);
	}
	if (a.held)
		for (int p = tid; p < a.pages; p += kPlanBlock)
			if (a.held[p]) atomicOr(&held[p >> 5], 1u << (p & 31));
	__syncthreads();
	const uint32_t most = s_most;
	const uint64_t cells = (uint64_t)a.rows * most;
	for (uint64_t c0 = tid; c0 < cells; c0 += 4 * kPlanBlock) {
		int r[4], p[4];
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			const uint64_t c = c0 + u * kPlanBlock;
			r[u] = cells >> 32 ? (int)(c / most) : (int)((uint32_t)c / most);
			const int i = (int)(c - (uint64_t)r[u] * most);
			const bool in = c < cells && i < s_len[min(r[u], a.rows - 1)];
			p[u] = in ? a.tables[(int64_t)r[u] * a.table_ld + i] : 0;
			r[u] = in ? r[u] : -1;
		}
#pragma unroll
		for (int u = 0; u < 4; ++u) {
			if (r[u] < 0) continue;
			if (p[u] < 0 || p[u] >= a.pages) atomicMin(&s_bad, r[u]);
			else atomicOr(&live[p[u] >> 5], 1u << (p[u] & 31));
		}
	}
	__syncthreads();
	if (s_bad < a.rows) {
		if (tid == 0) {
			a.result[0] = SSLM_INVALID_ARGUMENT;
			a.result[1] = a.result[2] = 0;
			a.result[3] = s_bad;
			w.state[0] = 0;
		}
		return;
	}
	const int per = (words + kPlanBlock - 1) / kPlanBlock, w0 = tid * per, w1 = min(words, w0 + per);
	auto valid = [&](int i) { return a.pages - 32 * i >= 32 ? ~0u : (1u << (a.pages - 32 * i)) - 1; };
	int at;
	int64_t both = 0, all;  // movable pages above 2^32, those that nobody holds below
	for (int i = w0; i < w1; ++i) both += (int64_t)__popc(live[i] & ~held[i]) << 32 | __popc(~held[i] & valid(i));
	at = (int)block_before<int64_t>(both, &all, s_scan);
	const int movable = (int)(all >> 32);
	for (int i = w0; i < w1; ++i) {  // the boundary: one past the last of the first `movable` pages that nobody holds
		const uint32_t b = ~held[i] & valid(i);
		const int n = __popc(b);
		if (at < movable && at + n >= movable) {
			uint32_t x = b;
			for (int k = movable - at; k > 1; --k) x &= x - 1;
			s_edge = 32 * i + __builtin_ctz(x) + 1;
		}
		at += n;
	}
	if (tid == 0 && movable == 0) s_edge = 0;
	__syncthreads();
	const int edge = s_edge;
	auto below = [&](int i) { return 32 * i + 32 <= edge ? ~0u : (32 * i >= edge ? 0u : (1u << (edge - 32 * i)) - 1); };
	auto holes = [&](int i) { return ~live[i] & ~held[i] & below(i) & valid(i); };
	auto movers = [&](int i) { return live[i] & ~held[i] & ~below(i); };
	both = 0;
	for (int i = w0; i < w1; ++i) both += (int64_t)__popc(movers(i)) << 32 | __popc(holes(i));
	both = block_before<int64_t>(both, &all, s_scan);
	const int n2 = (int)(all >> 32);  // as many as there are holes
	at = (int)both;
	for (int i = w0; i < w1; ++i)
		for (uint32_t b = holes(i); b; b &= b - 1) w.free[at++] = 32 * i + __builtin_ctz(b);
	at = (int)(both >> 32);
	for (int i = w0; i < w1; ++i) {
		rank[i] = at;
		for (uint32_t b = movers(i); b; b &= b - 1) w.from[at++] = 32 * i + __builtin_ctz(b);
	}
	__syncthreads();  // the block's own writes of w.free are seen past it
	int top = 0;
	for (int p = tid; p < a.pages; p += kPlanBlock) {
		const int i = p >> 5;
		const uint32_t bit = 1u << (p & 31);
		int to = -1;
		if (movers(i) & bit) to = w.free[rank[i] + __popc(movers(i) & (bit - 1))];
		else if (live[i] & bit) to = p;
		a.map[p] = to;
		if (to >= 0) top = max(top, to + 1);
		if (held[i] & bit) top = max(top, p + 1);
	}
	for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
	if ((tid & 63) == 0) atomicMax(&s_top, top);
	__syncthreads();
	if (tid == 0) {
		a.result[0] = SSLM_OK;
		a.result[1] = s_top;
		a.result[2] = n2;
		a.result[3] = -1;
		w.state[0] = 1;
		w.state[1] = n2;
	}
}

__global__ __launch_bounds__(256) void k_compact_apply(PageCompactArgs a, PlanWork w) {
	if (!w.state[0]) return;
	const int64_t cells = (int64_t)a.rows * a.table_ld;
	for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < cells; c += (int64_t)gridDim.x * 256) {
		const int r = (int)(c / a.table_ld), i = (int)(c - (int64_t)r * a.table_ld);
		const int p = i < pages_for(a.lengths[r], a.lp) ? a.map[a.tables[c]] : -1;
		a.new_tables[c] = p;
	}
	copy_pages(a.pool, a.page_bytes, w.state[1], [&](int c, int* from, int* to) {
		*from = w.from[c];
		*to = w.free[c];
	});
}

// ------------------------------------------------------------------------------------------
// new tokens land in pages
// ------------------------------------------------------------------------------------------

// A row's tokens, as far as the tables and lengths admit them.
struct CacheRow {
	int64_t start;
	int t0, n;
	bool ok;
};
__device__ __forceinline__ CacheRow cache_row(const int32_t* row_tokens, const int64_t* row_start, int r, int tokens, int max_new, int64_t cap) {
	CacheRow c;
	c.t0 = row_tokens[r];
	const int t1 = row_tokens[r + 1];
	c.start = row_start[r];
	c.n = t1 - c.t0;
	c.ok = c.t0 >= 0 && t1 >= c.t0 && t1 <= tokens;
	if (!c.ok) c.n = 0;
	c.ok = c.ok && c.n <= max_new && c.start >= 0 && c.start <= cap - c.n;
	return c;
}

// A block per row: whether its tokens can land, 2.5 us beside the span's 16: the span's blocks would each have to look at every token.
__global__ __launch_bounds__(256) void k_store_check(CacheStoreArgs a) {
	__shared__ int s_st;
	const int r = blockIdx.x;
	int64_t cap = (int64_t)a.pg.table_ld << a.pg.lp;
	if (a.rope_dim) cap = i64min(cap, a.rope_rows);
	const CacheRow c = cache_row(a.row_tokens, a.row_start, r, a.tokens, a.max_new, cap);
	if (threadIdx.x == 0) s_st = c.ok ? 0 : 2;
	__syncthreads();
	if (c.ok && c.n > 0) {
		int st = 0;
		const int p0 = (int)(c.start >> a.pg.lp), p1 = (int)((c.start + c.n - 1) >> a.pg.lp);
		for (int i = p0 + (int)threadIdx.x; i <= p1; i += 256) {
			const int p = a.pg.tables[(int64_t)r * a.pg.table_ld + i];
			if (p < 0 || p >= a.pg.pages) st = 2;
		}
		for (int i = threadIdx.x; i < c.n; i += 256)
			if (!fits_i32(a.k_scale[c.t0 + i].m) || !fits_i32(a.v_scale[c.t0 + i].m)) st = max(st, 1);
		if (st) atomicMax(&s_st, st);
	}
	__syncthreads();
	if (threadIdx.x == 0) {
		a.clamped[r] = 0;
		a.status[r] = s_st == 2 ? kPositionOverCap : (s_st == 1 ? kCarriedScaleMantissaOutOfDomain : kOk);
	}
}

struct __attribute__((packed)) unaligned8 {
	uint64_t v;
};

// Eight dims of a head that turn or stay together, group g of D / 8: with halves, dims 4 g .. + 3 and the ones
// rope_dim / 2 further on; else 8 g .. + 7.  Element i of a pair is x[2 i], x[2 i + 1].
struct Octet {
	int32_t x[8];
};
__device__ __forceinline__ bool octet_split(const CacheStoreArgs& a, int g) { return a.halves && 8 * g < a.rope_dim; }
__device__ __forceinline__ Octet octet_load(const CacheStoreArgs& a, const int8_t* head, int g) {
	Octet o;
	uint64_t w;
	if (octet_split(a, g)) {
		const uint32_t lo = (uint32_t)((const unaligned4*)(head + 4 * g))->v, hi = (uint32_t)((const unaligned4*)(head + a.rope_dim / 2 + 4 * g))->v;
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			o.x[2 * i] = (int8_t)(lo >> 8 * i);
			o.x[2 * i + 1] = (int8_t)(hi >> 8 * i);
		}
		return o;
	}
	w = ((const unaligned8*)(head + 8 * g))->v;
#pragma unroll
	for (int i = 0; i < 8; ++i) o.x[i] = (int8_t)(w >> 8 * i);
	return o;
}
__device__ __forceinline__ void octet_store(const CacheStoreArgs& a, int8_t* head, int g, const Octet& o) {
	if (octet_split(a, g)) {
		uint32_t lo = 0, hi = 0;
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			lo |= (uint32_t)(uint8_t)o.x[2 * i] << 8 * i;
			hi |= (uint32_t)(uint8_t)o.x[2 * i + 1] << 8 * i;
		}
		((unaligned4*)(head + 4 * g))->v = (int32_t)lo;
		((unaligned4*)(head + a.rope_dim / 2 + 4 * g))->v = (int32_t)hi;
		return;
	}
	uint64_t w = 0;
#pragma unroll
	for (int i = 0; i < 8; ++i) w |= (uint64_t)(uint8_t)o.x[i] << 8 * i;
	((unaligned8*)(head + 8 * g))->v = w;
}
// The angles of four pairs at `pos`, and the pairs turned by them (rope_pair), clamped to +-top; returns how many values were.
// In doubles, the tables' entries taken as 32 bits: a value of 16 bits times an entry's 31, and the sum of two of these, are exact at the scale 2^-30, and so is half a
// unit added away from zero before the conversion truncates.  Five instructions a value, the 64-bit form takes some thirty: 512 tokens of
// 28 + 2 x 4 heads for each of four rows 18.4 -> 16.2 us.
struct Turn {
	double c[4], s[4];
};
__device__ __forceinline__ Turn turn_at(const CacheStoreArgs& a, int64_t pos, int g) {
	Turn t;
	const int64_t at = pos * (a.rope_dim / 2) + 4 * g;
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		t.c[i] = (double)(int32_t)a.rope_cos[at + i] * 0x1p-30;
		t.s[i] = (double)(int32_t)a.rope_sin[at + i] * 0x1p-30;
	}
	return t;
}
__device__ __forceinline__ int octet_turn(Octet& o, const Turn& t, int32_t top) {
	int n = 0;
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		const double x = (double)o.x[2 * i], y = (double)o.x[2 * i + 1];
		const double u[2] = {fma(-y, t.s[i], x * t.c[i]), fma(y, t.c[i], x * t.s[i])};
#pragma unroll
		for (int j = 0; j < 2; ++j) {
			const int32_t v = (int32_t)(u[j] + copysign(0.5, u[j]));
			const int32_t w = max(-top, min(v, top));
			n += v != w;
			o.x[2 * i + j] = w;
		}
	}
	return n;
}

// x / 2^e in units, ties away from zero, at exponent `at` and then at each of `levels` past it: a page's codes are
// rounded once more whenever it grows.
__device__ __forceinline__ int32_t grown_code(int32_t x, int at, uint32_t levels) {
	x = rdbpot32(x, at);
	for (uint32_t m = levels & ~((2u << at) - 1); m; m &= m - 1) {
		const int to = __builtin_ctz(m);
		x = rdbpot32(x, to - at);
		at = to;
	}
	return x;
}
// the least exponent that keeps a code of magnitude m within 127
__device__ __forceinline__ int exponent_for(int32_t m) {
	int e = 0;
	while (rdbpot32(m, e) > 127) ++e;
	return e;
}

// A code landed in units and clamped; whether it had to be.  residual_land's infinity has no sign.
__device__ __forceinline__ int land_units(int32_t& x, int64_t m, int64_t r_t, int64_t k, double f) {
	const double y = fabs(residual_land(x, m, r_t, k, f));
	const int32_t u = (int32_t)fmin(y, (double)kMaxUnits);
	x = (x < 0) != (m < 0) ? -u : u;
	return y > (double)kMaxUnits;
}

// octet g of a token's query head, turned
__device__ __forceinline__ void q_octet(const CacheStoreArgs& a, int t, int h, int g, bool turns, const Turn& turn) {
	Octet o = octet_load(a, a.q + (int64_t)t * a.q_ld + h * a.pg.D, g);
	if (turns) octet_turn(o, turn, 127);
	octet_store(a, a.q_out + ((int64_t)t * a.NH + h) * a.pg.D, g, o);
}
// octet g of token t's K or V in units, turned; the values clamped
__device__ __forceinline__ int land_octet(const CacheStoreArgs& a, bool isv, int kvh, int t, int64_t pos, int g, const Scale& sc, int64_t rt, int64_t et, Octet* out) {
	Octet o = octet_load(a, (isv ? a.v + t * a.v_ld : a.k + t * a.k_ld) + kvh * a.pg.D, g);
	const int64_t k = composed_exponent(sc.e, et);
	const double f = landing_scale(sc.m, rt, k).f;
	int over = 0;
#pragma unroll
	for (int j = 0; j < 8; ++j) over += land_units(o.x[j], sc.m, rt, k, f);
	if (!isv && 8 * g < a.rope_dim) over += octet_turn(o, turn_at(a, pos, g), kMaxUnits);
	*out = o;
	return over;
}
// a KV head's largest magnitude over the lanes of its octets
template <int GP>
__device__ __forceinline__ int32_t octets_max(const Octet& o) {
	int32_t mx = 0;
#pragma unroll
	for (int j = 0; j < 8; ++j) mx = max(mx, abs(o.x[j]));
	for (int d = 1; d < GP; d *= 2) mx = max(mx, __shfl_xor(mx, d, 64));
	return mx;
}
// eight old codes of a page that grows from exponent `init` through `levels`
__device__ __forceinline__ void regrow(int8_t* at, int init, uint32_t levels) {
	const uint64_t w = ((const unaligned8*)at)->v;
	uint64_t out = 0;
#pragma unroll
	for (int j = 0; j < 8; ++j) out |= (uint64_t)(uint8_t)grown_code((int8_t)(w >> 8 * j), 0, levels >> init & ~1u) << 8 * j;
	((unaligned8*)at)->v = out;
}

// K or V of one KV head (z) in one page (x) of one row (y): the page's tokens land in LDS, their exponents run up the
// page, then the codes are written; the waves of blocks past the last page take q's tokens, one each.
// Bound by its instructions (a landing and a rotation are some 40 of doubles to a code) and, as one block takes a page's tokens, by that
// block's length: 4 rows of 512 tokens, 28 + 2 x 4 heads of 128, 16 us, without queries 14.5; their 16.5 MB are 3.5.
constexpr int kStoreBlock = 512;
template <int D>
__global__ __launch_bounds__(kStoreBlock) void k_store_span(CacheStoreArgs a, int pages) {
	extern __shared__ __attribute__((aligned(16))) int16_t s_x[];  // [page's tokens][D], groups of eight in octet order
	__shared__ uint8_t s_need[256];
	__shared__ uint32_t s_levels;
	__shared__ int s_init, s_clamped;
	constexpr int GP = D / 8;
	const int r = blockIdx.y, z = blockIdx.z, tid = threadIdx.x;
	if (a.status[r] != kOk) return;
	const int t0 = a.row_tokens[r], n = a.row_tokens[r + 1] - t0;
	const int64_t start = a.row_start[r];
	if ((int)blockIdx.x >= pages) {
		const int i = (((int)blockIdx.x - pages) * (int)gridDim.z + z) * (kStoreBlock / 64) + (tid >> 6);
		if (i >= n) return;
		const int g = tid % GP;
		const bool turns = 8 * g < a.rope_dim;
		Turn t;
		if (turns) t = turn_at(a, start + i, g);
		for (int h = (tid & 63) / GP; h < a.NH; h += 64 / GP) q_octet(a, t0 + i, h, g, turns, t);
		return;
	}
	const int P = 1 << a.pg.lp;
	const int64_t page0 = start >> a.pg.lp, first = (page0 + blockIdx.x) << a.pg.lp;
	const int i0 = (int)(first > start ? first - start : 0), i1 = (int)i64min(n, first + P - start);  // the row's tokens in the page
	if (i0 >= i1) return;
	const int slot0 = (int)(start + i0 - first), cnt = i1 - i0, kvh = z >> 1;
	const bool isv = z & 1;
	int8_t* page = a.pg.pool + a.pg.tables[(int64_t)r * a.pg.table_ld + page0 + blockIdx.x] * a.pg.page_bytes;
	int8_t* head = page + (isv ? a.pg.v_off : a.pg.k_off) + ((int64_t)kvh << a.pg.lp) * D;
	uint8_t* exp = (uint8_t*)page + a.pg.e_off + (isv ? a.pg.NKV : 0) + kvh;
	if (tid == 0) {
		s_levels = 0;
		s_clamped = 0;
		s_init = slot0 ? min((int)*exp, kMaxShift) : 0;
	}
	__syncthreads();
	const int64_t rt = isv ? a.r_t_v[kvh] : a.r_t_k[kvh], et = isv ? a.e_t_v[kvh] : a.e_t_k[kvh];
	int clamped = 0;
	for (int u = tid; u < (cnt * GP + kStoreBlock - 1) / kStoreBlock * kStoreBlock; u += kStoreBlock) {
		const bool in = u < cnt * GP;
		const int i = in ? u / GP : 0, g = u % GP, t = t0 + i0 + i;
		Octet o;
		const int over = land_octet(a, isv, kvh, t, start + i0 + i, g, isv ? a.v_scale[t] : a.k_scale[t], rt, et, &o);
		const int32_t mx = octets_max<GP>(o);
		union {
			int16_t h[8];
			v4i v;
		} pk;
#pragma unroll
		for (int j = 0; j < 8; ++j) pk.h[j] = (int16_t)o.x[j];
		if (in) {
			*(v4i*)(s_x + (int64_t)u * 8) = pk.v;
			if (g == 0) s_need[i] = (uint8_t)exponent_for(mx);
			clamped += over;
		}
	}
	clamped = wave_sum32(clamped);
	if ((tid & 63) == 0 && clamped) atomicAdd(&s_clamped, clamped);
	__syncthreads();
	if (tid < 64) {  // the exponents the page has after each of its tokens
		int e[4], m = 0;
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			if (4 * tid + j < cnt) m = max(m, (int)s_need[4 * tid + j]);
			e[j] = m;
		}
		for (int d = 1; d < 64; d *= 2) {
			const int y = __shfl_up(m, d, 64);
			m = tid >= d ? max(m, y) : m;
		}
		int before = __shfl_up(m, 1, 64);
		before = max(tid ? before : 0, s_init);
		uint32_t levels = 0;
#pragma unroll
		for (int j = 0; j < 4; ++j)
			if (4 * tid + j < cnt) {
				e[j] = max(e[j], before);
				s_need[4 * tid + j] = (uint8_t)e[j];
				levels |= 1u << e[j];
			}
		if (levels) atomicOr(&s_levels, levels);
	}
	__syncthreads();
	const uint32_t levels = s_levels;
	for (int u = tid; u < cnt * GP; u += kStoreBlock) {
		const int i = u / GP, g = u % GP;
		Octet o;
		union {
			int16_t h[8];
			v4i v;
		} pk;
		pk.v = *(const v4i*)(s_x + (int64_t)u * 8);
#pragma unroll
		for (int j = 0; j < 8; ++j) o.x[j] = grown_code(pk.h[j], s_need[i], levels);
		octet_store(a, head + (int64_t)(slot0 + i) * D, g, o);
	}
	const int init = s_init;
	if (slot0 && levels >> (init + 1)) {
		for (int u = tid; u < slot0 * GP; u += kStoreBlock) regrow(head + (int64_t)u * 8, init, levels);
	}
	if (tid == 0) {
		*exp = (uint8_t)(31 - __builtin_clz(levels));
		if (s_clamped) atomicAdd(&a.clamped[r], s_clamped);
	}
}

// Single tokens in one launch, a block per row: K's and V's octets, then q's.  The lanes of a head's octets find its
// exponent; a page that grows is rounded by the whole block once all heads are known.  Its chain of loads bounds it: 8 rows 5.5 us, with
// the span's two launches 9.7.
template <int D>
__global__ __launch_bounds__(kStoreBlock) void k_store_token(CacheStoreArgs a) {
	__shared__ uint16_t s_grow[2 * 256];  // of each KV head's K and V: the exponents before and after
	__shared__ int s_clamped;
	constexpr int GP = D / 8;
	const int r = blockIdx.x, tid = threadIdx.x, kv = 2 * a.pg.NKV * GP, total = kv + (a.q ? a.NH * GP : 0);
	int64_t cap = (int64_t)a.pg.table_ld << a.pg.lp;
	if (a.rope_dim) cap = i64min(cap, a.rope_rows);
	const CacheRow c = cache_row(a.row_tokens, a.row_start, r, a.tokens, a.max_new, cap);
	int st = c.ok ? kOk : kPositionOverCap;
	int32_t entry = 0;
	if (c.ok && c.n > 0) {
		entry = a.pg.tables[(int64_t)r * a.pg.table_ld + (c.start >> a.pg.lp)];
		const bool scales = fits_i32(a.k_scale[c.t0].m) && fits_i32(a.v_scale[c.t0].m);
		st = entry < 0 || entry >= a.pg.pages ? kPositionOverCap : (scales ? kOk : kCarriedScaleMantissaOutOfDomain);
	}
	if (tid == 0) {
		s_clamped = 0;
		a.status[r] = st;
	}
	__syncthreads();
	if (st != kOk || c.n == 0) {
		if (tid == 0) a.clamped[r] = 0;
		return;
	}
	const int slot = (int)(c.start & ((1 << a.pg.lp) - 1)), g = tid % GP;
	int8_t* page = a.pg.pool + entry * a.pg.page_bytes;
	const bool turns = 8 * g < a.rope_dim;
	Turn turn;
	if (turns) turn = turn_at(a, c.start, g);
	auto head = [&](int z) { return page + (z & 1 ? a.pg.v_off : a.pg.k_off) + ((int64_t)(z >> 1) << a.pg.lp) * D; };
	int clamped = 0;
	for (int u0 = tid - tid % 64; u0 < total; u0 += kStoreBlock) {  // whole waves
		const int u = u0 + tid % 64;
		if (u0 < kv) {
			const bool in = u < kv;
			const int z = in ? u / GP : 0, kvh = z >> 1;
			const bool isv = z & 1;
			Octet o;
			const int over = land_octet(a, isv, kvh, c.t0, c.start, g, isv ? a.v_scale[c.t0] : a.k_scale[c.t0], isv ? a.r_t_v[kvh] : a.r_t_k[kvh],
			                            isv ? a.e_t_v[kvh] : a.e_t_k[kvh], &o);
			const int need = exponent_for(octets_max<GP>(o));
			if (in) {
				uint8_t* exp = (uint8_t*)page + a.pg.e_off + (isv ? a.pg.NKV : 0) + kvh;
				const int was = slot ? min((int)*exp, kMaxShift) : 0, now = max(was, need);
				clamped += over;
				if (g == 0) {
					*exp = (uint8_t)now;
					s_grow[z] = (uint16_t)(was | now << 8);
				}
#pragma unroll
				for (int j = 0; j < 8; ++j) o.x[j] = rdbpot32(o.x[j], now);
				octet_store(a, head(z) + (int64_t)slot * D, g, o);
			}
		}
		if (u >= kv && u < total) q_octet(a, c.t0, (u - kv) / GP, g, turns, turn);
	}
	if (clamped) atomicAdd(&s_clamped, clamped);
	__syncthreads();
	if (tid == 0) a.clamped[r] = s_clamped;
	for (int z = 0; slot && z < 2 * a.pg.NKV; ++z) {
		const int was = s_grow[z] & 255, now = s_grow[z] >> 8;
		if (now == was) continue;
		for (int u = tid; u < slot * GP; u += kStoreBlock) regrow(head(z) + (int64_t)u * 8, was, 1u << now);
	}
}

// ------------------------------------------------------------------------------------------
// attention over pages
// ------------------------------------------------------------------------------------------

// The layout of one call's launches.  The unit of work is a wave with a tile of 16 query rows (token, head) of one KV
// head and a range of positions, a "plane" of sp.  The softmax's maximum and sum run over the whole row and each
// probability is rounded by itself, so nothing is rescaled: maxima, sums and P V are launches of their own, and the
// planes' integers join exactly in any order.
// Single tokens: a tile is one token's heads, four waves take the positions in turn, scores are kept for the later
// launches (4 G bytes a position beside the 2 D of its K and V).  Chunks: four neighbouring tiles of a row share each step of 64 positions that
// their block stages, and the scores are computed again, 8 MFMAs a step at D = 128.
struct CaPlan {
	int whole;       // single tokens' rows in one launch and the join (k_cr_row): cr_form's answer
	int ht;          // single tokens: tiles of a token's heads
	int groups;      // chunks: blocks of 64 query rows, at least those of every row together
	int sp, planes;  // positions of a plane (a multiple of 256), planes of the widest row
	int ps, parts;   // positions of one block of sums, blocks of the widest row
	int64_t wpad;    // kept scores of a (token, head)
};

struct CaWork {
	SaConst* cst;     // [tokens, NKV]
	int32_t* pmax;    // [planes][tokens NH]
	int32_t* top;     // [tokens NH] single tokens: the row's maximum
	int64_t* psum;    // [parts or planes][tokens NH]; negative: an i-exp value was refused
	int32_t* part;    // [planes][tokens][NH D]
	int32_t* hst;     // [tokens NH] refusals of the softmax
	int32_t* scores;  // [tokens NH][wpad] single tokens
};

constexpr int kCaWaves = 4;

__device__ __forceinline__ CacheRow attn_row(const CacheAttnArgs& a, int r) {
	return cache_row(a.row_tokens, a.row_start, r, a.tokens, a.max_new, i64min((int64_t)a.pg.table_ld << a.pg.lp, a.max_width));
}

// A wave's next 64 pages of a row, one to a lane, from position p0's on (lanes past position `last`'s page repeat it), with the
// KV head's exponents; false for the whole wave when one is not a page.  Positions are below 2^24 from here on.
struct LanePages {
	int32_t page, ke, ve, first;
};
__device__ __forceinline__ bool lane_pages(const Pages& g, int r, int kvh, int p0, int last, LanePages* o) {
	o->first = p0 >> g.lp;
	o->page = g.tables[(int64_t)r * g.table_ld + o->first + min((int)threadIdx.x & 63, (last >> g.lp) - o->first)];
	if (__any(o->page < 0 || o->page >= g.pages)) return false;
	const uint8_t* e = (const uint8_t*)g.pool + o->page * g.page_bytes + g.e_off;
	o->ke = min((int)e[kvh], kMaxShift);
	o->ve = min((int)e[g.NKV + kvh], kMaxShift);
	return true;
}
// where the 64 pages from position p's on end
__device__ __forceinline__ int pages_end(const Pages& g, int p) { return ((p >> g.lp) + 64) << g.lp; }
// whether every page of the row's first `width` positions is one (by all lanes of a wave)
__device__ __forceinline__ bool row_pages_ok(const Pages& g, int r, int64_t width) {
	bool bad = false;
	for (int64_t i = threadIdx.x & 63; i < pages_for(width, g.lp); i += 64) {
		const int p = g.tables[(int64_t)r * g.table_ld + i];
		bad |= p < 0 || p >= g.pages;
	}
	return !__any(bad);
}

// K or V of the page under 16 positions from p on, as a buffer: a load is then this in scalars and 32 bits of a lane's own.  Past
// `last` the buffer is empty: its loads give zeros and move nothing, and the loads in flight are the same number on every path.
// `off`: the head's K or V in its page.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rows(const Pages& g, const LanePages& lp, int p, int last, int64_t off) {
	const int page = __builtin_amdgcn_readlane(lp.page, (min(p, last) >> g.lp) - lp.first);
	return __builtin_amdgcn_make_buffer_rsrc(g.pool + (page * g.page_bytes + off), 0, p <= last ? g.D << g.lp : 0, 0x00020000);
}
__device__ __forceinline__ v4i buffer16(__amdgpu_buffer_rsrc_t b, uint32_t at) {
	return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0));
}
// Rows of 64 positions from p on (a multiple of 64) as a wave loads them: 16 positions never leave a page.
template <int D>
__device__ __forceinline__ void load_rows(SaRows<D>& x, const Pages& g, const LanePages& lp, int p, int last, int64_t off) {
	constexpr int PER = D / 16, R = 64 / PER;  // rows of one load
	const int lane = threadIdx.x & 63, mask = (1 << g.lp) - 1;
	__amdgpu_buffer_rsrc_t b[4];
	b[0] = page_rows(g, lp, p, last, off);
#pragma unroll
	for (int t = 1; t < 4; ++t) b[t] = page_rows(g, lp, p + 16 * t, last, off);
	x.load_at([&](int u) {
		const int row = u * R + lane / PER;
		const uint32_t at = (uint32_t)(((p + row) & mask) * D + lane % PER * 16);
		if constexpr (R > 16) return buffer16(b[2 * u], lane / PER < 16 ? at : ~0u) | buffer16(b[2 * u + 1], lane / PER < 16 ? ~0u : at);
		else return buffer16(b[u * R / 16], at);
	});
	__builtin_amdgcn_sched_barrier(0);  // loads stay in this order: a wait for the older rows then leaves the newer in flight
}
// the exponents of 16 positions from p
__device__ __forceinline__ int page_exp(const Pages& g, const LanePages& lp, int32_t e, int p, int last) {
	return __builtin_amdgcn_readlane(e, (min(p, last) >> g.lp) - lp.first);
}

// Whether a row's i-exp values are the doubles' (sa_exp): 0 <= q_b and q_ln2 <= 2 q_b + 1, then no value leaves [0, ceil],
// ceil <= 2^47.  A unit of score is small here (a page's exponents are above it), so sums pass 2^53 often: a lane adds 16 values in
// a double, below 2^51, and those to an integer.
__device__ __forceinline__ bool ca_fast(const SaConst& c) { return c.q_b >= 0 && c.q_ln2 >= 1 && c.ceil >= 1 && c.q_ln2 <= 2 * c.q_b + 1; }

// sa_prob for sums d of up to 2^62.  From 2^36 on: q, the estimate from below, is the quotient or one less; with
// d = dh + dl, dh a multiple of 2^20, e - (q + 1) dh 2^-15 is an integer below 2^49 and (q + 1) dl 2^-15 has 36 bits, both exact.
struct CaProb {
	double c1, c2, dh, dl;
};
__device__ __forceinline__ CaProb ca_prob_of(int64_t d, bool small) {
	const int64_t low = d & ((1 << 20) - 1);
	CaProb p;
	p.dh = (double)(d - low) * 0x1p-15;
	p.dl = (double)low * 0x1p-15;
	p.c1 = small ? 32768.0 / (double)d : (1.0 - 0x1p-50) * 32768.0 / (double)d;
	p.c2 = 0.5 / (double)d;
	return p;
}
template <bool SMALL>
__device__ __forceinline__ int32_t ca_prob(const CaProb& p, double e) {
	if constexpr (SMALL) return (int32_t)fma(e, p.c1, p.c2);
	const double q = floor(e * p.c1), n = q + 1.0;
	return (int32_t)q + (fma(-n, p.dh, e) >= n * p.dl ? 1 : 0);
}

// Which bits some live lane of the block has set: what its waves branch on alike.
__device__ __forceinline__ int block_vote(int bits, int* s) {
	const int all = (__any(bits & 1) ? 1 : 0) | (__any(bits & 2) ? 2 : 0);
	if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = all;
	__syncthreads();
	return __builtin_amdgcn_readfirstlane(s[0] | s[1] | s[2] | s[3]);
}

// A single token's block: a plane of a (row, KV head, tile of heads).  A step is 256 positions, 64 to a wave.
constexpr int kCdStep = 64 * kCaWaves;
struct CdJob {
	int r, t, kvh, tile, plane, h0, heads;  // h0: the tile's first head
	int width, p0, p1;
	CacheRow row;
};
__device__ __forceinline__ bool cd_job(const CacheAttnArgs& a, const CaPlan& pl, CdJob* j) {
	const int w = blockIdx.x, G = a.NH / a.pg.NKV;
	j->plane = w % pl.planes;
	j->tile = w / pl.planes % pl.ht;
	j->kvh = w / pl.planes / pl.ht % a.pg.NKV;
	j->r = w / pl.planes / pl.ht / a.pg.NKV;
	j->row = attn_row(a, j->r);
	if (!j->row.ok || j->row.n < 1) return false;
	j->t = j->row.t0;
	j->h0 = j->kvh * G + j->tile * 16;
	j->heads = min(16, G - j->tile * 16);
	j->width = (int)j->row.start + 1;
	j->p0 = j->plane * pl.sp;
	j->p1 = min(j->width, j->p0 + pl.sp);
	return j->p0 < j->p1;
}

// The scores of a plane, kept, and their maxima: written once and read twice they cost less than two more products with K.  8 rows of
// 28 heads / 4 KV x 128 by 16000 positions: 18.8 us, 66 MB of K and 14 of scores at 4.2 TB/s; then k_cd_sum 7.7, k_cd_pv 21.6 and the join 7.9.
// 2 rows of 12 / 2 by 8000, a chain of four launches: 5.9 + 4.2 + 8.6 + 4.3.  The first wave of a row's first plane also settles its constants.
template <int D>
__global__ __launch_bounds__(64 * kCaWaves) void k_cd_scores(CacheAttnArgs a, CaPlan pl, CaWork w) {
	constexpr int NC = (D + 63) / 64;
	__shared__ __attribute__((aligned(16))) int8_t s_k[kCaWaves][32 * D];
	__shared__ int32_t s_m[kCaWaves][16];
	const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	CdJob j;
	if (!cd_job(a, pl, &j)) return;
	int8_t* lds = s_k[wave];
	const bool mine = ri < j.heads;
	const int h = j.h0 + (mine ? ri : 0);
	v4i q[NC];
#pragma unroll
	for (int c = 0; c < NC; ++c) q[c] = mine && c * 64 + g * 16 < D ? load16(a.q + ((size_t)j.t * a.NH + h) * D + c * 64 + g * 16) : v4i{0, 0, 0, 0};
	// dead lanes and positions past the plane store outside the descriptor, which drops them: no branch between the loads
	const auto out = __builtin_amdgcn_make_buffer_rsrc(w.scores + ((size_t)j.t * a.NH + j.h0) * pl.wpad, 0, (int)(j.heads * pl.wpad * 4), 0x00020000);
	const uint32_t mine_at = mine ? (uint32_t)((ri * pl.wpad + 4 * g) * 4) : ~0u;
	const int64_t off = a.pg.k_off + ((int64_t)j.kvh << a.pg.lp) * D;
	int32_t m = INT32_MIN;
	for (int s0 = j.p0; s0 < j.p1; s0 = pages_end(a.pg, s0)) {
		const int s1 = min(j.p1, pages_end(a.pg, s0)), last = s1 - 1;
		LanePages lp;
		if (!lane_pages(a.pg, j.r, j.kvh, s0, last, &lp)) break;
		SaRows<D> k[2];
#pragma unroll
		for (int b = 0; b < 2; ++b) load_rows(k[b], a.pg, lp, s0 + 64 * wave + b * kCdStep, last, off);
		for (int p0 = s0 + 64 * wave; p0 < s1; p0 += 2 * kCdStep) {
#pragma unroll
			for (int b = 0; b < 2; ++b) {
				const int p = p0 + b * kCdStep;
				v4i s[4] = {};
				k[b].scores(lds, q, s);
				load_rows(k[b], a.pg, lp, p + 2 * kCdStep, last, off);
				const int left = s1 - p - 4 * g;
				const uint32_t at = p < s1 ? mine_at : ~0u;
#pragma unroll
				for (int t = 0; t < 4; ++t) {
					const int e = page_exp(a.pg, lp, lp.ke, p + 16 * t, last);
#pragma unroll
					for (int v = 0; v < 4; ++v) {
						s[t][v] <<= e;
						m = max(m, t * 16 + v < left ? s[t][v] : INT32_MIN);
					}
					__builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, s[t]), out, at, (p + 16 * t) * 4, 0);
				}
			}
		}
	}
	if (j.plane == 0 && j.tile == 0 && wave == 0) {
		SaConst c{0, 0, 0, 0, kPositionOverCap, 0};
		if (row_pages_ok(a.pg, j.r, j.width)) {
			const RowConst rc = row_const(RowScales{a.q_scale[j.t], a.khead_m[j.kvh], a.khead_e[j.kvh]}, a.ln2_q, a.b_q, a.ca_q, j.width);
			c = SaConst{rc.q_ln2, rc.q_b, rc.q_c, rc.ceil, rc.st, 0};
		}
		if (lane == 0) w.cst[(size_t)j.t * a.pg.NKV + j.kvh] = c;
	}
	m = max(m, __shfl_xor(m, 16, 64));
	m = max(m, __shfl_xor(m, 32, 64));
	if (g == 0) s_m[wave][ri] = m;
	__syncthreads();
	if (threadIdx.x < j.heads)
		w.pmax[((size_t)j.plane * a.tokens + j.t) * a.NH + j.h0 + threadIdx.x] = max(max(s_m[0][threadIdx.x], s_m[1][threadIdx.x]), max(s_m[2][threadIdx.x], s_m[3][threadIdx.x]));
}

// The sum of one (token, head) over a part of its positions, from the kept scores: all of a thread's are loaded ahead of the
// constants and maxima that they wait for.
constexpr int kCdSumLoads = 4, kCdSum = 1024 * kCdSumLoads;
__global__ __launch_bounds__(256) void k_cd_sum(CacheAttnArgs a, CaPlan pl, CaWork w) {
	__shared__ int32_t s_m[4];
	__shared__ int64_t s_s[4];
	const int part = blockIdx.x, h = blockIdx.y, r = blockIdx.z, tid = threadIdx.x, kvh = h / (a.NH / a.pg.NKV);
	const CacheRow row = attn_row(a, r);
	if (!row.ok || row.n < 1) return;
	const int t = row.t0;
	const int width = (int)row.start + 1, p0 = part * pl.ps, p1 = min(width, p0 + pl.ps);
	if (p0 >= p1) return;
	const int32_t* sc = w.scores + ((size_t)t * a.NH + h) * pl.wpad;
	v4i x[kCdSumLoads];
#pragma unroll
	for (int i = 0; i < kCdSumLoads; ++i) x[i] = *(const v4i*)(sc + min(p0 + 1024 * i + 4 * tid, (p1 - 1) & ~3));
	const SaConst c = w.cst[(size_t)t * a.pg.NKV + kvh];
	int32_t top = INT32_MIN;
	const int n = (width + pl.sp - 1) / pl.sp;
	for (int i = tid; i < n; i += 256) top = max(top, w.pmax[((size_t)i * a.tokens + t) * a.NH + h]);
	for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, 64));
	if ((tid & 63) == 0) s_m[tid >> 6] = top;
	__syncthreads();
	if (c.st != kOk) return;
	top = max(max(s_m[0], s_m[1]), max(s_m[2], s_m[3]));
	int64_t sum = 0;
	int bad = 0;
	if (ca_fast(c)) {
		const SaExp e = sa_exp_of(c, top);
		double acc = 0.0;  // 16 values
#pragma unroll
		for (int i = 0; i < kCdSumLoads; ++i) {
			const int p = p0 + 1024 * i + 4 * tid;
			if (p0 + 1024 * i >= p1) break;
#pragma unroll
			for (int k = 0; k < 4; ++k) {
				const double y = sa_exp(e, x[i][k]);
				acc += p + k < p1 ? y : 0.0;
			}
		}
		sum = (int64_t)acc;
	} else {
		const double inv = 1.0 / (double)c.q_ln2;
#pragma unroll
		for (int i = 0; i < 4 * kCdSumLoads; ++i) {
			if (p0 + 1024 * (i >> 2) + 4 * tid + (i & 3) >= p1) continue;
			const int64_t y = iexp_fast_cold((int64_t)x[i >> 2][i & 3] - top, c.q_ln2, inv, c.q_b, c.q_c, c.ceil);
			bad |= y < 0;
			sum += y < 0 ? 0 : y;
		}
	}
	for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
	bad = __any(bad);
	if ((tid & 63) == 0) s_s[tid >> 6] = bad ? -1 : sum;
	__syncthreads();
	if (tid == 0) {
		sum = 0;
		for (int i = 0; i < 4; ++i) {
			bad |= s_s[i] < 0;
			sum += s_s[i];
		}
		w.psum[((size_t)part * a.tokens + t) * a.NH + h] = bad ? -1 : sum;
		if (part == 0) w.top[(size_t)t * a.NH + h] = top;
	}
}

// P V of a plane, a block of four waves: probabilities of 256 positions at a time, a wave to a head, go to LDS as three
// int8 operands (sa_pack3) in the order the MFMAs read them, then each wave multiplies 64 of the positions; the waves'
// contexts are joined at the end.  The next 256 positions' scores and V rows are in flight meanwhile.
template <int D, int R>
__global__ __launch_bounds__(64 * kCaWaves, D <= 128 ? 2 : 1) void k_cd_pv(CacheAttnArgs a, CaPlan pl, CaWork w) {
	constexpr int DT = D / 16;
	// [parity][operand][64 positions' bytes of 16 heads], V staged by each wave; the join reuses it: [wave][dt][lane]
	struct Step {
		uint32_t p[2][3][kCaWaves][256];
		int8_t v[kCaWaves][32 * D];
	};
	union Lds {
		Step s;
		v4i join[kCaWaves][DT][64];
	};
	__shared__ __attribute__((aligned(16))) Lds lds;
	__shared__ int s_vote[kCaWaves];
	const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	CdJob j;
	if (!cd_job(a, pl, &j)) return;
	const int64_t off = a.pg.v_off + ((int64_t)j.kvh << a.pg.lp) * D;
	const SaConst c = w.cst[(size_t)j.t * a.pg.NKV + j.kvh];
	const int parts = (j.width + pl.ps - 1) / pl.ps;
	// this wave's heads wave, wave + 4, ..: the maximum and the sum
	int32_t top[R];
	int64_t den[R];
	int refused = 0, form = 0;
#pragma unroll
	for (int i = 0; i < R; ++i) {
		const size_t th = (size_t)j.t * a.NH + j.h0 + min(wave + 4 * i, j.heads - 1);
		top[i] = w.top[th];
		int64_t sum = 0;
		bool bad = false;
		for (int k = 0; k < parts; ++k) {
			const int64_t x = w.psum[(size_t)k * a.tokens * a.NH + th];
			bad |= x < 0;
			sum += x;
		}
		refused |= bad ? 1 << i : 0;
		den[i] = !bad && sum > 1 ? sum : 1;
		form |= den[i] >= (int64_t)1 << 36 ? 2 : 0;
		if (c.st == kOk && j.plane == 0 && lane == 0 && wave + 4 * i < j.heads) w.hst[th] = bad ? kSoftmaxKernelRefusedAfterGateAccepted : kOk;
	}
	if (c.st != kOk) return;
	form = block_vote(form | !ca_fast(c), s_vote);
	v4i acc[DT][3];
#pragma unroll
	for (int d = 0; d < DT; ++d) acc[d][0] = acc[d][1] = acc[d][2] = v4i{0, 0, 0, 0};
	// value(i, score, in): the probability of a score of head wave + 4 i
	auto run = [&](auto&& value) {
		int b = 0;
		for (int s0 = j.p0; s0 < j.p1; s0 = pages_end(a.pg, s0)) {
			const int s1 = min(j.p1, pages_end(a.pg, s0)), last = s1 - 1;
			LanePages lp;
			if (!lane_pages(a.pg, j.r, j.kvh, s0, last, &lp)) return;  // alike for the block's waves
			SaRows<D> v;
			v4i s[R];
			auto scores = [&](int p) {
#pragma unroll
				for (int i = 0; i < R; ++i)
					s[i] = *(const v4i*)(w.scores + ((size_t)j.t * a.NH + j.h0 + min(wave + 4 * i, j.heads - 1)) * pl.wpad + p + 4 * lane);
			};
			scores(s0);
			load_rows(v, a.pg, lp, s0 + 64 * wave, last, off);
			for (int p = s0; p < s1; p += kCdStep) {
				const int left = s1 - p - 4 * lane;
				// lane 4 i + k of a head has positions 16 i + 4 k .. + 3: word i of the operand's lane (head, k)
				const int sh = __shfl(lp.ve, (min(p + 4 * lane, last) >> a.pg.lp) - lp.first, 64);
#pragma unroll
				for (int i = 0; i < R; ++i) {
					const int head = wave + 4 * i;
					if (head >= j.heads) break;
					int32_t pr[4];
#pragma unroll
					for (int k = 0; k < 4; ++k) {
						const int32_t y = value(i, s[i][k], k < left);
						pr[k] = k < left && !(refused >> i & 1) ? y << sh : 0;
					}
					uint32_t x[3];
					sa_pack3_word(pr[0], pr[1], pr[2], pr[3], x);
					const int at = head * 16 + (lane & 3) * 4 + (lane >> 2 & 3);
#pragma unroll
					for (int n = 0; n < 3; ++n) lds.s.p[b][n][lane >> 4][at] = x[n];
				}
				scores(p + kCdStep < s1 ? p + kCdStep : p);
				__syncthreads();
				v4i x[3];
#pragma unroll
				for (int n = 0; n < 3; ++n) x[n] = *(const v4i*)&lds.s.p[b][n][wave][ri * 16 + g * 4];
				v.multiply(lds.s.v[wave], x, acc);
				load_rows(v, a.pg, lp, p + kCdStep + 64 * wave, last, off);
				b ^= 1;
			}
		}
	};
	if (!(form & 1)) {
		SaExp e = sa_exp_of(c, 0);
		const int32_t add = e.add;
		CaProb pb[R];
#pragma unroll
		for (int i = 0; i < R; ++i) pb[i] = ca_prob_of(den[i], form == 0);
		auto exp = [&](int i, int32_t x) {
			e.add = add - top[i];
			return sa_exp(e, x);
		};
		if (form == 0) run([&](int i, int32_t x, bool) { return ca_prob<true>(pb[i], exp(i, x)); });
		else run([&](int i, int32_t x, bool) { return ca_prob<false>(pb[i], exp(i, x)); });
	} else {
		const double inv = 1.0 / (double)c.q_ln2;
		run([&](int i, int32_t x, bool in) {
			return in ? (int32_t)div_rcp_cold(iexp_fast_cold((int64_t)x - top[i], c.q_ln2, inv, c.q_b, c.q_c, c.ceil) << 15, den[i], 1.0 / (double)den[i], 32768) : 0;
		});
	}
	__syncthreads();
#pragma unroll
	for (int d = 0; d < DT; ++d) lds.join[wave][d][lane] = acc[d][0] - 256 * acc[d][1] - 65536 * acc[d][2];
	__syncthreads();
#pragma unroll
	for (int i = 0; i < (DT + kCaWaves - 1) / kCaWaves; ++i) {
		const int d = wave + kCaWaves * i;
		if (DT % kCaWaves && d >= DT) break;
		v4i y = lds.join[0][d][lane];
#pragma unroll
		for (int k = 1; k < kCaWaves; ++k) y += lds.join[k][d][lane];
		if (ri < j.heads) *(v4i*)(w.part + (((size_t)j.plane * a.tokens + j.t) * a.NH + j.h0 + ri) * D + 16 * d + 4 * g) = y;
	}
}

// The whole of a single token's row in one launch, a block per (row, KV head, tile of heads): its waves take 64 positions in
// turn and keep their scores in LDS, or where these are too many (GS) in the workspace, from which i-exp and probabilities
// run on full waves, four heads at a time; maxima, sums and contexts are joined in LDS.  k_ca_out finds one plane.
// 12 heads / 2 KV x 128: 2 rows by 100 positions 10.8 us, the chain of one block's stages; 24 by 1500 19.9; 64 rows of 28 / 4 by up to
// 8000 95.7 with the scores in the workspace, 298 MB at 3.1 TB/s: the longest rows' blocks end last, and i-exp and probabilities are
// some 30 instructions of doubles to a score.
template <int D>
struct CrShape {
	static constexpr int NW = D <= 128 ? 8 : 4, STEP = 64 * NW, LD = 68;  // LD: a head's 64 scores, moved apart by a few banks
	static constexpr size_t kWave = 32 * D + 3 * 1024, kJoin = (size_t)NW * D * 64;
	static size_t lds(int heads, int64_t width, bool gs) {
		const size_t n = NW * kWave + (gs ? 0 : (size_t)((width + STEP - 1) / STEP) * NW * heads * LD * 4);
		return n > kJoin ? n : kJoin;
	}
};
constexpr int kCrSteps = 16;  // a lane holds the page of 16 positions of one of a wave's next 16 steps
template <int D, int R, bool GS>
__global__ __launch_bounds__(64 * CrShape<D>::NW, D <= 128 ? 2 : 1) void k_cr_row(CacheAttnArgs a, CaPlan pl, CaWork w) {
	constexpr int NW = CrShape<D>::NW, STEP = CrShape<D>::STEP, LD = GS ? 64 : CrShape<D>::LD, DT = D / 16, NC = (D + 63) / 64, PER = D / 16, RL = 64 / PER;
	extern __shared__ __attribute__((aligned(16))) int8_t row_lds[];
	__shared__ int32_t s_max[NW][16], s_bad[NW];
	__shared__ int64_t s_sum[NW][16];
	const int lane = threadIdx.x & 63, ri = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int G = a.NH / a.pg.NKV, tile = blockIdx.x % pl.ht, kvh = blockIdx.x / pl.ht % a.pg.NKV, r = blockIdx.x / pl.ht / a.pg.NKV;
	const int h0 = kvh * G + tile * 16, heads = min(16, G - tile * 16);
	// lane 4 i + t of a segment of kCrSteps steps from n on: positions 64 (wave + NW (n + i)) + 16 t .. + 15
	auto first_of = [&](int n) { return 64 * (wave + NW * (n + (lane >> 2))) + 16 * (lane & 3); };
	auto entry_of = [&](int n) { return a.pg.tables[(int64_t)r * a.pg.table_ld + min(first_of(n) >> a.pg.lp, a.pg.table_ld - 1)]; };
	const int32_t entry0 = entry_of(0);
	const CacheRow row = attn_row(a, r);
	if (!row.ok || row.n < 1) return;
	const int t = row.t0, last = (int)row.start, width = last + 1, steps = (width - 64 * wave + STEP - 1) / STEP;  // the wave's
	int32_t page = 0, ke = 0, ve = 0;
	bool wrong = false;
	auto enter = [&](int n) {
		const int32_t entry = n ? entry_of(n) : entry0;
		const bool out = entry < 0 || entry >= a.pg.pages;
		wrong |= (bool)__any(out && first_of(n) <= last);
		page = out ? 0 : entry;
		const uint8_t* ex = (const uint8_t*)a.pg.pool + page * a.pg.page_bytes + a.pg.e_off;
		ke = min((int)ex[kvh], kMaxShift);
		ve = min((int)ex[a.pg.NKV + kvh], kMaxShift);
	};
	const int64_t head = ((int64_t)kvh << a.pg.lp) * D;
	const int mask = (1 << a.pg.lp) - 1;
	// step n's rows, n0 + kCrSteps the segment's end; none past that, the row's end or behind a page that is none
	auto load = [&](SaRows<D>& x, int n, int n0, int64_t off) {
		const int p = 64 * (wave + NW * n);
		__amdgpu_buffer_rsrc_t b[4];
#pragma unroll
		for (int i = 0; i < 4; ++i) {
			const int pg = __builtin_amdgcn_readlane(page, min(4 * (n - n0) + i, 63));
			b[i] = __builtin_amdgcn_make_buffer_rsrc(a.pg.pool + (pg * a.pg.page_bytes + off + head), 0, p + 16 * i <= last && n - n0 < kCrSteps && !wrong ? D << a.pg.lp : 0, 0x00020000);
		}
		x.load_at([&](int u) {
			const int rr = u * RL + lane / PER;
			const uint32_t at = (uint32_t)(((p + rr) & mask) * D + lane % PER * 16);
			if constexpr (RL > 16) return buffer16(b[2 * u], lane / PER < 16 ? at : ~0u) | buffer16(b[2 * u + 1], lane / PER < 16 ? ~0u : at);
			else return buffer16(b[u * RL / 16], at);
		});
		__builtin_amdgcn_sched_barrier(0);
	};
	int8_t* stage = row_lds + wave * CrShape<D>::kWave;
	uint32_t* ops = (uint32_t*)(stage + 32 * D);  // [operand][256]: 64 positions' bytes of 16 heads
	int32_t* sc = (GS ? w.scores + ((size_t)t * a.NH + h0) * pl.wpad : (int32_t*)(row_lds + NW * CrShape<D>::kWave)) + wave * heads * LD;
	const int sc_step = NW * heads * LD;
	v4i q[NC];
	const int hq = h0 + min(ri, heads - 1);
#pragma unroll
	for (int c = 0; c < NC; ++c) q[c] = c * 64 + g * 16 < D ? load16(a.q + ((size_t)t * a.NH + hq) * D + c * 64 + g * 16) : v4i{0, 0, 0, 0};
	const RowScales rs{a.q_scale[t], a.khead_m[kvh], a.khead_e[kvh]};
	const RowConst rc = row_const(rs, a.ln2_q, a.b_q, a.ca_q, width);
	const SaConst c{rc.q_ln2, rc.q_b, rc.q_c, rc.ceil, rc.st, 0};
	int32_t m = INT32_MIN;
	int seg = 0;
	for (;; seg += kCrSteps) {
		enter(seg);
		SaRows<D> k[2];
		load(k[0], seg, seg, a.pg.k_off);
		load(k[1], seg + 1, seg, a.pg.k_off);
		for (int n0 = seg; n0 < min(steps, seg + kCrSteps); n0 += 2) {
#pragma unroll
			for (int b = 0; b < 2; ++b) {
				const int n = n0 + b, left = width - 64 * (wave + NW * n) - 4 * g;
				v4i s[4] = {};
				k[b].scores(stage, q, s);
				load(k[b], n + 2, seg, a.pg.k_off);
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					const int e = __builtin_amdgcn_readlane(ke, min(4 * (n - seg) + i, 63));
#pragma unroll
					for (int v = 0; v < 4; ++v) {
						s[i][v] <<= e;
						m = max(m, 16 * i + v < left ? s[i][v] : INT32_MIN);
					}
					if (ri < heads && n < steps) *(v4i*)(sc + n * sc_step + ri * LD + 16 * i + 4 * g) = s[i];
				}
			}
		}
		if (seg + kCrSteps >= steps) break;
	}
	SaRows<D> v;
	if (seg) {
		seg = 0;
		enter(0);
	}
	load(v, 0, 0, a.pg.v_off);  // in flight through the softmax
	m = max(m, __shfl_xor(m, 16, 64));
	m = max(m, __shfl_xor(m, 32, 64));
	if (g == 0) s_max[wave][ri] = m;
	if (lane == 0) s_bad[wave] = wrong;
	__syncthreads();
	int st = c.st;
#pragma unroll
	for (int i = 0; i < NW; ++i) st = s_bad[i] ? (int)kPositionOverCap : st;
	if (threadIdx.x == 0 && tile == 0) w.cst[(size_t)t * a.pg.NKV + kvh] = SaConst{0, 0, 0, 0, st, 0};
	if (st != kOk) return;
	// from here on a lane has four positions 4 ri .. + 3 of a step and the heads g, g + 4, ..
	const bool fast = ca_fast(c);
	const SaExp e0 = sa_exp_of(fast ? c : SaConst{1, 1, 0, 1, 0, 0}, 0);
	const double inv = 1.0 / (double)c.q_ln2;
	int32_t top[R];
#pragma unroll
	for (int i = 0; i < R; ++i) {
		const int h = min(g + 4 * i, heads - 1);
		top[i] = s_max[0][h];
#pragma unroll
		for (int x = 1; x < NW; ++x) top[i] = max(top[i], s_max[x][h]);
	}
	double acc1[R];
	int64_t sum[R];
	int bad = 0;
#pragma unroll
	for (int i = 0; i < R; ++i) {
		acc1[i] = 0.0;
		sum[i] = 0;
	}
	v4i x[R];
	auto scores = [&](int n) {
#pragma unroll
		for (int i = 0; i < R; ++i) x[i] = *(const v4i*)(sc + min(n, steps - 1) * sc_step + min(g + 4 * i, heads - 1) * LD + 4 * ri);
	};
	if (steps > 0) scores(0);
	for (int n = 0; n < steps; ++n) {
		const int left = width - 64 * (wave + NW * n) - 4 * ri;
		v4i now[R];
#pragma unroll
		for (int i = 0; i < R; ++i) now[i] = x[i];
		scores(n + 1);
#pragma unroll
		for (int i = 0; i < R; ++i) {
			if (fast) {
				SaExp e = e0;
				e.add -= top[i];
#pragma unroll
				for (int k4 = 0; k4 < 4; ++k4) {
					const double y = sa_exp(e, now[i][k4]);
					acc1[i] += k4 < left ? y : 0.0;
				}
				if ((n & 15) == 15) {  // 64 values of 2^47
					sum[i] += (int64_t)acc1[i];
					acc1[i] = 0.0;
				}
			} else {
#pragma unroll
				for (int k4 = 0; k4 < 4; ++k4) {
					if (k4 >= left) continue;
					const int64_t y = iexp_fast_cold((int64_t)now[i][k4] - top[i], c.q_ln2, inv, c.q_b, c.q_c, c.ceil);
					bad |= y < 0 ? 1 << i : 0;
					sum[i] += y < 0 ? 0 : y;
				}
			}
		}
	}
#pragma unroll
	for (int i = 0; i < R; ++i) {
		const int64_t x = row16_sum(sum[i] + (int64_t)acc1[i]);
		const bool b = row16_max(bad >> i & 1) != 0;
		if (ri == 0 && g + 4 * i < heads) s_sum[wave][g + 4 * i] = b ? -1 : x;
	}
	__syncthreads();
	CaProb pb[R];
	int64_t den[R];
	int refused = 0, big = 0;
#pragma unroll
	for (int i = 0; i < R; ++i) {
		const int h = min(g + 4 * i, heads - 1);
		int64_t x = 0;
#pragma unroll
		for (int y = 0; y < NW; ++y) {
			refused |= s_sum[y][h] < 0 ? 1 << i : 0;
			x += s_sum[y][h];
		}
		den[i] = !(refused >> i & 1) && x > 1 ? x : 1;
		big |= den[i] >= (int64_t)1 << 36;
		if (wave == 0 && ri == 0 && g + 4 * i < heads) w.hst[(size_t)t * a.NH + h0 + g + 4 * i] = refused >> i & 1 ? kSoftmaxKernelRefusedAfterGateAccepted : kOk;
	}
	const bool small = !__any(big);
#pragma unroll
	for (int i = 0; i < R; ++i) pb[i] = ca_prob_of(den[i], small);
	v4i acc[DT][3];
#pragma unroll
	for (int d = 0; d < DT; ++d) acc[d][0] = acc[d][1] = acc[d][2] = v4i{0, 0, 0, 0};
	if (steps > 0) scores(0);
	for (int n = 0; n < steps; ++n) {
		if (n == seg + kCrSteps) {
			seg = n;
			enter(n);
			load(v, n, seg, a.pg.v_off);
		}
		const int left = width - 64 * (wave + NW * n) - 4 * ri;
		const int sh = __shfl(ve, 4 * (n - seg) + (ri >> 2), 64);
#pragma unroll
		for (int i = 0; i < R; ++i) {
			SaExp e = e0;
			e.add -= top[i];
			int32_t pr[4];
#pragma unroll
			for (int k4 = 0; k4 < 4; ++k4) {
				if (fast) pr[k4] = small ? ca_prob<true>(pb[i], sa_exp(e, x[i][k4])) : ca_prob<false>(pb[i], sa_exp(e, x[i][k4]));
				else pr[k4] = k4 < left ? (int32_t)div_rcp_cold(iexp_fast_cold((int64_t)x[i][k4] - top[i], c.q_ln2, inv, c.q_b, c.q_c, c.ceil) << 15, den[i], 1.0 / (double)den[i], 32768) : 0;
				pr[k4] = k4 < left && !(refused >> i & 1) ? pr[k4] << sh : 0;
			}
			uint32_t y[3];
			sa_pack3_word(pr[0], pr[1], pr[2], pr[3], y);
			const int at = (g + 4 * i) * 16 + (ri & 3) * 4 + (ri >> 2);
#pragma unroll
			for (int z = 0; z < 3; ++z) ops[z * 256 + at] = y[z];
		}
		scores(n + 1);
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		__builtin_amdgcn_wave_barrier();
		v4i op[3];
#pragma unroll
		for (int z = 0; z < 3; ++z) op[z] = *(const v4i*)(ops + z * 256 + ri * 16 + g * 4);
		v.multiply(stage, op, acc);
		load(v, n + 1, seg, a.pg.v_off);
	}
	__syncthreads();
	v4i* join = (v4i*)row_lds;
#pragma unroll
	for (int d = 0; d < DT; ++d) join[(wave * DT + d) * 64 + lane] = acc[d][0] - 256 * acc[d][1] - 65536 * acc[d][2];
	__syncthreads();
#pragma unroll
	for (int i = 0; i < (DT + NW - 1) / NW; ++i) {
		const int d = wave + NW * i;
		if (DT % NW && d >= DT) break;
		v4i y = join[d * 64 + lane];
#pragma unroll
		for (int x = 1; x < NW; ++x) y += join[(x * DT + d) * 64 + lane];
		if (ri < heads) *(v4i*)(w.part + ((size_t)t * a.NH + h0 + ri) * D + 16 * d + 4 * g) = y;
	}
}

// A chunk's block: number `b` of the row groups, 64 query rows from the group's, and a plane.
struct CcJob {
	int r, kvh, plane, i0, count;  // i0: the block's first query row of `count` in the row
	int width, p0, p1;             // width: of the block's last token
	CacheRow row;
};
// The rows' groups are counted 64 rows at a time, a row to a lane.
__device__ __forceinline__ bool cc_job(const CacheAttnArgs& a, const CaPlan& pl, CcJob* j) {
	const int G = a.NH / a.pg.NKV, blk = blockIdx.x, lane = threadIdx.x & 63;
	// blocks go to the XCDs in turn: a (KV head, plane)'s groups stay on one, whose L2 then holds its K/V
	const int grp = (blk / 8 / pl.groups) * 8 + blk % 8;
	int b = (blk / 8) % pl.groups;
	if (grp >= a.pg.NKV * pl.planes) return false;
	j->plane = grp / a.pg.NKV;
	j->kvh = grp % a.pg.NKV;
	for (int r0 = 0;; r0 += 64) {
		if (r0 >= a.rows) return false;
		int n = 0;
		if (r0 + lane < a.rows) {
			const CacheRow row = attn_row(a, r0 + lane);
			n = row.ok ? (row.n * G + 63) / 64 : 0;
		}
		int x = n;
		for (int o = 1; o < 64; o *= 2) {
			const int y = __shfl_up(x, o, 64);
			x += lane >= o ? y : 0;
		}
		const uint64_t hit = __ballot(b < x);
		if (hit) {
			const int at = __builtin_ctzll(hit);
			b -= __builtin_amdgcn_readlane(x, at) - __builtin_amdgcn_readlane(n, at);
			j->r = r0 + at;
			break;
		}
		b -= __builtin_amdgcn_readlane(x, 63);
	}
	j->row = attn_row(a, j->r);
	j->i0 = b * 64;
	j->count = j->row.n * G;
	j->width = (int)j->row.start + (min(j->i0 + 64, j->count) - 1) / G + 1;
	j->p0 = j->plane * pl.sp;
	j->p1 = min(j->width, j->p0 + pl.sp);
	return j->p0 < j->p1;
}
// what a lane of the block has: its token, head and width (t < 0: none)
struct CcLane {
	int t, h, width;
};
__device__ __forceinline__ CcLane cc_lane(const CacheAttnArgs& a, const CcJob& j) {
	const int G = a.NH / a.pg.NKV, i = j.i0 + (int)(threadIdx.x >> 6) * 16 + (int)(threadIdx.x & 15);
	CcLane l{-1, j.kvh * G, 0};
	if (i < j.count) {
		l.t = j.row.t0 + i / G;
		l.h += i % G;
		l.width = (int)j.row.start + i / G + 1;
	}
	return l;
}
template <int D, int NC>
__device__ __forceinline__ void cc_load_q(const CacheAttnArgs& a, const CcLane& l, v4i (&q)[NC]) {
	const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
	for (int c = 0; c < NC; ++c)
		q[c] = l.t >= 0 && c * 64 + g * 16 < D ? load16(a.q + ((size_t)l.t * a.NH + l.h) * D + c * 64 + g * 16) : v4i{0, 0, 0, 0};
}

// Steps of 64 positions over the block's plane: `step(p, last, scores, pages, multiply)`.  Each thread loads its share of a
// step's rows two steps ahead and stages it into one of two buffers, so a step costs one barrier.  LDS: 64 D bytes a buffer, K's two and then V's
// two.  False, for the whole block, when one of the plane's pages is none.
template <int D, bool WITH_V, int NC, typename F>
__device__ __forceinline__ bool cc_steps(const CacheAttnArgs& a, const CcJob& j, int8_t* lds, const v4i (&q)[NC], F&& step) {
	constexpr int BS = 64 * kCaWaves, CH = 4 * D, PT = (CH + BS - 1) / BS, PER = D / 16, AHEAD = D <= 128 ? 2 : 1;
	const Pages& g = a.pg;
	const int64_t head = ((int64_t)j.kvh << g.lp) * D;
	const int mask = (1 << g.lp) - 1;
	int b = 0;
	for (int s0 = j.p0; s0 < j.p1; s0 = pages_end(g, s0)) {
		const int s1 = min(j.p1, pages_end(g, s0)), last = s1 - 1;
		LanePages lp;
		if (!lane_pages(g, j.r, j.kvh, s0, last, &lp)) return false;
		v4i kr[AHEAD][PT], vr[AHEAD][PT], s[4];
		auto load = [&](int p, v4i (&k)[PT], v4i (&v)[PT]) {
#pragma unroll
			for (int u = 0; u < PT; ++u) {
				const int c = min((int)threadIdx.x + u * BS, CH - 1), row = c / PER;
				// a wave's rows of one load: within 16 (32 at D = 32)
				const int r0 = p + (__builtin_amdgcn_readfirstlane(row) & ~15);
				const uint32_t at = (uint32_t)(((p + row) & mask) * D + c % PER * 16);
				auto get = [&](int64_t off) {
					const auto b = page_rows(g, lp, r0, last, off);
					if constexpr (D == 32) {
						const bool second = (row & 16) != (__builtin_amdgcn_readfirstlane(row) & 16);
						return buffer16(b, second ? ~0u : at) | buffer16(page_rows(g, lp, r0 + 16, last, off), second ? at : ~0u);
					} else return buffer16(b, at);
				};
				k[u] = get(g.k_off + head);
				if (WITH_V) v[u] = get(g.v_off + head);
			}
		};
#pragma unroll
		for (int i = 0; i < AHEAD; ++i) load(s0 + 64 * i, kr[i], vr[i]);
		for (int p0 = s0; p0 < s1; p0 += 64 * AHEAD) {
#pragma unroll
			for (int i = 0; i < AHEAD; ++i) {
				const int p = p0 + 64 * i;
				if (i && p >= s1) break;
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
				const int lane = threadIdx.x & 63, ri = lane & 15, gg = lane >> 4;
#pragma unroll
				for (int t = 0; t < 4; ++t) {
					s[t] = v4i{0, 0, 0, 0};
#pragma unroll
					for (int c = 0; c < NC; ++c) {
						const int ch = c * 4 + gg;
						const v4i k = *(const v4i*)(kb + SaRows<D>::at(t * 16 + ri, D < 64 ? ch & (PER - 1) : ch));
						s[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k, q[c], s[t], 0, 0, 0);
					}
					const int e = page_exp(g, lp, lp.ke, p + 16 * t, last);
#pragma unroll
					for (int v = 0; v < 4; ++v) s[t][v] <<= e;
				}
				step(p, last, s, lp, [&](const v4i (&x)[3], v4i (&acc)[D / 16][3]) {
					const int k = ri >> 1, row = (k >> 2) * 16 + gg * 4 + (k & 3);
#pragma unroll
					for (int dt = 0; dt < D / 16; ++dt) {
						const int8_t* from = vb + SaRows<D>::at(row, dt) + 8 * (ri & 1);  // rows 32 apart change places alike
						const v2i y = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)from);
						const v2i z = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) v2i*)(from + 32 * D));
						const v4i m = v4i{y.x, y.y, z.x, z.y};
#pragma unroll
						for (int n = 0; n < 3; ++n) acc[dt][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(m, x[n], acc[dt][n], 0, 0, 0);
					}
				});
				b ^= 1;
			}
		}
	}
	return true;
}

// how many of a step's positions, counted from the lane's first (4 g), lie before `end`
__device__ __forceinline__ int ca_left(int p, int end) { return end - p - ((threadIdx.x & 63) >> 4) * 4; }

// a (token, head)'s maximum or sum over its planes; the lanes ri, ri + 16, ri + 32, ri + 48 share the work
__device__ __forceinline__ int32_t cc_top(const CacheAttnArgs& a, const CaPlan& pl, const CaWork& w, const CcLane& l, bool live) {
	const int n = live ? (l.width + pl.sp - 1) / pl.sp : 0;
	int32_t m = INT32_MIN;
	for (int i = (threadIdx.x & 63) >> 4; i < n; i += 4) m = max(m, w.pmax[((size_t)i * a.tokens + l.t) * a.NH + l.h]);
	m = max(m, __shfl_xor(m, 16, 64));
	return max(m, __shfl_xor(m, 32, 64));
}
__device__ __forceinline__ int64_t cc_sum(const CacheAttnArgs& a, const CaPlan& pl, const CaWork& w, const CcLane& l, bool live) {
	const int n = live ? (l.width + pl.sp - 1) / pl.sp : 0;
	int64_t sum = 0;
	int bad = 0;
	for (int i = (threadIdx.x & 63) >> 4; i < n; i += 4) {
		const int64_t x = w.psum[((size_t)i * a.tokens + l.t) * a.NH + l.h];
		bad |= x < 0;
		sum += x;
	}
	for (int o = 16; o < 64; o *= 2) {
		sum += __shfl_xor(sum, o, 64);
		bad |= __shfl_xor(bad, o, 64);
	}
	return bad ? -1 : sum;
}

// The maxima of 64 query rows over a plane: scores on the MFMAs from K tiles of 64 positions that the block's waves share through LDS.
// The softmax rounds each probability by the whole row's sum, so a running maximum with rescaling would not be exact: maxima, sums
// and P V are three passes that compute the scores again, less than keeping chunk x width of them would cost.  A chunk of 500 at 2000,
// 12 heads / 2 KV x 128: 9.6 + 15.8 + 34.3 us.
template <int D>
__global__ __launch_bounds__(64 * kCaWaves) void k_cc_max(CacheAttnArgs a, CaPlan pl, CaWork w) {
	constexpr int NC = (D + 63) / 64;
	__shared__ __attribute__((aligned(16))) int8_t lds[2 * 64 * D];
	CcJob j;
	if (!cc_job(a, pl, &j)) return;
	const CcLane l = cc_lane(a, j);
	const int g = (threadIdx.x & 63) >> 4;
	v4i q[NC];
	cc_load_q<D>(a, l, q);
	if (j.plane == 0) {  // a token's constants, by every lane that has a head of it
		SaConst c{0, 0, 0, 0, kPositionOverCap, 0};
		if (row_pages_ok(a.pg, j.r, j.row.start + j.row.n) && l.t >= 0) {
			const RowConst rc = row_const(RowScales{a.q_scale[l.t], a.khead_m[j.kvh], a.khead_e[j.kvh]}, a.ln2_q, a.b_q, a.ca_q, l.width);
			c = SaConst{rc.q_ln2, rc.q_b, rc.q_c, rc.ceil, rc.st, 0};
		}
		if (g == 0 && l.t >= 0) w.cst[(size_t)l.t * a.pg.NKV + j.kvh] = c;
	}
	const int end = min(j.p1, l.width);
	int32_t m = INT32_MIN;
	cc_steps<D, false>(a, j, lds, q, [&](int p, int, v4i (&s)[4], const LanePages&, auto&&) {
		const int left = ca_left(p, end);
#pragma unroll
		for (int t = 0; t < 4; ++t)
#pragma unroll
			for (int v = 0; v < 4; ++v) m = max(m, t * 16 + v < left ? s[t][v] : INT32_MIN);
	});
	m = max(m, __shfl_xor(m, 16, 64));
	m = max(m, __shfl_xor(m, 32, 64));
	if (g == 0 && l.t >= 0) w.pmax[((size_t)j.plane * a.tokens + l.t) * a.NH + l.h] = m;
}

// The sums of i-exp: the same scores again; bound by the doubles of i-exp, some 12 instructions to a score and lane.
template <int D>
__global__ __launch_bounds__(64 * kCaWaves, D <= 128 ? 4 : 2) void k_cc_sum(CacheAttnArgs a, CaPlan pl, CaWork w) {
	constexpr int NC = (D + 63) / 64;
	__shared__ __attribute__((aligned(16))) int8_t lds[2 * 64 * D];
	__shared__ int s_vote[kCaWaves];
	CcJob j;
	if (!cc_job(a, pl, &j)) return;
	const CcLane l = cc_lane(a, j);
	const int g = (threadIdx.x & 63) >> 4;
	const SaConst c = w.cst[(size_t)max(l.t, 0) * a.pg.NKV + j.kvh];
	const bool live = l.t >= 0 && c.st == kOk;
	v4i q[NC];
	cc_load_q<D>(a, l, q);
	const int32_t top = cc_top(a, pl, w, l, live);
	const int end = live ? min(j.p1, l.width) : 0;
	int64_t sum = 0;
	int bad = 0;
	if (!block_vote(live && !ca_fast(c), s_vote)) {
		const SaExp e = sa_exp_of(live ? c : SaConst{1, 1, 0, 1, 0, 0}, top);
		cc_steps<D, false>(a, j, lds, q, [&](int p, int, v4i (&s)[4], const LanePages&, auto&&) {
			const int left = ca_left(p, end);
			double acc = 0.0;
#pragma unroll
			for (int t = 0; t < 4; ++t)
#pragma unroll
				for (int v = 0; v < 4; ++v) {
					const double x = sa_exp(e, s[t][v]);
					acc += t * 16 + v < left ? x : 0.0;
				}
			sum += (int64_t)acc;
		});
	} else {
		const double inv = 1.0 / (double)c.q_ln2;
		cc_steps<D, false>(a, j, lds, q, [&](int p, int, v4i (&s)[4], const LanePages&, auto&&) {
			const int left = ca_left(p, end);
#pragma unroll
			for (int i = 0; i < 16; ++i) {
				if ((i >> 2) * 16 + (i & 3) >= left) continue;
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
	if (g == 0 && live) w.psum[((size_t)j.plane * a.tokens + l.t) * a.NH + l.h] = bad ? -1 : sum;
}

// P V: the scores a third time, i-exp and the exact probability of each (some 20 instructions of doubles, which bound it), its 16 bits
// and the page's exponent as three int8 operands, and three MFMAs for each 16 dims.
template <int D>
__global__ __launch_bounds__(64 * kCaWaves, D <= 128 ? 2 : 1) void k_cc_pv(CacheAttnArgs a, CaPlan pl, CaWork w) {
	constexpr int NC = (D + 63) / 64, DT = D / 16;
	__shared__ __attribute__((aligned(16))) int8_t lds[4 * 64 * D];
	__shared__ int s_vote[kCaWaves];
	CcJob j;
	if (!cc_job(a, pl, &j)) return;
	const CcLane l = cc_lane(a, j);
	const int g = (threadIdx.x & 63) >> 4;
	const SaConst c = w.cst[(size_t)max(l.t, 0) * a.pg.NKV + j.kvh];
	bool live = l.t >= 0 && c.st == kOk;
	v4i q[NC], acc[DT][3];
	cc_load_q<D>(a, l, q);
	const int32_t top = cc_top(a, pl, w, l, live);
	const int64_t sum = cc_sum(a, pl, w, l, live);
	if (j.plane == 0 && g == 0 && live) w.hst[(size_t)l.t * a.NH + l.h] = sum < 0 ? kSoftmaxKernelRefusedAfterGateAccepted : kOk;
	live = live && sum >= 0;
	const int64_t den = live && sum > 1 ? sum : 1;
	const int end = live ? min(j.p1, l.width) : 0;
#pragma unroll
	for (int d = 0; d < DT; ++d) acc[d][0] = acc[d][1] = acc[d][2] = v4i{0, 0, 0, 0};
	const int form = block_vote((live && !ca_fast(c) ? 1 : 0) | (den >= ((int64_t)1 << 36) ? 2 : 0), s_vote);
	auto run = [&](auto&& value) {
		cc_steps<D, true>(a, j, lds, q, [&](int p, int last, v4i (&s)[4], const LanePages& lp, auto&& multiply) {
			const int left = ca_left(p, end);
			int32_t pr[16];
#pragma unroll
			for (int t = 0; t < 4; ++t) {
				const int sh = page_exp(a.pg, lp, lp.ve, p + 16 * t, last);
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					const int32_t x = value(s[t][i], 16 * t + i < left);
					pr[4 * t + i] = 16 * t + i < left ? x << sh : 0;
				}
			}
			v4i x[3];
			sa_pack3(pr, x);
			multiply(x, acc);
		});
	};
	const SaExp e = sa_exp_of(live && !(form & 1) ? c : SaConst{1, 1, 0, 1, 0, 0}, top);
	const CaProb pb = ca_prob_of(den, !(form & 2));
	if (form == 0) run([&](int32_t x, bool) { return ca_prob<true>(pb, sa_exp(e, x)); });
	else if (form == 2) run([&](int32_t x, bool) { return ca_prob<false>(pb, sa_exp(e, x)); });
	else {
		const double inv = 1.0 / (double)c.q_ln2, dinv = 1.0 / (double)den;
		run([&](int32_t x, bool in) {
			return in ? (int32_t)div_rcp_cold(iexp_fast_cold((int64_t)x - top, c.q_ln2, inv, c.q_b, c.q_c, c.ceil) << 15, den, dinv, 32768) : 0;
		});
	}
	if (l.t < 0) return;
	int32_t* out = w.part + (((size_t)j.plane * a.tokens + l.t) * a.NH + l.h) * D + 4 * g;
#pragma unroll
	for (int d = 0; d < DT; ++d) *(v4i*)(out + 16 * d) = acc[d][0] - 256 * acc[d][1] - 65536 * acc[d][2];
}

// The planes' contexts of one token joined, folded and requantized (checked_chain_funnel.cpp:257-364), U units of
// four dims to a thread.
template <int BS, int U>
__global__ __launch_bounds__(BS) void k_ca_out(CacheAttnArgs a, CaPlan pl, CaWork w) {
	__shared__ uint32_t s_red[2 * BS / 64];
	const int r = blockIdx.y, tid = threadIdx.x, N = a.NH * a.pg.D, G = a.NH / a.pg.NKV;
	const CacheRow c = attn_row(a, r);
	if (!c.ok) {
		for (int i = blockIdx.x * BS + tid; i < c.n; i += gridDim.x * BS) a.status[c.t0 + i] = kPositionOverCap;
		return;
	}
	if ((int)blockIdx.x >= c.n) return;
	const int t = c.t0 + blockIdx.x;
	const int n = (int)((c.start + blockIdx.x + pl.sp) / pl.sp);
	// the first refusing head, heads of one KV head sharing its constants' status
	uint32_t first = 0xffffffffu;
	for (int h = tid; h < a.NH; h += BS) {
		const int32_t st = w.cst[(size_t)t * a.pg.NKV + h / G].st, x = st != kOk ? st : w.hst[(size_t)t * a.NH + h];
		if (x != kOk) first = min(first, (uint32_t)h << 8 | (uint32_t)x);
	}
	FoldConsts fc[U];
	v4i v[U];
	const int32_t* at[U];
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int i = 4 * min(tid + u * BS, N / 4 - 1);
		const int32_t* cf = a.ctx_fold + 3 * (i / a.pg.D);
		fc[u] = fold_consts(cf[0], cf[1], cf[2]);
		v[u] = v4i{0, 0, 0, 0};
		at[u] = w.part + (size_t)t * N + i;
	}
	constexpr int PK = 8 / U;  // planes in flight
	for (int k = 0; k < n; k += PK) {
		v4i x[PK][U];
#pragma unroll
		for (int e = 0; e < PK; ++e)
#pragma unroll
			for (int u = 0; u < U; ++u) x[e][u] = *(const v4i*)(at[u] + (size_t)min(k + e, n - 1) * a.tokens * N);
#pragma unroll
		for (int e = 0; e < PK; ++e)
#pragma unroll
			for (int u = 0; u < U; ++u) v[u] += k + e < n ? x[e][u] : v4i{0, 0, 0, 0};
	}
	uint32_t mx = 0;
#pragma unroll
	for (int u = 0; u < U; ++u)  // a clamped unit repeats the last one
#pragma unroll
		for (int x = 0; x < 4; ++x) {
			v[u][x] = fold_bounded(v[u][x], fc[u]);  // |context| <= 2^15 kMaxUnits, and half of a fold's 2^31 more stays in 32 bits
			mx = max(mx, (uint32_t)(v[u][x] < 0 ? -v[u][x] : v[u][x]));
		}
	mx = wave_max32(mx);
	first = ~wave_max32(~first);
	if ((tid & 63) == 0) {
		s_red[tid >> 6] = mx;
		s_red[BS / 64 + (tid >> 6)] = first;
	}
	__syncthreads();
#pragma unroll
	for (int i = 0; i < BS / 64; ++i) {
		mx = max(mx, s_red[i]);
		first = min(first, s_red[BS / 64 + i]);
	}
	if (first != 0xffffffffu) {
		if (tid == 0) a.status[t] = (int32_t)(first & 0xff);
		return;
	}
	FunnelPlan plan;
	const int32_t st = funnel_plan(__builtin_amdgcn_readfirstlane(mx), nullptr, 0, a.site, &plan);
	if (tid == 0) {
		a.status[t] = st;
		if (st == kOk) a.scales[t] = plan.out;
	}
	if (st != kOk) return;
#pragma unroll
	for (int u = 0; u < U; ++u) {
		const int i = tid + u * BS;
		if (4 * i < N) {
			uint32_t o = 0;
#pragma unroll
			for (int x = 0; x < 4; ++x) o |= (uint32_t)(uint8_t)requant_code_f(v[u][x], plan.f) << 8 * x;
			((unaligned4*)(a.codes + (size_t)t * N + 4 * i))->v = (int32_t)o;
		}
	}
}

}  // namespace sslm

// ------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------
namespace sslm_launch {

static size_t plan_work(int rows, int pages, int table_ld, char* base, PlanWork* w) {
	size_t at = 0;
	auto take = [&](size_t n) {
		int32_t* p = (int32_t*)(base + at);
		at += up256(n * 4);
		return p;
	};
	w->state = take(2);
	w->row = (v4i*)take(4 * (size_t)rows);
	w->free = take(pages);
	w->from = take(std::max(rows, pages));
	w->to = take(rows);
	w->old = take((size_t)rows * table_ld);
	return at;
}

size_t page_update_workspace(int rows, int pages, int table_ld) {
	PlanWork w;
	return plan_work(rows, pages, table_ld, nullptr, &w);
}
size_t page_compact_workspace(int rows, int pages, int table_ld) {
	PlanWork w;
	return plan_work(rows, pages, table_ld, nullptr, &w);
}

// The most dynamic LDS that a launch here asks for; beside it the plans' 9 KB of their own.  A kernel's limit is always set to
// this, so that calls of other sizes from other threads leave it where it is.
constexpr int kMostLds = 150 * 1024;
template <typename K>
static void allow_lds(K kernel, size_t bytes) {
	if (bytes > 32768 && (bytes > kMostLds || hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kMostLds) != hipSuccess))
		throw LaunchRefused{"dynamic LDS"};
}

// blocks for a launch over `cells` entries and up to `copies` pages
static int apply_blocks(int64_t cells, int64_t copies, int64_t page_bytes) {
	const int64_t want = std::max((cells + 255) / 256, copies * ((page_bytes + kCopyChunk - 1) / kCopyChunk));
	return (int)std::min<int64_t>(2048, std::max<int64_t>(1, want));
}

void page_update(const PageUpdateArgs& a, hipStream_t s) {
	PlanWork w;
	plan_work(a.rows, a.pages, a.table_ld, (char*)a.ws, &w);
	const int64_t cells = (int64_t)a.rows * a.table_ld;
	const int32_t* tables = a.tables;
	if (a.new_tables < a.tables + cells && a.tables < a.new_tables + cells) {  // in place: rows are read by others' blocks
		hipLaunchKernelGGL(k_table_copy, dim3((int)std::min<int64_t>(1024, (cells + 255) / 256)), dim3(256), 0, s, a.tables, w.old, cells);
		tables = w.old;
	}
	const size_t lds = 3 * (size_t)((a.pages + 31) / 32) * 4 + (size_t)a.rows * 12;
	allow_lds(k_update_plan, lds);
	hipLaunchKernelGGL(k_update_plan, dim3(1), dim3(kPlanBlock), lds, s, a, tables, w);
	hipLaunchKernelGGL(k_update_apply, dim3(apply_blocks(cells, a.rows, a.page_bytes)), dim3(256), 0, s, a, tables, w);
}

void page_compact(const PageCompactArgs& a, hipStream_t s) {
	PlanWork w;
	plan_work(a.rows, a.pages, a.table_ld, (char*)a.ws, &w);
	const size_t lds = 3 * (size_t)((a.pages + 31) / 32) * 4 + (size_t)a.rows * 4;
	allow_lds(k_compact_plan, lds);
	hipLaunchKernelGGL(k_compact_plan, dim3(1), dim3(kPlanBlock), lds, s, a, w);
	hipLaunchKernelGGL(k_compact_apply, dim3(apply_blocks((int64_t)a.rows * a.table_ld, a.pages, a.page_bytes)), dim3(256), 0, s, a, w);
}

template <int D>
static void store_launch(const CacheStoreArgs& a, hipStream_t s) {
	if (a.max_new == 1) {
		hipLaunchKernelGGL(k_store_token<D>, dim3(a.rows), dim3(kStoreBlock), 0, s, a);
		return;
	}
	const int P = 1 << a.pg.lp, pages = (a.max_new + P - 2) / P + 1;
	const int qs = a.q ? (a.max_new + kStoreBlock / 64 * 2 * a.pg.NKV - 1) / (kStoreBlock / 64 * 2 * a.pg.NKV) : 0;
	const size_t lds = (size_t)std::min(P, a.max_new) * D * 2;
	allow_lds(k_store_span<D>, lds);
	hipLaunchKernelGGL(k_store_check, dim3(a.rows), dim3(256), 0, s, a);
	hipLaunchKernelGGL(k_store_span<D>, dim3(pages + qs, a.rows, 2 * a.pg.NKV), dim3(kStoreBlock), lds, s, a, pages);
}

void cache_store(const CacheStoreArgs& a, hipStream_t s) {
	switch (a.pg.D) {
		case 32: return store_launch<32>(a, s);
		case 64: return store_launch<64>(a, s);
		case 128: return store_launch<128>(a, s);
		default: return store_launch<256>(a, s);
	}
}

// Blocks that fill the chip: more cost their own start, fewer leave CUs idle.  A call at 768, 1536, 2560 and 4096 blocks: 64 rows of
// 12 heads / 2 KV x 128 by 4000 positions 50, 48, 60 and 60 us, 2 rows by 8000 25, 23, 25 and 25, 8 rows of 28 / 4 by 16000 56 each.  A chunk of 500 at 2000, its three launches: 62 at 384, 59 at 768, 73 at 1536.
constexpr int kCdTargetBlocks = 1536, kCcTargetBlocks = 768;

// Rows of up to max_width by k_cr_row: 1 with their scores in LDS, 2 in the workspace, 0 by planes.  A block takes some 6.8 us for 1000
// positions of 128 dims by itself; the planes' three launches take 8 us more to start and then share the chip, so that they are
// the faster form the longer the rows and the fewer the (row, KV head)s.  Row kernel / planes, us: 2 x 2 KV heads 19.5 / 21.3 at 1000
// positions, 26.6 / 20.6 at 2000; 16 x 4 28 / 27 at 2000, 45 / 40 at 4000; 64 x 2 46 / 47 at 4000, 78 / 72 at 8000; 64 x 4 59 / 78 at
// 4000, 313 / 326 at 20000; 32 x 2 x 64 dims 18 / 20 at 1000, 24 / 23 at 2000; 24 x 2 x 256 25 / 25 at 1000, 38 / 35 at 2000.  These are rows
// of one length.  From 210 blocks on every batch takes this form, also one whose longest row is far from the others, which then ends the
// launch by itself: 110 rows of 100 positions and one of 100000, 2 KV heads, 745 / 197.
template <int D>
static int cr_form(int64_t units, int NH, int NKV, int64_t max_width) {
	if (max_width * (210 - units) > 257000) return 0;
	return CrShape<D>::lds(std::min(16, NH / NKV), max_width, false) <= kMostLds ? 1 : 2;
}
static int cr_form(int64_t units, int NH, int NKV, int D, int64_t max_width) {
	switch (D) {
		case 32: return cr_form<32>(units, NH, NKV, max_width);
		case 64: return cr_form<64>(units, NH, NKV, max_width);
		case 128: return cr_form<128>(units, NH, NKV, max_width);
		default: return cr_form<256>(units, NH, NKV, max_width);
	}
}

// Planes: as many as fill the chip, at most some 4 sqrt(steps) of them, as their maxima and contexts are joined by
// each (token, head) and token.
static CaPlan ca_plan(int rows, int tokens, int max_new, int NH, int NKV, int D, int64_t max_width) {
	CaPlan p{};
	const int G = NH / NKV, step = max_new == 1 ? kCdStep : 64;
	p.ht = (G + 15) / 16;
	p.groups = max_new == 1 ? 0 : (int)((int64_t)tokens * G / 64 + rows);
	const int64_t units = max_new == 1 ? (int64_t)rows * NKV * p.ht : (int64_t)p.groups * NKV;
	p.whole = max_new == 1 ? cr_form(units, NH, NKV, D, max_width) : 0;
	const int64_t steps = (max_width + step - 1) / step;
	int64_t planes = p.whole ? 1 : std::min(steps, std::max<int64_t>(1, (max_new == 1 ? kCdTargetBlocks : kCcTargetBlocks) / units));
	planes = std::min(planes, std::max<int64_t>(1, (int64_t)std::sqrt(16.0 * (double)steps)));
	p.sp = (int)((steps + planes - 1) / planes * step);
	p.planes = (int)((max_width + p.sp - 1) / p.sp);
	p.ps = kCdSum;
	p.parts = p.whole ? 0 : (max_new == 1 ? (int)((max_width + p.ps - 1) / p.ps) : p.planes);
	p.wpad = p.whole == 1 ? 0 : (max_width + 511) / 512 * 512;
	return p;
}

static size_t ca_work(const CaPlan& p, int tokens, int max_new, int NH, int NKV, int D, char* base, CaWork* w) {
	size_t at = 0;
	auto take = [&](size_t n) {
		char* q = base + at;
		at += up256(n);
		return q;
	};
	const size_t th = (size_t)tokens * NH;
	w->cst = (SaConst*)take((size_t)tokens * NKV * sizeof(SaConst));
	w->pmax = (int32_t*)take(p.planes * th * 4);
	w->top = (int32_t*)take(th * 4);
	w->psum = (int64_t*)take(p.parts * th * 8);
	w->part = (int32_t*)take(p.planes * th * D * 4);
	w->hst = (int32_t*)take(th * 4);
	w->scores = (int32_t*)take(max_new == 1 ? th * p.wpad * 4 : 0);
	return at;
}

size_t cache_attn_workspace(int rows, int tokens, int max_new, int NH, int NKV, int D, int64_t max_width) {
	// a launch takes fewer than 2^32 threads along x
	constexpr int64_t kMost = 1ll << 32;
	if ((int64_t)max_new * 1024 >= kMost || (max_new > 1 && (int64_t)tokens * (NH / NKV) / 64 + rows >= kMost / 256)) return 0;
	const CaPlan p = ca_plan(rows, tokens, max_new, NH, NKV, D, max_width);
	const int64_t blocks = max_new == 1 ? (int64_t)rows * NKV * p.ht * p.planes : (int64_t)((p.planes * NKV + 7) / 8 * 8) * p.groups;
	if (blocks * (p.whole ? 512 : 64 * kCaWaves) >= kMost) return 0;
	// kept scores pass 64 bits of bytes at 2^38 (token, head)s by 2^24 positions; all the others stay below 2^58
	if (max_new == 1 && (double)tokens * NH * (double)p.wpad * 4.0 >= 0x1p62) return 0;
	CaWork w;
	return ca_work(p, tokens, max_new, NH, NKV, D, nullptr, &w);
}

template <int D>
static void attn_launch(const CacheAttnArgs& a, hipStream_t s) {
	const int NKV = a.pg.NKV, N = a.NH * D;
	const CaPlan p = ca_plan(a.rows, a.tokens, a.max_new, a.NH, NKV, D, a.max_width);
	CaWork w;
	ca_work(p, a.tokens, a.max_new, a.NH, NKV, D, (char*)a.ws, &w);
	const dim3 bs(64 * kCaWaves);
	const int G = a.NH / NKV;
	if (p.whole) {
		const size_t lds = CrShape<D>::lds(std::min(16, G), a.max_width, p.whole == 2);
		auto run = [&](auto kernel) {
			allow_lds(kernel, lds);
			hipLaunchKernelGGL(kernel, dim3((unsigned)(a.rows * NKV * p.ht)), dim3(64 * CrShape<D>::NW), lds, s, a, p, w);
		};
		if (p.whole == 1) {
			if (G <= 4) run(k_cr_row<D, 1, false>);
			else if (G <= 8) run(k_cr_row<D, 2, false>);
			else run(k_cr_row<D, 4, false>);
		} else {
			if (G <= 4) run(k_cr_row<D, 1, true>);
			else if (G <= 8) run(k_cr_row<D, 2, true>);
			else run(k_cr_row<D, 4, true>);
		}
	} else if (a.max_new == 1) {
		const dim3 grid((unsigned)(a.rows * NKV * p.ht * p.planes));
		hipLaunchKernelGGL(k_cd_scores<D>, grid, bs, 0, s, a, p, w);
		hipLaunchKernelGGL(k_cd_sum, dim3(p.parts, a.NH, a.rows), dim3(256), 0, s, a, p, w);
		if (G <= 4) hipLaunchKernelGGL((k_cd_pv<D, 1>), grid, bs, 0, s, a, p, w);
		else if (G <= 8) hipLaunchKernelGGL((k_cd_pv<D, 2>), grid, bs, 0, s, a, p, w);
		else hipLaunchKernelGGL((k_cd_pv<D, 4>), grid, bs, 0, s, a, p, w);
	} else {
		const dim3 grid((unsigned)((p.planes * NKV + 7) / 8 * 8 * p.groups));
		hipLaunchKernelGGL(k_cc_max<D>, grid, bs, 0, s, a, p, w);
		hipLaunchKernelGGL(k_cc_sum<D>, grid, bs, 0, s, a, p, w);
		hipLaunchKernelGGL(k_cc_pv<D>, grid, bs, 0, s, a, p, w);
	}
	const dim3 out(a.max_new, a.rows);
	if (N <= 1024) hipLaunchKernelGGL((k_ca_out<256, 1>), out, dim3(256), 0, s, a, p, w);
	else if (N <= 2048) hipLaunchKernelGGL((k_ca_out<512, 1>), out, dim3(512), 0, s, a, p, w);
	else if (N <= 4096) hipLaunchKernelGGL((k_ca_out<1024, 1>), out, dim3(1024), 0, s, a, p, w);
	else hipLaunchKernelGGL((k_ca_out<1024, 2>), out, dim3(1024), 0, s, a, p, w);
}

void cache_attn(const CacheAttnArgs& a, hipStream_t s) {
	switch (a.pg.D) {
		case 32: return attn_launch<32>(a, s);
		case 64: return attn_launch<64>(a, s);
		case 128: return attn_launch<128>(a, s);
		default: return attn_launch<256>(a, s);
	}
}

}  // namespace sslm_launch

// ------------------------------------------------------------------------------------------
// C entries
// ------------------------------------------------------------------------------------------
using namespace sslm_launch;

static int log2_page(int32_t positions) {
	for (int lp = 4; lp <= 8; ++lp)
		if (positions == 1 << lp) return lp;
	return -1;
}

static bool plan_ok(int32_t rows, int32_t pages, int32_t table_ld) {
	return rows >= 1 && rows <= SSLM_HIP_CACHE_MAX_ROWS && pages >= 1 && pages <= SSLM_HIP_CACHE_MAX_PAGES && table_ld >= 1 &&
	       table_ld <= SSLM_HIP_CACHE_MAX_WIDTH / 16;
}

static bool pool_ok(const void* pool, int64_t page_bytes, int32_t pages) {
	return pool && (uintptr_t)pool % 16 == 0 && page_bytes >= 16 && page_bytes % 16 == 0 && page_bytes <= ((int64_t)1 << 40) / pages;
}

// One layer's view: K, V and the exponents within a page.
static bool layer_ok(const Pages& g) {
	const int64_t half = ((int64_t)g.NKV << g.lp) * g.D;
	return g.k_off >= 0 && g.v_off >= 0 && g.e_off >= 0 && g.k_off % 16 == 0 && g.v_off % 16 == 0 && g.page_bytes >= half &&
	       g.k_off <= g.page_bytes - half && g.v_off <= g.page_bytes - half && g.e_off <= g.page_bytes - 2 * (int64_t)g.NKV;
}

static bool heads_ok(int32_t heads, int32_t kv_heads, int32_t d) {
	return heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0 && (d == 32 || d == 64 || d == 128 || d == 256) && (int64_t)heads * d <= 8192;
}

extern "C" {

size_t sslm_hip_cache_update_workspace(int32_t rows, int32_t pages, int32_t table_ld) {
	return plan_ok(rows, pages, table_ld) ? page_update_workspace(rows, pages, table_ld) : 0;
}

sslm_status sslm_hip_cache_update(const sslm_hip_cache_update_args* p, void* workspace, size_t workspace_bytes, void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_cache_update_workspace(p->rows, p->pages, p->table_ld);
	const int lp = log2_page(p->page_tokens);
	if (!need || lp < 0 || !pool_ok(p->pool, p->page_bytes, p->pages) || !p->tables || !p->lengths || !p->source || !p->keep || !p->room ||
	    !p->new_tables || !p->new_lengths || !p->result)
		return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	const PageUpdateArgs a{p->rows, p->pages, lp, p->table_ld, p->pool, p->page_bytes, p->tables, p->lengths, p->source, p->keep, p->room,
	                       p->held, p->new_tables, p->new_lengths, p->result, workspace};
	return on_stream(stream, [&](hipStream_t s) { page_update(a, s); });
}

size_t sslm_hip_cache_compact_workspace(int32_t rows, int32_t pages, int32_t table_ld) {
	return plan_ok(rows, pages, table_ld) ? page_compact_workspace(rows, pages, table_ld) : 0;
}

sslm_status sslm_hip_cache_compact(const sslm_hip_cache_compact_args* p, void* workspace, size_t workspace_bytes, void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_cache_compact_workspace(p->rows, p->pages, p->table_ld);
	const int lp = log2_page(p->page_tokens);
	if (!need || lp < 0 || !pool_ok(p->pool, p->page_bytes, p->pages) || !p->tables || !p->lengths || !p->new_tables || !p->map || !p->result)
		return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	const PageCompactArgs a{p->rows, p->pages, lp, p->table_ld, p->pool, p->page_bytes, p->tables, p->lengths, p->held, p->new_tables,
	                        p->map, p->result, workspace};
	return on_stream(stream, [&](hipStream_t s) { page_compact(a, s); });
}

sslm_status sslm_hip_cache_store(const sslm_hip_cache_store_args* p, void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const int lp = log2_page(p->page_tokens);
	if (lp < 0 || p->rows < 1 || p->rows > kMaxRows || p->tokens < 1 || p->max_new < 1 || p->max_new > p->tokens || p->max_new > SSLM_HIP_CACHE_MAX_WIDTH || p->pages < 1 ||
	    p->table_ld < 1 || p->table_ld > SSLM_HIP_CACHE_MAX_WIDTH / 16 || !heads_ok(p->heads, p->kv_heads, p->head_dim) || p->rope_dim < 0 ||
	    p->rope_dim % 8 || p->rope_dim > p->head_dim || !pool_ok(p->pool, p->page_bytes, p->pages) || !p->tables || !p->row_tokens ||
	    !p->row_start || !p->k || !p->v || !p->k_scale || !p->v_scale || !p->r_t_k || !p->e_t_k || !p->r_t_v || !p->e_t_v || !p->clamped || !p->status)
		return SSLM_INVALID_ARGUMENT;
	if (p->rope_dim && (!p->rope_cos || !p->rope_sin || p->rope_rows < 1 || p->rope_rows > SSLM_HIP_CACHE_MAX_WIDTH)) return SSLM_INVALID_ARGUMENT;
	const int64_t width = (int64_t)p->heads * p->head_dim, kv = (int64_t)p->kv_heads * p->head_dim;
	if (p->k_ld < kv || p->v_ld < kv || (p->q && (!p->q_out || p->q_ld < width || (p->q == p->q_out && p->q_ld != width))))
		return SSLM_INVALID_ARGUMENT;
	CacheStoreArgs a{};
	a.pg = Pages{p->pool, p->page_bytes, p->k_offset, p->v_offset, p->exp_offset, p->pages, lp, p->table_ld, p->kv_heads, p->head_dim, p->tables};
	if (!layer_ok(a.pg)) return SSLM_INVALID_ARGUMENT;
	a.rows = p->rows;
	a.tokens = p->tokens;
	a.max_new = p->max_new;
	a.NH = p->heads;
	a.rope_dim = p->rope_dim;
	a.halves = p->rope_halves != 0;
	a.row_tokens = p->row_tokens;
	a.row_start = p->row_start;
	a.rope_rows = p->rope_rows;
	a.rope_cos = p->rope_cos;
	a.rope_sin = p->rope_sin;
	a.q = p->q;
	a.k = p->k;
	a.v = p->v;
	a.q_ld = p->q_ld;
	a.k_ld = p->k_ld;
	a.v_ld = p->v_ld;
	a.k_scale = (const Scale*)p->k_scale;
	a.v_scale = (const Scale*)p->v_scale;
	a.r_t_k = p->r_t_k;
	a.e_t_k = p->e_t_k;
	a.r_t_v = p->r_t_v;
	a.e_t_v = p->e_t_v;
	a.q_out = p->q_out;
	a.clamped = p->clamped;
	a.status = p->status;
	return on_stream(stream, [&](hipStream_t s) { cache_store(a, s); });
}

size_t sslm_hip_cache_attention_workspace(int32_t rows, int32_t tokens, int32_t max_new, int32_t heads, int32_t kv_heads,
                                          int32_t head_dim, int32_t page_tokens, int64_t max_width) {
	const int lp = log2_page(page_tokens);
	if (lp < 0 || rows < 1 || rows > kMaxRows || tokens < 1 || max_new < 1 || max_new > tokens || !heads_ok(heads, kv_heads, head_dim) ||
	    max_width < 1 || max_width > SSLM_HIP_CACHE_MAX_WIDTH)
		return 0;
	return cache_attn_workspace(rows, tokens, max_new, heads, kv_heads, head_dim, max_width);
}

sslm_status sslm_hip_cache_attention(const sslm_hip_cache_attention_args* p, void* workspace, size_t workspace_bytes, void* stream) {
	if (!p || p->struct_size != sizeof(*p)) return SSLM_INVALID_ARGUMENT;
	const size_t need = sslm_hip_cache_attention_workspace(p->rows, p->tokens, p->max_new, p->heads, p->kv_heads, p->head_dim,
	                                                       p->page_tokens, p->max_width);
	if (!need || p->pages < 1 || p->table_ld < 1 || p->table_ld > SSLM_HIP_CACHE_MAX_WIDTH / 16 || !pool_ok(p->pool, p->page_bytes, p->pages) ||
	    !p->tables || !p->row_tokens || !p->row_start || !p->q || !p->q_scale || !p->khead_m || !p->khead_e || !p->ctx_fold || !p->codes ||
	    !p->scales || !p->status || (uintptr_t)p->q % 16)
		return SSLM_INVALID_ARGUMENT;
	CacheAttnArgs a{};
	a.pg = Pages{(int8_t*)p->pool, p->page_bytes, p->k_offset, p->v_offset, p->exp_offset, p->pages, log2_page(p->page_tokens), p->table_ld,
	             p->kv_heads, p->head_dim, p->tables};
	if (!layer_ok(a.pg)) return SSLM_INVALID_ARGUMENT;
	sslm_status st;
	if (!workspace_ok(workspace, workspace_bytes, need, &st)) return st;
	a.rows = p->rows;
	a.tokens = p->tokens;
	a.max_new = p->max_new;
	a.NH = p->heads;
	a.max_width = p->max_width;
	a.row_tokens = p->row_tokens;
	a.row_start = p->row_start;
	a.q = p->q;
	a.q_scale = (const Scale*)p->q_scale;
	a.khead_m = p->khead_m;
	a.khead_e = p->khead_e;
	a.ln2_q = p->ln2_q;
	a.b_q = p->b_q;
	a.ca_q = p->ca_q;
	a.ctx_fold = p->ctx_fold;
	a.site = Scale{p->site_m, p->site_e};
	a.codes = p->codes;
	a.scales = (Scale*)p->scales;
	a.status = p->status;
	a.ws = workspace;
	return on_stream(stream, [&](hipStream_t s) { cache_attn(a, s); });
}

}  // extern "C"
