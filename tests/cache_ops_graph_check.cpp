// The paged cache's operators and sampling as a serving loop runs them: pages change hands, the new tokens land and
// are attended to, the next tokens are drawn, enqueued one behind the other.  Two batches at once, each with
// workspaces of its own: on two non-blocking streams eagerly, as two captured graphs, and as the two branches of one graph.
// The inputs change in place between replays, with eager work of other workspaces and synchronizations between;
// every result must equal the eager one on the default stream, bit for bit.  Prints "ok" on success.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <vector>

#include "../include/sslm_hip.h"

#define CK(x)                                                                     \
	do {                                                                          \
		hipError_t e_ = (x);                                                      \
		if (e_ != hipSuccess) {                                                   \
			printf("HIP error %s at line %d\n", hipGetErrorString(e_), __LINE__); \
			exit(1);                                                              \
		}                                                                         \
	} while (0)
#define OK(x)                                                    \
	do {                                                         \
		const sslm_status s_ = (x);                              \
		if (s_ != SSLM_OK) {                                     \
			printf("status %d at line %d\n", (int)s_, __LINE__); \
			exit(1);                                             \
		}                                                        \
	} while (0)

static uint64_t g_s = 4242;
static uint32_t rnd() {
	g_s = g_s * 6364136223846793005ull + 1442695040888963407ull;
	return (uint32_t)(g_s >> 33);
}
static int below(int n) { return (int)(rnd() % (uint32_t)n); }

template <typename T>
struct Buf {
	T* d = nullptr;
	std::vector<T> h;
	void make(size_t n) {
		h.assign(n, T());
		CK(hipMalloc(&d, n * sizeof(T)));
	}
	void up() { CK(hipMemcpy(d, h.data(), h.size() * sizeof(T), hipMemcpyHostToDevice)); }
	void down() { CK(hipMemcpy(h.data(), d, h.size() * sizeof(T), hipMemcpyDeviceToHost)); }
};

// what a step changes or writes, and its workspaces
struct Out {
	Buf<int8_t> pool, q, ctx;
	Buf<int32_t> tables, result, clamped, store_status, status, tokens, map;
	Buf<int64_t> lengths, scales, mass;
	Buf<uint8_t> ws[4];
	bool same(const Out& o) const {
		return pool.h == o.pool.h && q.h == o.q.h && ctx.h == o.ctx.h && tables.h == o.tables.h && result.h == o.result.h && clamped.h == o.clamped.h &&
		       store_status.h == o.store_status.h && status.h == o.status.h && tokens.h == o.tokens.h && lengths.h == o.lengths.h && scales.h == o.scales.h &&
		       mass.h == o.mass.h && map.h == o.map.h;
	}
	void down() {
		pool.down(), q.down(), ctx.down(), tables.down(), result.down(), clamped.down(), store_status.down(), status.down(), tokens.down(), lengths.down();
		scales.down(), mass.down(), map.down();
	}
};

struct Batch {
	int rows, heads, kv, dim, page, pages, width, vocab, most;  // most: new tokens of a row at the most
	int64_t page_bytes;
	size_t bytes[4] = {};
	Buf<int8_t> pool, q, k, v;
	Buf<int32_t> tables, source, cuts, fold, logits;
	Buf<int64_t> lengths, keep, room, cos, sin, ks, vs, rk, ek, rv, ev, q_scale, km, ke;
	Buf<uint8_t> mask;
	Buf<sslm_hip_sampling> rules;
	Out out, ref;
	int tokens() const { return rows * most; }
	void make() {
		const size_t half = (size_t)kv * page * dim;
		page_bytes = (int64_t)((2 * half + 2 * kv + 15) / 16 * 16);
		pool.make((size_t)pages * page_bytes), q.make((size_t)tokens() * heads * dim), k.make((size_t)tokens() * kv * dim), v.make((size_t)tokens() * kv * dim);
		tables.make((size_t)rows * width), source.make(rows), cuts.make(rows + 1), fold.make(heads * 3), logits.make((size_t)rows * vocab);
		lengths.make(rows), keep.make(rows), room.make(rows), cos.make((size_t)width * page * dim / 2), sin.make((size_t)width * page * dim / 2);
		ks.make(2 * tokens()), vs.make(2 * tokens()), rk.make(kv), ek.make(kv), rv.make(kv), ev.make(kv), q_scale.make(2 * tokens()), km.make(kv), ke.make(kv);
		mask.make((size_t)rows * ((vocab + 7) / 8)), rules.make(rows);
		bytes[0] = sslm_hip_cache_update_workspace(rows, pages, width);
		bytes[1] = sslm_hip_cache_attention_workspace(rows, tokens(), most, heads, kv, dim, page, (int64_t)width * page);
		bytes[2] = sslm_hip_sample_workspace(rows, vocab);
		bytes[3] = sslm_hip_cache_compact_workspace(rows, pages, width);
		for (Out* o : {&out, &ref}) {
			o->pool.make(pool.h.size()), o->q.make(q.h.size()), o->ctx.make(q.h.size()), o->tables.make(tables.h.size()), o->result.make(8), o->clamped.make(rows);
			o->store_status.make(rows), o->status.make(tokens()), o->tokens.make(rows), o->lengths.make(rows), o->scales.make(2 * tokens()), o->mass.make(2 * rows);
			o->map.make(pages);
			for (int i = 0; i < 4; ++i) {
				if (!bytes[i]) {
					printf("a workspace of no bytes\n");
					exit(1);
				}
				o->ws[i].make(bytes[i]);
			}
		}
	}
	// rows of random lengths, some of which then fork, grow or end
	void fill() {
		for (auto* b : {&pool, &q, &k, &v}) {
			for (auto& x : b->h) x = (int8_t)(below(255) - 127);
			b->up();
		}
		const size_t half = (size_t)kv * page * dim;
		for (int p = 0; p < pages; ++p)
			for (int i = 0; i < 2 * kv; ++i) pool.h[p * page_bytes + 2 * half + i] = (int8_t)below(5);
		pool.up();
		std::vector<int> order(pages);
		for (int i = 0; i < pages; ++i) order[i] = i;
		for (int i = pages - 1; i > 0; --i) std::swap(order[i], order[below(i + 1)]);
		int used = 0;
		std::fill(tables.h.begin(), tables.h.end(), -1);
		for (int r = 0; r < rows; ++r) {
			lengths.h[r] = below((width - 2) * page / 2);
			for (int i = 0; i * page < lengths.h[r]; ++i) tables.h[(size_t)r * width + i] = order[used++];
		}
		cuts.h[0] = 0;
		for (int r = 0; r < rows; ++r) {
			const int s = below(8) == 0 ? -1 : (below(3) ? r : below(rows));
			source.h[r] = s;
			keep.h[r] = s < 0 ? 0 : (below(4) ? lengths.h[s] : lengths.h[s] / 2);
			const int n = most == 1 ? 1 : below(most + 1);
			room.h[r] = keep.h[r] + n;
			cuts.h[r + 1] = cuts.h[r] + n;
		}
		for (size_t i = 0; i < cos.h.size(); ++i) {
			const int a = below(1 << 15);  // any rotation: (1 - t^2, 2 t) / (1 + t^2)
			const double t = a / 32768.0;
			cos.h[i] = (int64_t)((1 - t * t) / (1 + t * t) * (1 << 30));
			sin.h[i] = (int64_t)(2 * t / (1 + t * t) * (1 << 30));
		}
		auto scale = [](Buf<int64_t>& b, int e, int spread) {
			for (size_t i = 0; i < b.h.size(); i += 2) b.h[i] = (1 << 30) + below(1 << 30), b.h[i + 1] = e - below(spread);
			b.up();
		};
		scale(ks, -36, 4), scale(vs, -36, 4), scale(q_scale, -36, 3);
		for (int i = 0; i < kv; ++i) {
			rk.h[i] = (1ll << 31) + below(1 << 30), rv.h[i] = (1ll << 31) + below(1 << 30);
			ek.h[i] = ev.h[i] = -41;
			km.h[i] = (1 << 30) + below(1 << 30), ke.h[i] = -43;
		}
		for (int i = 0; i < heads; ++i) fold.h[3 * i] = 0, fold.h[3 * i + 1] = (1 << 30) + below(1 << 30), fold.h[3 * i + 2] = below(6);
		for (auto& x : logits.h) x = below(1 << 19) + below(1 << 19) - (1 << 19);
		for (auto& x : mask.h) x = (uint8_t)below(256);
		for (int r = 0; r < rows; ++r) {
			const int64_t unit = 20000 + below(40000);
			rules.h[r] = sslm_hip_sampling{r % 3 ? nullptr : mask.d + (size_t)r * ((vocab + 7) / 8), unit * 69 / 100, unit * 135 / 100, unit * unit / 100 * 96,
			                               r % 2 ? below(300) : 0, r % 3 == 1 ? 65536 : 40000 + below(25000), r % 4 == 2 ? below(5000) : 0, rnd() * 2 + 1};
		}
		tables.up(), lengths.up(), source.up(), keep.up(), room.up(), cuts.up(), cos.up(), sin.up(), rk.up(), rv.up(), ek.up(), ev.up(), km.up(), ke.up();
		fold.up(), logits.up(), mask.up(), rules.up();
	}
	void reset(Out& o) {
		auto s = [](auto& b) { CK(hipMemset(b.d, 0x55, b.h.size() * sizeof(b.h[0]))); };
		s(o.q), s(o.ctx), s(o.result), s(o.clamped), s(o.store_status), s(o.status), s(o.tokens), s(o.mass), s(o.map);
		// tokens that no row has keep their scales, which the pool's rows then have to be: any
		s(o.scales);
		for (auto& w : o.ws) CK(hipMemset(w.d, 0xA5, w.h.size()));
		CK(hipMemcpy(o.pool.d, pool.d, pool.h.size(), hipMemcpyDeviceToDevice));
		CK(hipMemcpy(o.tables.d, tables.d, tables.h.size() * 4, hipMemcpyDeviceToDevice));
		CK(hipMemcpy(o.lengths.d, lengths.d, lengths.h.size() * 8, hipMemcpyDeviceToDevice));
		CK(hipDeviceSynchronize());
	}
	void enqueue(Out& o, hipStream_t s) {
		const int64_t half = (int64_t)kv * page * dim;
		sslm_hip_cache_update_args u{};
		u.struct_size = sizeof(u);
		u.rows = rows, u.pages = pages, u.page_tokens = page, u.table_ld = width, u.pool = o.pool.d, u.page_bytes = page_bytes;
		u.tables = u.new_tables = o.tables.d, u.lengths = u.new_lengths = o.lengths.d;
		u.source = source.d, u.keep = keep.d, u.room = room.d, u.result = o.result.d;
		OK(sslm_hip_cache_update(&u, o.ws[0].d, bytes[0], s));
		sslm_hip_cache_store_args t{};
		t.struct_size = sizeof(t);
		t.rows = rows, t.tokens = tokens(), t.max_new = most, t.heads = heads, t.kv_heads = kv, t.head_dim = dim, t.pages = pages, t.page_tokens = page;
		t.table_ld = width, t.rope_dim = dim, t.rope_halves = most > 1, t.pool = o.pool.d, t.page_bytes = page_bytes, t.v_offset = half, t.exp_offset = 2 * half;
		t.tables = o.tables.d, t.row_tokens = cuts.d, t.row_start = keep.d, t.rope_rows = (int64_t)width * page, t.rope_cos = cos.d, t.rope_sin = sin.d;
		t.q = q.d, t.k = k.d, t.v = v.d, t.q_ld = heads * dim, t.k_ld = t.v_ld = kv * dim, t.k_scale = ks.d, t.v_scale = vs.d;
		t.r_t_k = rk.d, t.e_t_k = ek.d, t.r_t_v = rv.d, t.e_t_v = ev.d, t.q_out = o.q.d, t.clamped = o.clamped.d, t.status = o.store_status.d;
		OK(sslm_hip_cache_store(&t, s));
		sslm_hip_cache_attention_args a{};
		a.struct_size = sizeof(a);
		a.rows = rows, a.tokens = tokens(), a.max_new = most, a.heads = heads, a.kv_heads = kv, a.head_dim = dim, a.pages = pages, a.page_tokens = page;
		a.table_ld = width, a.max_width = (int64_t)width * page, a.pool = o.pool.d, a.page_bytes = page_bytes, a.v_offset = half, a.exp_offset = 2 * half;
		a.tables = o.tables.d, a.row_tokens = cuts.d, a.row_start = keep.d, a.q = o.q.d, a.q_scale = q_scale.d, a.khead_m = km.d, a.khead_e = ke.d;
		a.ln2_q = 744261117, a.b_q = 1452772687, a.ca_q = 1030312935, a.ctx_fold = fold.d, a.site_m = 1518500250, a.site_e = -45;
		a.codes = o.ctx.d, a.scales = o.scales.d, a.status = o.status.d;
		OK(sslm_hip_cache_attention(&a, o.ws[1].d, bytes[1], s));
		sslm_hip_sample_args p{};
		p.struct_size = sizeof(p);
		p.rows = rows, p.vocab = vocab, p.logits = logits.d, p.logits_ld = vocab, p.rules = rules.d, p.tokens = o.tokens.d, p.mass = o.mass.d;
		OK(sslm_hip_sample_tokens(&p, o.ws[2].d, bytes[2], s));
		sslm_hip_cache_compact_args c{};
		c.struct_size = sizeof(c);
		c.rows = rows, c.pages = pages, c.page_tokens = page, c.table_ld = width, c.pool = o.pool.d, c.page_bytes = page_bytes, c.tables = c.new_tables = o.tables.d;
		c.lengths = o.lengths.d, c.map = o.map.d, c.result = o.result.d + 4;
		OK(sslm_hip_cache_compact(&c, o.ws[3].d, bytes[3], s));
	}
	// against the eager call on the default stream
	int check(const char* what, int round) {
		out.down();
		if (!out.same(ref)) {
			printf("%s, round %d: differs from the eager call\n", what, round);
			exit(1);
		}
		if (ref.result.h[0] != 0 || ref.result.h[4] != 0) {
			printf("round %d: pages refused (%d, %d)\n", round, ref.result.h[0], ref.result.h[4]);
			exit(1);
		}
		return (int)std::count(ref.status.h.begin(), ref.status.h.begin() + cuts.h[rows], 0) + (int)std::count_if(ref.tokens.h.begin(), ref.tokens.h.end(), [](int x) { return x >= 0; });
	}
};

template <typename F>
static hipGraphExec_t capture(hipStream_t s, F&& enqueue) {
	hipGraph_t g;
	hipGraphExec_t x;
	CK(hipStreamBeginCapture(s, hipStreamCaptureModeThreadLocal));
	enqueue();
	CK(hipStreamEndCapture(s, &g));
	CK(hipGraphInstantiate(&x, g, nullptr, nullptr, 0));
	CK(hipGraphDestroy(g));
	return x;
}

int main() {
	Batch b[3];
	// chunks of several rows over a vocabulary of several slices; single tokens of short rows; single tokens of long rows, by planes
	b[0].rows = 9, b[0].heads = 12, b[0].kv = 2, b[0].dim = 64, b[0].page = 32, b[0].pages = 400, b[0].width = 24, b[0].vocab = 40000, b[0].most = 50;
	b[1].rows = 30, b[1].heads = 8, b[1].kv = 4, b[1].dim = 32, b[1].page = 16, b[1].pages = 900, b[1].width = 20, b[1].vocab = 3000, b[1].most = 1;
	b[2].rows = 4, b[2].heads = 12, b[2].kv = 2, b[2].dim = 128, b[2].page = 64, b[2].pages = 300, b[2].width = 60, b[2].vocab = 9000, b[2].most = 1;
	int live = 0, want = 0;
	for (int pair = 0; pair < 2; ++pair) {
		Batch* x[2] = {&b[pair], &b[pair + 1]};
		hipStream_t s[2];
		hipEvent_t fork, join;
		CK(hipEventCreateWithFlags(&fork, hipEventDisableTiming));
		CK(hipEventCreateWithFlags(&join, hipEventDisableTiming));
		for (int i = 0; i < 2; ++i) {
			if (!x[i]->bytes[0]) x[i]->make();
			CK(hipStreamCreateWithFlags(&s[i], hipStreamNonBlocking));
		}
		hipGraphExec_t one[2], both;
		for (int i = 0; i < 2; ++i) one[i] = capture(s[i], [&] { x[i]->enqueue(x[i]->out, s[i]); });
		both = capture(s[0], [&] {
			CK(hipEventRecord(fork, s[0]));
			CK(hipStreamWaitEvent(s[1], fork, 0));
			for (int i = 0; i < 2; ++i) x[i]->enqueue(x[i]->out, s[i]);
			CK(hipEventRecord(join, s[1]));
			CK(hipStreamWaitEvent(s[0], join, 0));
		});
		for (int round = 0; round < 3; ++round) {
			for (auto* y : x) {
				y->fill();
				y->reset(y->ref);
				y->enqueue(y->ref, nullptr);
				CK(hipDeviceSynchronize());
				y->ref.down();
			}
			for (int how = 0; how < 3; ++how) {
				for (auto* y : x) y->reset(y->out);
				if (how == 0)
					for (int i = 0; i < 2; ++i) x[i]->enqueue(x[i]->out, s[i]);
				else if (how == 1)
					for (int i = 0; i < 2; ++i) CK(hipGraphLaunch(one[i], s[i]));
				else
					CK(hipGraphLaunch(both, s[0]));
				CK(hipDeviceSynchronize());
				const char* name[] = {"streams", "graphs", "branches"};
				for (auto* y : x) {
					live += y->check(name[how], round);
					want += y->cuts.h[y->rows] + y->rows;
				}
			}
			printf("pair %d round %d\n", pair, round);
			fflush(stdout);
		}
	}
	if (live * 10 < want * 9) {  // nearly all tokens computed
		printf("only %d of %d results: the check would say little\n", live, want);
		return 1;
	}
	printf("ok (%d of %d)\n", live, want);
	return 0;
}
