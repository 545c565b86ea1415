// The operators of a decode step whose rows are different requests, as a serving loop runs them: a batch's
// attention, the projection that takes its codes and scales, and the pick, enqueued one behind the other.
// Two batches at once, each with workspaces of its own: on two non-blocking streams eagerly, as two captured
// graphs, and as the two branches of one graph.  The inputs change in place between replays, with eager work
// of other workspaces and synchronizations between; every result must equal the eager one on the default
// stream, bit for bit.  Prints "ok" on success.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

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
#define OK(x)                                                      \
	do {                                                           \
		const sslm_status s_ = (x);                                \
		if (s_ != SSLM_OK) {                                       \
			printf("status %d at line %d\n", (int)s_, __LINE__);   \
			exit(1);                                               \
		}                                                          \
	} while (0)

static uint64_t g_s = 12345;
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

static void codes(Buf<int8_t>& b) {
	for (auto& v : b.h) v = (int8_t)(below(255) - 127);
	b.up();
}
// fold entries: identity now and then, multiplier in [2^30, 2^31), exponent in [lo, hi)
static void folds(Buf<int32_t>& b, int lo, int hi) {
	for (size_t j = 0; j < b.h.size() / 3; ++j) {
		b.h[3 * j] = below(16) == 0;
		b.h[3 * j + 1] = (1 << 30) + below(1 << 30);
		b.h[3 * j + 2] = lo + below(hi - lo);
	}
	b.up();
}

struct Out {
	Buf<int8_t> ctx, proj;
	Buf<int64_t> ctx_scale, proj_scale;
	Buf<int32_t> ctx_status, proj_status, adjusted, tokens;
	Buf<uint8_t> ws[3];
	void make(int rows, int h, int n, int vocab, const size_t* bytes) {
		ctx.make((size_t)rows * h), proj.make((size_t)rows * n);
		ctx_scale.make(rows * 2), proj_scale.make(rows * 2);
		ctx_status.make(rows), proj_status.make(rows), tokens.make(rows), adjusted.make((size_t)rows * vocab);
		for (int i = 0; i < 3; ++i) ws[i].make(bytes[i]);
	}
	void spoil() {
		auto s = [](auto& b, int v) { CK(hipMemset(b.d, v, b.h.size() * sizeof(b.h[0]))); };
		s(ctx, 0x55), s(proj, 0x55), s(adjusted, 0x55), s(tokens, 0x55), s(proj_status, 0x55), s(ctx_status, 0x55);
		// a refused row keeps its scale, which the projection then reads: any valid one
		std::fill(ctx_scale.h.begin(), ctx_scale.h.end(), 0);
		for (size_t i = 0; i < ctx_scale.h.size(); i += 2) ctx_scale.h[i] = 1 << 30, ctx_scale.h[i + 1] = -37;
		ctx_scale.up();
		s(proj_scale, 0x55);
		for (auto& w : ws) s(w, 0xA5);
		CK(hipDeviceSynchronize());
	}
	void down() { ctx.down(), proj.down(), ctx_scale.down(), proj_scale.down(), ctx_status.down(), proj_status.down(), adjusted.down(), tokens.down(); }
	bool same(const Out& o) const {
		return ctx.h == o.ctx.h && proj.h == o.proj.h && ctx_scale.h == o.ctx_scale.h && proj_scale.h == o.proj_scale.h &&
		       ctx_status.h == o.ctx_status.h && proj_status.h == o.proj_status.h && adjusted.h == o.adjusted.h && tokens.h == o.tokens.h;
	}
};

struct Batch {
	int rows, heads, kv, dim, prefixes, n, vocab, adapters;
	int64_t longest, own, cap;
	size_t bytes[3];
	Buf<int8_t> pool, q, w;
	std::vector<Buf<int8_t>> la, lb;
	std::vector<Buf<int32_t>> lu, ld;
	Buf<int64_t> q_scale, km, ke, width, plen;
	Buf<int32_t> cfold, fold, row_block, prow, pblock, row_adapter, logits, history, bias_ids, bias_values;
	Buf<uint8_t> mask;
	Buf<sslm_hip_lora> lora;
	Buf<sslm_hip_logit_rule> rules;
	Out out, ref;

	int h() const { return heads * dim; }
	int blocks() const { return rows + prefixes; }
	void make() {
		cap = longest + own + 1;
		pool.make((size_t)blocks() * 2 * kv * cap * dim), q.make((size_t)rows * h()), w.make((size_t)n * h());
		q_scale.make(rows * 2), km.make(kv), ke.make(kv), width.make(rows), plen.make(prefixes);
		cfold.make(heads * 3), fold.make(n * 3), row_block.make(rows), prow.make(prefixes + 1), pblock.make(prefixes), row_adapter.make(rows);
		logits.make((size_t)rows * vocab), history.make(rows * 40), bias_ids.make(rows * 9), bias_values.make(rows * 9), mask.make((size_t)rows * ((vocab + 7) / 8));
		lora.make(adapters), rules.make(rows), la.resize(adapters), lb.resize(adapters), lu.resize(adapters), ld.resize(adapters);
		for (int i = 0; i < adapters; ++i) {
			const int rank = 1 + i * 17 % 64;
			la[i].make((size_t)rank * h()), lb[i].make((size_t)n * rank), lu[i].make(rank * 3), ld[i].make(n * 3);
			lora.h[i] = sslm_hip_lora{la[i].d, lu[i].d, lb[i].d, ld[i].d, rank, 0};
		}
		lora.up();
		bytes[0] = sslm_hip_shared_attention_workspace(rows, heads, kv, dim, prefixes, longest, own);
		bytes[1] = sslm_hip_gemm_lora_workspace(rows, n, h());
		bytes[2] = sslm_hip_pick_workspace(rows, vocab);
		if (!bytes[0] || !bytes[1] || !bytes[2]) {
			printf("a workspace of no bytes\n");
			exit(1);
		}
		out.make(rows, h(), n, vocab, bytes), ref.make(rows, h(), n, vocab, bytes);
	}
	void fill() {
		codes(pool), codes(q), codes(w);
		for (int i = 0; i < adapters; ++i) codes(la[i]), codes(lb[i]), folds(lu[i], 13, 16), folds(ld[i], -3, 9);
		folds(cfold, 0, 3), folds(fold, 0, 12);
		for (int i = 0; i < rows; ++i) q_scale.h[2 * i] = (1 << 30) + below(1 << 30), q_scale.h[2 * i + 1] = -37;
		for (int i = 0; i < kv; ++i) km.h[i] = (1 << 30) + below(1 << 30), ke.h[i] = -39;
		for (int p = 0; p < prefixes; ++p) plen.h[p] = longest - below((int)longest / 2 + 1), pblock.h[p] = rows + p;
		for (int p = 0; p <= prefixes; ++p) prow.h[p] = (rows - 1) * p / prefixes;  // the last row has none
		for (int i = 0; i < rows; ++i) {
			int p = 0;
			while (p < prefixes && i >= prow.h[p + 1]) ++p;
			row_block.h[i] = rows - 1 - i;
			width.h[i] = (p < prefixes ? plen.h[p] : 0) + below((int)own + 1);
			row_adapter.h[i] = below(adapters + 1) - 1;
		}
		for (auto& v : logits.h) v = below(1 << 20) - (1 << 19);
		for (auto& v : history.h) v = below(vocab);
		for (auto& v : bias_ids.h) v = below(vocab);
		for (auto& v : bias_values.h) v = below(1 << 21) - (1 << 20);
		for (auto& v : mask.h) v = (uint8_t)below(256);
		for (int i = 0; i < rows; ++i)
			rules.h[i] = sslm_hip_logit_rule{history.d + i * 40, bias_ids.d + i * 9, bias_values.d + i * 9, i % 3 ? mask.d + (size_t)i * ((vocab + 7) / 8) : nullptr,
			                                 below(41), below(10), 65536 + below(65536), below(1000), below(1000), 0};
		q_scale.up(), km.up(), ke.up(), plen.up(), pblock.up(), prow.up(), row_block.up(), width.up(), row_adapter.up();
		logits.up(), history.up(), bias_ids.up(), bias_values.up(), mask.up(), rules.up();
	}
	void enqueue(Out& o, hipStream_t s) {
		sslm_hip_shared_attention_args a{};
		a.struct_size = sizeof(a);
		a.rows = rows, a.heads = heads, a.kv_heads = kv, a.head_dim = dim, a.prefixes = prefixes, a.blocks = blocks();
		a.max_prefix = longest, a.max_own = own;
		a.kv_pool = pool.d, a.block_bytes = 2 * (int64_t)kv * cap * dim, a.v_offset = (int64_t)kv * cap * dim, a.cap = cap;
		a.q = q.d, a.q_scale = q_scale.d, a.khead_m = km.d, a.khead_e = ke.d;
		a.ln2_q = 744261117, a.b_q = 1452772687, a.ca_q = 1030312935;
		a.ctx_fold = cfold.d, a.site_m = 1518500250, a.site_e = -45;
		a.row_block = row_block.d, a.row_width = width.d, a.prefix_rows = prow.d, a.prefix_block = pblock.d, a.prefix_len = plen.d;
		a.codes = o.ctx.d, a.scales = o.ctx_scale.d, a.status = o.ctx_status.d;
		OK(sslm_hip_shared_attention(&a, o.ws[0].d, bytes[0], s));
		sslm_hip_gemm_lora_args g{};
		g.struct_size = sizeof(g);
		g.m = rows, g.n = n, g.k = h(), g.adapter_count = adapters;
		g.a = o.ctx.d, g.w = w.d, g.fold = fold.d, g.in_scale = o.ctx_scale.d, g.site_m = a.site_m, g.site_e = a.site_e;
		g.adapters = lora.d, g.row_adapter = row_adapter.d, g.codes = o.proj.d, g.scales = o.proj_scale.d, g.status = o.proj_status.d;
		OK(sslm_hip_gemm_lora_requant(&g, o.ws[1].d, bytes[1], s));
		sslm_hip_pick_args p{};
		p.struct_size = sizeof(p);
		p.rows = rows, p.vocab = vocab, p.logits = logits.d, p.logits_ld = p.adjusted_ld = vocab;
		p.rules = rules.d, p.adjusted = o.adjusted.d, p.tokens = o.tokens.d;
		OK(sslm_hip_pick_tokens(&p, o.ws[2].d, bytes[2], s));
	}
	// against the eager call on the default stream
	int check(const char* what, int round) {
		out.down();
		if (!out.same(ref)) {
			printf("%s, round %d: differs from the eager call\n", what, round);
			exit(1);
		}
		return (int)std::count(ref.ctx_status.h.begin(), ref.ctx_status.h.end(), 0) + (int)std::count(ref.proj_status.h.begin(), ref.proj_status.h.end(), 0);
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
	Batch b[2];
	// rows cut over the chip, a projection by GEMM and whole rows; and the small forms of all three
	b[0].rows = 70, b[0].heads = 12, b[0].kv = 2, b[0].dim = 128, b[0].prefixes = 3, b[0].n = 1536, b[0].vocab = 9001, b[0].adapters = 5;
	b[0].longest = 700, b[0].own = 90;
	b[1].rows = 9, b[1].heads = 8, b[1].kv = 4, b[1].dim = 64, b[1].prefixes = 2, b[1].n = 256, b[1].vocab = 500, b[1].adapters = 2;
	b[1].longest = 60, b[1].own = 20;
	hipStream_t s[2];
	hipEvent_t fork, join;
	CK(hipEventCreateWithFlags(&fork, hipEventDisableTiming));
	CK(hipEventCreateWithFlags(&join, hipEventDisableTiming));
	for (int i = 0; i < 2; ++i) {
		b[i].make();
		CK(hipStreamCreateWithFlags(&s[i], hipStreamNonBlocking));
	}
	hipGraphExec_t one[2], both;
	for (int i = 0; i < 2; ++i) one[i] = capture(s[i], [&] { b[i].enqueue(b[i].out, s[i]); });
	both = capture(s[0], [&] {
		CK(hipEventRecord(fork, s[0]));
		CK(hipStreamWaitEvent(s[1], fork, 0));
		for (int i = 0; i < 2; ++i) b[i].enqueue(b[i].out, s[i]);
		CK(hipEventRecord(join, s[1]));
		CK(hipStreamWaitEvent(s[0], join, 0));
	});
	int live = 0;
	for (int round = 0; round < 4; ++round) {
		for (auto& x : b) {
			x.fill();
			x.ref.spoil();
			x.enqueue(x.ref, nullptr);
			CK(hipDeviceSynchronize());
			x.ref.down();
		}
		for (int how = 0; how < 3; ++how) {
			for (auto& x : b) x.out.spoil();
			if (how == 0)
				for (int i = 0; i < 2; ++i) b[i].enqueue(b[i].out, s[i]);
			else if (how == 1)
				for (int i = 0; i < 2; ++i) CK(hipGraphLaunch(one[i], s[i]));
			else
				CK(hipGraphLaunch(both, s[0]));
			b[1].enqueue(b[1].ref, nullptr);  // beside them, with its own workspaces and outputs
			CK(hipDeviceSynchronize());
			const char* name[] = {"streams", "graphs", "branches"};
			for (auto& x : b) live += x.check(name[how], round);
		}
		printf("round %d\n", round);
		fflush(stdout);
	}
	if (live < 4 * 3 * 79) {  // at least half of the rows of both operators computed
		printf("only %d rows of results: the check would say little\n", live);
		return 1;
	}
	printf("ok (%d rows)\n", live);
	return 0;
}
