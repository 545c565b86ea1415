// A cache in pages: its pages' changes of hands, the landing of new tokens, attention over it (cache_ops.hip); and
// the next token by sampling (sample.hip).
#pragma once

#include "kernels.h"

namespace sslm_launch {
using namespace sslm;

constexpr int kMaxShift = 8;                       // a page's largest exponent
constexpr int32_t kMaxUnits = 127 << kMaxShift;    // and the largest value it holds

// One layer's view of the pages and the rows' tables.
struct Pages {
	int8_t* pool;
	int64_t page_bytes, k_off, v_off, e_off;
	int32_t pages, lp, table_ld, NKV, D;  // lp: log2 of a page's positions
	const int32_t* tables;
};

struct PageUpdateArgs {
	int rows, pages, lp, table_ld;
	int8_t* pool;
	int64_t page_bytes;
	const int32_t* tables;
	const int64_t* lengths;
	const int32_t* source;
	const int64_t *keep, *room;
	const uint8_t* held;
	int32_t* new_tables;
	int64_t* new_lengths;
	int32_t* result;
	void* ws;
};
size_t page_update_workspace(int rows, int pages, int table_ld);
void page_update(const PageUpdateArgs& a, hipStream_t s);

struct PageCompactArgs {
	int rows, pages, lp, table_ld;
	int8_t* pool;
	int64_t page_bytes;
	const int32_t* tables;
	const int64_t* lengths;
	const uint8_t* held;
	int32_t *new_tables, *map, *result;
	void* ws;
};
size_t page_compact_workspace(int rows, int pages, int table_ld);
void page_compact(const PageCompactArgs& a, hipStream_t s);

struct CacheStoreArgs {
	Pages pg;
	int rows, tokens, max_new, NH, rope_dim, halves;
	const int32_t* row_tokens;
	const int64_t* row_start;
	int64_t rope_rows;
	const int64_t *rope_cos, *rope_sin;
	const int8_t *q, *k, *v;
	int64_t q_ld, k_ld, v_ld;
	const Scale *k_scale, *v_scale;
	const int64_t *r_t_k, *e_t_k, *r_t_v, *e_t_v;
	int8_t* q_out;
	int32_t *clamped, *status;
};
void cache_store(const CacheStoreArgs& a, hipStream_t s);

struct CacheAttnArgs {
	Pages pg;
	int rows, tokens, max_new, NH;
	int64_t max_width;
	const int32_t* row_tokens;
	const int64_t* row_start;
	const int8_t* q;
	const Scale* q_scale;
	const int64_t *khead_m, *khead_e;
	int64_t ln2_q, b_q, ca_q;
	const int32_t* ctx_fold;
	Scale site;
	int8_t* codes;
	Scale* scales;
	int32_t* status;
	void* ws;
};
size_t cache_attn_workspace(int rows, int tokens, int max_new, int NH, int NKV, int D, int64_t max_width);
void cache_attn(const CacheAttnArgs& a, hipStream_t s);

struct Sampling {
	const uint8_t* mask;
	int64_t q_ln2, q_b, q_c;
	int32_t top_k, top_p, min_p;
	uint32_t random;
};
struct SampleArgs {
	int rows, vocab;
	const int32_t* logits;
	int64_t ld;
	const Sampling* rules;
	int32_t* tokens;
	int64_t* mass;
	void* ws;
};
size_t sample_workspace(int rows, int vocab);
void sample_tokens(const SampleArgs& a, hipStream_t s);

}  // namespace sslm_launch
