// Operators of a decode step whose rows differ: attention of rows that share prompts, a projection
// with an adapter of its own per row, and the next token under each row's own rules (batch_ops.hip).
#pragma once

#include "kernels.h"

namespace sslm_launch {
using namespace sslm;

// Decode attention of `rows` rows, row r at position row_width[r] - 1 of its context.  Positions
// below its prefix's length lie in the prefix's KV block, the others in its own, each at its own
// position.  Rows [prefix_rows[p], prefix_rows[p + 1]) have prefix p, all others none.
struct SharedAttnArgs {
	int rows, NH, NKV, D, prefixes, blocks;
	int64_t max_prefix, max_own;  // at least every prefix's length, every row's own positions
	const int8_t* pool;
	int64_t block_bytes, k_off, v_off, cap;  // K and V of (KV head, position): block + off + (head cap + position) D
	const int8_t* q;                         // [rows, NH D] rotated codes
	const Scale* q_scale;                    // [rows]
	const int64_t *khead_m, *khead_e;        // [NKV]
	int64_t ln2_q, b_q, ca_q;
	const int32_t* ctx_fold;  // [NH, 3]
	Scale site;
	const int32_t* row_block;
	const int64_t* row_width;
	const int32_t *prefix_rows, *prefix_block;
	const int64_t* prefix_len;
	int8_t* codes;    // [rows, NH D]
	Scale* scales;    // [rows]
	int32_t* status;  // [rows]; with `tok` the slots' status words instead
	// a model's decode step: a row whose slot holds a refusal is left alone, its own refusal is reported as
	// `layer`'s (set_status).  Null: status[r] of every row is written.
	const TokenInfo* tok;
	int32_t layer;
	void* ws;         // shared_attn_workspace() bytes
};
size_t shared_attn_workspace(int rows, int NH, int NKV, int D, int prefixes, int64_t max_prefix, int64_t max_own);
bool shared_attn_ok(int rows, int NH, int NKV, int D);
void shared_attn(const SharedAttnArgs& a, hipStream_t s);
// Whether a decode unit whose rows have adopted prompts takes it.
struct SharedUnit {
	int rows, NH, NKV, D;
	int64_t width;         // the most positions of a row
	int64_t adopted, own;  // positions in the rows' prompts and past them, of all rows together
	bool per_head;         // otherwise one block per query head runs for want of the fused launch or of LDS for the scores
};
bool shared_attn_pays(const SharedUnit& u, int cus);

// A projection of m rows, row t with adapter row_adapter[t] (negative: none) and incoming scale in_scale[t].
struct LoraGemmArgs {
	int m, n, k, count;
	const int8_t *a, *w;
	const int32_t* fold;
	const Scale* in_scale;
	Scale site;
	const LoraRef* adapters;
	const int32_t* row_adapter;
	int8_t* codes;
	Scale* scales;
	int32_t* status;
	void* ws;  // lora_gemm_workspace() bytes
};
size_t lora_gemm_workspace(int m, int n, int k);
void lora_gemm(const LoraGemmArgs& g, hipStream_t s);

// The rows' adapters of a launch sequence: out[(l 7 + p) ld + t] = rows[t][l 7 + p], nothing where rows[t] is null,
// for layers l in [l0, l1), the 7 projections p and rows t < M.
void lora_table(const LoraRef* const* rows, int M, int l0, int l1, LoraRef* out, int ld, hipStream_t s);

// u = clamp(amp_fold(A x)) of the rows' own adapters for up to 3 projections sharing one input
struct RowsUArgs {
	int M, K, nproj;
	const int8_t* x;          // [M, K]
	const LoraRef* refs[3];   // [M]
	int8_t* u[3];             // [M, kMaxRank]
};
void rows_u(const RowsUArgs& a, hipStream_t s);

// The rules of one row of logits.
struct LogitRule {
	const int32_t *history, *bias_ids, *bias_values;
	const uint8_t* mask;  // bit j: token j is legal; null: every token is
	int32_t history_len, bias_count, repetition_q16, presence, frequency, reserved;
};

struct PickArgs {
	int rows, vocab;
	const int32_t* logits;
	int64_t ld, adjusted_ld;
	const LogitRule* rules;
	int32_t* adjusted;  // or null
	int32_t* tokens;
	void* ws;  // pick_workspace() bytes
};
size_t pick_workspace(int rows, int vocab);
// *at[i] = token[i] for every i < n with at[i]
void append_tokens(int32_t* const* at, const int32_t* token, int n, hipStream_t s);
void pick_tokens(const PickArgs& a, hipStream_t s);

}  // namespace sslm_launch
