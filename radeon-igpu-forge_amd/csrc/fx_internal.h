// Entry points of the library that only the host module (host.cpp) calls: products whose shapes
// the C ABI's functions refuse or whose workspace they have no argument for.  The conventions
// are the ABI's (fx_abi.h); return codes and messages too.
#pragma once

#include <stdint.h>

namespace fx {

// dX (M, N) = dY (M, K) W (K, N), times G (the GELU derivative, row stride N) when given, on the
// small tiles: any M, N and K multiples of 8, W and dX contiguous, 16-byte aligned buffers.
// Few tiles of a long K are cut into K slices whose fp32 partials go through `work`.
int64_t input_grad_workspace(int64_t M, int64_t N, int64_t K, bool gated);
int input_grad(const uint16_t* dY, int64_t ldy, const uint16_t* W, const uint16_t* G, uint16_t* dX, float* work, int64_t M,
               int64_t N, int64_t K, void* stream);

// out (cols) = bf16(column sums of g (rows, cols), row stride cols), fp32 sums in a fixed order;
// cols a multiple of 8, g, work and out 16-byte aligned
int64_t column_sums_workspace(int64_t rows, int64_t cols);
int column_sums(const uint16_t* g, int64_t rows, int64_t cols, float* work, uint16_t* out, void* stream);

// A decode step's small ends, one launch each.
// tok_out[0..n) = tok, *pos_out = pos, lens[0..n) = pos + 1
int decode_inputs(const int64_t* tok, int64_t n, int64_t pos, int64_t* tok_out, int64_t* pos_out, int32_t* lens, void* stream);
// x (n, D) = bf16(E[tok[i]] + P[*pos]), E (V, D) and P (T, D) contiguous, D a multiple of 8; a row of
// NaN for an id or a position outside its table
int decode_embed(const int64_t* tok, const int64_t* pos, const uint16_t* E, int64_t V, const uint16_t* P, int64_t T, uint16_t* x,
                 int64_t n, int64_t D, void* stream);
// x (B, N, D) = bf16(E[tok] + P[ctx + depth]) of the nodes first .. first + N - 1 of drafted trees behind ctx cached
// tokens, E (V, D) and P (L, D) contiguous; a node whose own bit is set in its tree word is a row of NaN if its token or
// position is outside the table or its row ctx + node outside a cache of Tmax.  Strides in elements, b / n.
struct TreeEmbedArgs {
    const int64_t *tok, *tree;
    const int32_t *ctx, *depth;
    const uint16_t *E, *P;
    uint16_t* x;
    int64_t tokb, tokn, depthb, depthn, treeb, treen, V, L, Tmax, D;
    int32_t N, first;
};
int tree_embed(const TreeEmbedArgs& a, int64_t B, void* stream);
// out (M, N) fp32 = the bf16 values of norm(X) W^T (fx_linear_fwd_ex with the norm, M <= 64), X rows
// ldx apart
int few_rows_logits(const uint16_t* X, int64_t ldx, const uint16_t* W, const uint16_t* norm_w, float eps, float* out, int64_t M,
                    int64_t N, int64_t K, void* stream);

// ---- drafted decoding ----

// Attention of a tree of drafted tokens over a cache (tree.hip).  Strides in elements; b / t / h (cache),
// b / n / h (q, new keys and values), b / n (tree).
struct TreeArgs {
    const uint16_t *q, *k, *v, *knew, *vnew;
    const int32_t* ctx;
    const int64_t* tree;
    uint16_t* o;
    float *lse, *work;
    int64_t qb, qn, qh, kb, kt, kh, vb, vt, vh, knb, knn, knh, vnb, vnn, vnh, treeb, treen;
    int32_t B, N, first, H, Hkv, Tmax, D;
    float scale;
};
int64_t tree_attention_workspace(int32_t B, int32_t N, int32_t H, int32_t Hkv, int32_t Tmax, int32_t D);
int tree_attention(const TreeArgs& a, void* stream);

// probs (rows, V) fp32 = softmax(logits / temperature) over the top_k largest logits of a row and their
// equals (top_k <= 0 or >= V: over all); logits (rows, V) contiguous, fp32 or (bf16) bfloat16.  A row
// without a finite maximum: zeros where every logit is -inf, else NaN.
int sampling_probs(const void* logits, bool bf16, float* probs, int64_t rows, int64_t V, double temperature, int64_t top_k, void* stream);

// The walk of drafted trees (draft.hip).  probs, draft (B, N, V) fp32 contiguous (draft may be null),
// tokens (B, N) int64, parents (B, N) int32, uniform (B, N) fp32; out (B, N) int64, path (B, N) int32,
// counts (B) int32.
int verify_draft(const float* probs, const float* draft, const int64_t* tokens, const int32_t* parents, const float* uniform,
                 int64_t* out, int32_t* path, int32_t* counts, int32_t B, int32_t N, int64_t V, void* stream);

// Rows of caches moved: row ctx[b] + path[b, d] -> ctx[b] + d for d < counts[b], in the order of d; ctx_out = ctx +
// counts.  Caches (B, T, H, D) of one shape with strides b / t / h.
constexpr int kCompactTensors = 64;
struct CompactArgs {
    uint16_t* at[kCompactTensors];
    int64_t sb[kCompactTensors], st[kCompactTensors], sh[kCompactTensors];
    const int32_t *ctx, *path, *counts;
    int32_t* ctx_out;   // null: another launch writes it
    int32_t count, B, T, H, D, N;
};
int compact_cache(const CompactArgs& a, void* stream);

// ---- paged cache ----
// Pools (N, P, Hkv, D), P = 2^shift rows a page, strides p / t / h; a row's pages are the first of its line of `table`
// (R, M), lines `tab` apart; a page's uses count the rows that hold it.

// Attention of one new token a row over its pages (paged.hip): q (R, H, D), o (R, H, D) and lse (R, H) contiguous.
// Strides in elements, r / h.  A table entry that is no page: its keys are nobody's.
struct PagedArgs {
    const uint16_t *q, *knew, *vnew;
    uint16_t *k, *v;
    const int32_t *table, *lens;
    uint16_t* o;
    float *lse, *work;
    int64_t qr, qh, kp, kt, kh, vp, vt, vh, knr, knh, vnr, vnh, tab;
    int32_t R, H, Hkv, N, shift, M, D;
    float scale;
};
int64_t paged_attention_workspace(int32_t R, int32_t H, int32_t Hkv, int32_t N, int32_t M, int32_t shift, int32_t D);
int paged_attention(const PagedArgs& a, void* stream);

// Pages and slots for tokens to be added (pages.hip).  slots (R, most) int64, out (R) int32 the lengths after it;
// `work`: extend_pages_workspace bytes, whose first R int4 are each row's copy: (page, to page, rows or 0 for none, whether the row has what it wanted).
constexpr int kPagesRows = 8192;   // rows of a table, at most
struct ExtendArgs {
    int32_t *table, *uses;
    const int32_t *lens, *add;
    int64_t* slots;
    int32_t *out, *work;
    int64_t tab;
    int32_t R, M, N, shift, most;
    bool copies;   // false: rows whose open page others hold get nothing
};
int64_t extend_pages_workspace(int32_t R, int32_t M, int32_t N, int32_t shift, int32_t most, bool copies);
int extend_pages(const ExtendArgs& a, void* stream);
// the copies of extend_pages in up to kCopyTensors pools of one shape
constexpr int kCopyTensors = 64;
struct CopyPagesArgs {
    uint16_t* at[kCopyTensors];
    int64_t sp[kCopyTensors], st[kCopyTensors], sh[kCopyTensors];
    const int32_t* copies;
    int32_t count, R, H, D;
};
int copy_pages(const CopyPagesArgs& a, void* stream);

// Rows k, v (R, T, H, D) to slots (R, T) int64 of the pools; a slot outside them is passed over.  Strides r / t / h.
struct StorePagesArgs {
    const uint16_t *k, *v;
    const int64_t* slots;
    uint16_t *kp, *vp;
    int64_t kr, kt, kh, vr, vt, vh, sr, st, kpp, kpt, kph, vpp, vpt, vph;
    int64_t N;
    int32_t R, T, H, D, shift;
};
int store_pages(const StorePagesArgs& a, void* stream);

// Row r becomes row parents[r], or ends where that is no row; out (R) the lengths after it.
struct ReorderArgs {
    int32_t *table, *uses;
    const int32_t *lens, *parents;
    int32_t* out;
    int64_t tab;
    int32_t R, M, N, shift;
};
int reorder_pages(const ReorderArgs& a, void* stream);

// The best K continuations of each sequence's K beams (beam.hip): logits (B, K, V) contiguous, fp32 or (bf16) bfloat16;
// scores, weight (B, K) fp32 and done (B, K) bytes contiguous, weight and done may be null; out (B, K) fp32, rows (B, K)
// int32, tokens (B, K) int64.  `work`: beam_select_workspace bytes.
constexpr int kBeamMost = 32;             // beams
constexpr int64_t kBeamVocab = 1 << 20;   // logits of a row
struct BeamArgs {
    const void* logits;
    const float *scores, *weight;
    const uint8_t* done;
    float* out;
    int32_t* rows;
    int64_t* tokens;
    void* work;
    int64_t V, fill;
    int32_t B, K;
    bool bf16;
};
int64_t beam_select_workspace(int32_t B, int32_t K, int64_t V, bool bf16);
int beam_select(const BeamArgs& a, void* stream);

}  // namespace fx
