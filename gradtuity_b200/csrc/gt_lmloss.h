// What the losses of the language-model head share between gt_lmloss.cu (targets, rows, entry points) and
// gt_lmloss_umma.cu (the tensor-core kernel of the linear forms).
#pragma once

#include "gt_internal.h"

constexpr int LM_TOP_MAX = 1024;             // targets of a row: they are sorted in shared memory
constexpr int LM_UNUSED = 0x7fffffff;        // id of a place that is not in use; sorts behind every word

// Values that a call computes on the device and later launches of it read.
struct LmScalars {
  int count;            // rows that count
  unsigned amax_x;      // largest finite |x|, |w| as float bits (whole-number maximum: the order does not matter)
  unsigned amax_w;
  float logit2;         // log2(e) / T times the operands' scales: accumulator -> z log2(e)
  float dx, dw;         // accumulator -> dx, dw
};

// A word in which the blocks of a launch count themselves out, so that the last one can go on with what all have written: zero
// between launches, the last block sees to that.  One for each stream that the context launches on.
inline unsigned long long* lm_ticket(gt_ctx* ctx) { return (unsigned long long*)(ctx->d_status + 1016 + (ctx->side_saved ? 2 : 0)); }
#ifdef __CUDACC__
// Called by one thread of each block once the block's writes are done (behind a barrier).  True in the last block of `blocks`; `sum` is
// then the sum of all blocks' `mine` (whole numbers: the order does not matter).
__device__ __forceinline__ bool lm_count_out(unsigned long long* ticket, unsigned blocks, unsigned mine, unsigned* sum) {
  __threadfence();
  const unsigned long long was = atomicAdd(ticket, (1ull << 32) + mine);
  if ((unsigned)(was >> 32) != blocks - 1) return false;
  *ticket = 0;
  __threadfence();
  *sum = (unsigned)was + mine;
  return true;
}
#endif

// What the forward pass leaves for the backward pass, in one block of memory.
struct LmSaved {
  LmScalars* scalars;
  float* weight;    // by row: 1, or 0 for a row that does not count
  float* konst;     // by row: sum of q log q
  int* ids;         // (M, K), ascending, UNUSED at the end
  float* q;         // (M, K), 0 where unused
  int* row_of;      // rows that count, in order
  float2* stats;    // (m, s): by row, m a logit (distillation of given logits); by compact row, m in units of log 2 (linear forms)
  float2* factor;   // by compact row, see LmProblem
  size_t bytes;
};
inline size_t lm_up256(size_t n) { return (n + 255) & ~(size_t)255; }
struct LmCarve {
  char* p; size_t at;
  template <class T> T* take(size_t n) { T* r = (T*)(p + at); at += lm_up256(n * sizeof(T)); return r; }
};
inline LmSaved lm_saved(LmCarve& c, long long M, long long K) {
  LmSaved s;
  s.scalars = c.take<LmScalars>(1);
  s.weight = c.take<float>(M);
  s.konst = c.take<float>(M);
  s.ids = c.take<int>(M * K);
  s.q = c.take<float>(M * K);
  s.row_of = c.take<int>(M);
  s.stats = c.take<float2>(M);
  s.factor = c.take<float2>(M);
  s.bytes = c.at;
  return s;
}
inline LmSaved lm_saved(void* base, long long M, long long K) {
  LmCarve c = {(char*)base, 0};
  return lm_saved(c, M, K);
}

// Two products' operands as 16-bit halves: v = 2^e (hi + lo), both fp16, scaled so that the matrix's largest value lies in
// [2^14, 2^15).  Rows are `pitch` halves apart.
struct LmSplit { uint16_t* hi; uint16_t* lo; };

struct LmProblem {
  long long M, V, E;
  long long pitch_e;             // of the x and w halves
  long long words;               // of one piece
  long long pitch_v;             // of the G halves (two pieces of them)
  int products;                  // 3: hi hi + hi lo + lo hi, 1: hi hi
  LmScalars* scalars;
  const int* row_of;             // compact row -> row of x
  LmSplit x, w, g[2];
  float2* partial;               // (V tiles x 2, M) maxima and sums of the forward pass
  float* target_z;               // forward: z log2(e) of the targets, (M, K) by compact row
  const float2* stats;           // (m log2(e), s) by compact row
  const float2* factor;          // G = factor.x e^(z - m) - factor.y q, by compact row
  const int* ids; const float* q; int K;
  float* dx; float* dw; int acc_dx, acc_dw;
  float* dx_partial; int dx_split;   // dx of a piece in `dx_split` shares of its words, when that is over 1: (dx_split, M, E)
  float* dw_partial;                 // dW of a piece in lm_dw_split shares of the rows, when that is over 1: (shares, words of the piece, E)
  int* counters;                 // one zeroed int per launch: the next unit of work
};

constexpr int LM_TILE = 256;     // rows and columns of the tile that a pair of CTAs computes
constexpr int LM_KBLOCK = 64;    // k elements of one stage

inline bool lm_bad_sizes(long long M, long long V, long long K) {      // ids are float-encoded: exact below 2^24
  return M <= 0 || V <= 0 || K <= 0 || M > 0x7fffffff || V >= (1ll << 24) || K > LM_TOP_MAX;
}
inline bool lm_bad_temperature(float T) { return !(T >= 1.0e-6f && T <= 1.0e6f); }      // T^2, 1 / T and their products stay finite
inline bool lm_bad_reduction(int r) { return r != GT_REDUCE_NONE && r != GT_REDUCE_MEAN && r != GT_REDUCE_SUM; }

// Sorted targets, weights and the count of the rows of a distillation (top_targets_kernel); also 0 for the loss of rows that do not count.
int gt_lm_top_targets(gt_ctx* ctx, const LmSaved& s, float* row_loss, const float* ids, const float* teacher, long long M, long long V, long long K,
                      float T);

// The sums of a step: what a pair of CTAs has to do in it, in stages, times `pairs`.
inline long long lm_step_stages(const LmProblem& p, long long words_mul, long long words_grad) {
  auto tiles = [](long long n) { return (n + LM_TILE - 1) / LM_TILE; };
  auto stages = [](long long n) { return (n + LM_KBLOCK - 1) / LM_KBLOCK; };
  return tiles(p.M) * tiles(p.E) * stages(words_mul) + tiles(words_mul) * tiles(p.E) * stages(p.M) + tiles(p.M) * tiles(words_grad) * stages(p.E);
}
// A dx (dW) tile runs over all words of a piece (all rows).  Where these `k` stages are long against a pair's part of the step, they are
// shared out and the shares added up afterwards: into units of a quarter of a pair's part, since it is not known how many rows
// count, and of 16 stages at least.
inline int lm_shares(long long k, long long step, long long pairs) {
  long long n = 3 * k * pairs > 2 * step ? (4 * k * pairs + step - 1) / step : 1;
  if (n > k / 16) n = k / 16;
  return (int)(n < 1 ? 1 : n);
}
inline int lm_dw_split(gt_ctx* ctx, const LmProblem& p, long long words_mul, long long words_grad) {
  return words_mul ? lm_shares((p.M + LM_KBLOCK - 1) / LM_KBLOCK, lm_step_stages(p, words_mul, words_grad), ctx->sm_count / 2) : 1;
}
inline long long lm_piece_words(const LmProblem& p, long long piece) {
  const long long v0 = piece * p.words;
  return v0 < 0 || v0 >= p.V ? 0 : p.V - v0 < p.words ? p.V - v0 : p.words;
}

// Forward: per row and half tile of words, (maximum, sum of exponentials); and the targets' logits.
int gt_lm_stats(gt_ctx* ctx, const LmProblem& p);
// One step of the backward walk over the pieces: G of piece `piece` (if it exists), and dx, dw of the piece before.
int gt_lm_step(gt_ctx* ctx, const LmProblem& p, int piece);
// Pairs of CTAs that run at the same time; 0 when the query fails.
int gt_lm_pairs(gt_ctx* ctx);

// ---- few rows, or little work (gt_lmloss_rows.cu) ----
struct LmRows {
  int M, V, E, K;
  const float* x; const float* w;
  float T;
  const float* targets; float ignore;      // cross entropy: the forward kernel takes the losses itself
  LmSaved s;
  float2* partial;                         // (parts, M)
  int parts;                               // blocks over the words
  float* row_loss; float* loss;            // either may be null
  const float* upstream; int reduction;
  float* dw; int acc_dw;
  float* dx_part;                          // (parts, M, E); null: no dx wanted
  unsigned long long* ticket;
  int cw, c;                               // warps that share the columns, columns a lane
};
constexpr long long LM_ROWS_WORK = 64ll << 20;
bool gt_lm_few_rows(long long M, long long V, long long E);
int gt_lm_rows_parts(gt_ctx* ctx, long long M, long long V, bool backward);
int gt_lm_rows_forward(gt_ctx* ctx, const LmRows& p);
int gt_lm_rows_backward(gt_ctx* ctx, const LmRows& p, float* dx, int acc_dx);
