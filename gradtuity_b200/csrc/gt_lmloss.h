// What the losses of the language-model head share between gt_lmloss.cu (targets, rows, entry points) and
// gt_lmloss_umma.cu (the tensor-core kernel of the linear forms).
#pragma once

#include "gt_internal.h"

// Values that a call computes on the device and later launches of it read.
struct LmScalars {
  int count;            // rows that count
  unsigned amax_x;      // largest finite |x|, |w| as float bits (whole-number maximum: the order does not matter)
  unsigned amax_w;
  float logit2;         // log2(e) / T times the operands' scales: accumulator -> z log2(e)
  float dx, dw;         // accumulator -> dx, dw
};

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
  const float2* stats;           // (m log2(e), s) by compact row
  const float2* factor;          // G = factor.x e^(z - m) - factor.y q, by compact row
  const int* ids; const float* q; int K;
  float* dx; float* dw; int acc_dx, acc_dw;
  float* dx_partial; int dx_split;   // dx of a piece in `dx_split` shares of its words, when that is over 1
  int* counters;                 // one zeroed int per launch: the next unit of work
};

constexpr int LM_TILE = 256;     // rows and columns of the tile that a pair of CTAs computes
constexpr int LM_KBLOCK = 64;    // k elements of one stage

// Forward: per row and half tile of words, (maximum, sum of exponentials).
int gt_lm_stats(gt_ctx* ctx, const LmProblem& p);
// One step of the backward walk over the pieces: G of piece `piece` (if it exists), and dx, dw of the piece before.
int gt_lm_step(gt_ctx* ctx, const LmProblem& p, int piece);
// Pairs of CTAs that run at the same time; 0 when the query fails.
int gt_lm_pairs(gt_ctx* ctx);
