// Losses of the language-model head with sparse targets, and their gradients: the targets, and the linear forms.
// (Distillation of given logits: gt_distill.cu.)
//
// For token t and word v, z_tv = logit_tv / T (T = 1 for cross entropy; the linear forms compute logit = x W^T themselves):
//     p_tv = exp(z_tv - m_t) / s_t,  m_t = max_v z_tv,  s_t = sum_v exp(z_tv - m_t)
//     loss_t = T^2 sum_k q_tk (log q_tk - (z_t,id_tk - m_t - log s_t))
//     d loss_t / d logit_tv = T (p_tv - sum of the q_tk with id_tk = v)
// The targets of a row are (id, q) pairs sorted by id: one pair with q = 1 for cross entropy; for distillation the softmax of
// the teacher's top logits / T over the entries in use.  A row without any target in use has weight 0: no loss, no gradient.
// m and s are kept apart instead of as m + log s: p then carries no rounding of a sum of that size.
//
// Linear forms: the (tokens x words) logits are never kept.  The forward pass keeps each row's m and s, the backward pass walks
// over pieces of the vocabulary, computes a piece's logits again, turns them into the logits' gradient G, and multiplies:
//     dx += G W_piece,   dW_piece = G^T x      (gt_lmloss_umma.cu)
// Rows that do not count are left out from the start: the products work on the others, closed up ("compact" rows).

#include <math.h>

#include <cuda_fp16.h>

#include "gt_lmloss.h"

namespace {

// What G of one piece of the vocabulary may occupy (two pieces of it exist at a time).  8192 x 768 x 50257 with gradients, at 64 / 96 /
// 128 / 160 / 256 MB: 6.80 / 6.59 / 6.58 / 6.41 / 6.37 ms; the logits alone would be 1.65 GB, and so would their gradient.
constexpr long long PIECE_BYTES = 128ll << 20;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ---- targets -------------------------------------------------------------------------------------

// Rows that count, in order, a block of 1024 threads at a time: `counts` is this thread's row t.  base: rows before.
__device__ __forceinline__ void append_rows(bool counts, long long t, int& base, int* row_of) {
  __shared__ int sums[32];
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  const unsigned mask = __ballot_sync(0xffffffffu, counts);
  if (l == 0) sums[w] = __popc(mask);
  __syncthreads();
  const int mine = sums[l];
  int before = w > l ? mine : 0, all = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if (counts) row_of[base + before + __popc(mask & ((1u << l) - 1))] = (int)t;
  base += all;
  __syncthreads();
}

// Cross entropy: one target of q = 1 per row, and the rows that count.  An id outside the vocabulary sets the status word.  One block,
// which also clears what later kernels count in.
__global__ void __launch_bounds__(1024) hard_targets_kernel(const float* __restrict__ targets, long long M, long long V, float ignore, LmSaved s,
                                                            float* __restrict__ row_loss, int* counters, int* status) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  int base = 0;
  for (long long t0 = 0; t0 < M; t0 += 1024) {
    const long long t = t0 + threadIdx.x;
    bool used = false;
    if (t < M) {
      const float f = targets[t];
      const bool in_range = f >= 0.0f && f < (float)V;
      used = f != ignore && in_range;
      if (f != ignore && !in_range) atomicExch(status, GT_ERR_INVALID_ARG);
      s.ids[t] = used ? (int)f : LM_UNUSED;
      s.q[t] = used ? 1.0f : 0.0f;
      s.weight[t] = used ? 1.0f : 0.0f;
      s.konst[t] = 0.0f;
      if (!used) row_loss[t] = 0.0f;
    }
    append_rows(used, t, base, s.row_of);
  }
  if (threadIdx.x == 0) {
    *counters = 0;
    s.scalars->count = base; s.scalars->amax_x = 0; s.scalars->amax_w = 0;
  }
}

// Distillation: a warp per row.  q = softmax(teacher / T) over the places in use (id >= 0, logit above -inf), sorted by id by
// counting, for each place, the places that go before it (K^2 comparisons, K is tens to a few hundred).
__global__ void __launch_bounds__(128) top_targets_kernel(const float* __restrict__ ids, const float* __restrict__ teacher, long long M,
                                                          long long V, int K, float inv_T, LmSaved s,
                                                          float* __restrict__ row_loss, unsigned long long* ticket, int* status) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  extern __shared__ float smem[];
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  int* key = reinterpret_cast<int*>(smem) + (size_t)w * 2 * K;
  float* val = reinterpret_cast<float*>(key + K);
  const long long t = (long long)blockIdx.x * 4 + w;
  float mx = -INFINITY;
  bool any = false;
  if (t < M) {
    for (int k = l; k < K; k += 32) {
      const float f = ids[t * K + k], v = teacher[t * K + k];
      bool used = !(f < 0.0f) && v > -INFINITY;
      if (used && !(f < (float)V)) { atomicExch(status, GT_ERR_INVALID_ARG); used = false; }
      key[k] = used ? (int)f : LM_UNUSED;
      val[k] = used ? v : -INFINITY;
      if (used) { any = true; mx = fmaxf(mx, v); }
    }
    any = __any_sync(0xffffffffu, any);
    mx = warp_max(mx);
    __syncwarp();
    float sum = 0.0f;
    for (int k = l; k < K; k += 32)
      if (key[k] != LM_UNUSED) sum += expf((val[k] - mx) * inv_T);
    sum = warp_sum(sum);
    const float log_sum = logf(sum), inv = 1.0f / sum;
    float konst = 0.0f;
    constexpr int MINE = 4;                                   // places ranked together, against one reading of the keys
    for (int k0 = l; k0 < K; k0 += 32 * MINE) {
      int id[MINE], before[MINE];
#pragma unroll
      for (int i = 0; i < MINE; ++i) { id[i] = k0 + 32 * i < K ? key[k0 + 32 * i] : LM_UNUSED; before[i] = 0; }
#pragma unroll 8
      for (int j = 0; j < K; ++j) {
        const int o = key[j];
#pragma unroll
        for (int i = 0; i < MINE; ++i) before[i] += (o < id[i]) || (o == id[i] && j < k0 + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int k = k0 + 32 * i;
        if (k >= K) break;
        float q = 0.0f;
        if (id[i] != LM_UNUSED) {
          const float u = (val[k] - mx) * inv_T;
          q = expf(u) * inv;
          if (q != 0.0f) konst += q * (u - log_sum);          // 0 log 0 = 0
        }
        s.ids[t * K + before[i]] = id[i];
        s.q[t * K + before[i]] = q;
      }
    }
    konst = warp_sum(konst);
    if (l == 0) {
      s.weight[t] = any ? 1.0f : 0.0f;
      s.konst[t] = konst;
      if (!any) row_loss[t] = 0.0f;
    }
  }
  const int n = __syncthreads_count(any && l == 0);
  unsigned sum;
  if (threadIdx.x == 0 && lm_count_out(ticket, gridDim.x, n, &sum)) s.scalars->count = (int)sum;
}

// The same for a distillation's rows, whose targets are there.
__global__ void __launch_bounds__(1024) compact_rows_kernel(long long M, LmSaved s, int* counters) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  int base = 0;
  for (long long t0 = 0; t0 < M; t0 += 1024) {
    const long long t = t0 + threadIdx.x;
    append_rows(t < M && s.weight[t] != 0.0f, t, base, s.row_of);
  }
  if (threadIdx.x == 0) { *counters = 0; s.scalars->count = base; s.scalars->amax_x = 0; s.scalars->amax_w = 0; }
}

// ---- operands of the linear forms: largest value, then the split into halves ------------------------

// Whole matrix w, and of x the rows that count.  A maximum of bits as whole numbers, so the order of the additions is no matter.
__global__ void __launch_bounds__(256) largest_kernel(const float* __restrict__ x, const float* __restrict__ w, long long V, long long E, LmSaved s,
                                                      int blocks_x) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const bool is_x = (int)blockIdx.x < blocks_x;
  const long long rows = is_x ? s.scalars->count : V;
  const int first = is_x ? blockIdx.x : blockIdx.x - blocks_x, step = is_x ? blocks_x : gridDim.x - blocks_x;
  const float* src = is_x ? x : w;
  const bool vec = ((uintptr_t)src & 15) == 0;
  unsigned m = 0;
  auto see = [&](float f) {
    const unsigned b = __float_as_uint(f) & 0x7fffffffu;
    if (b < 0x7f800000u && b > m) m = b;                     // infinities and NaN do not set the scale
  };
  if (!is_x && vec) {
    const float4* p = reinterpret_cast<const float4*>(src);
    const long long n = rows * E / 4;
    long long i = (long long)first * 256 + threadIdx.x;
    for (; i + 3ll * step * 256 < n; i += 4ll * step * 256) {
      float4 a[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) a[k] = p[i + (long long)k * step * 256];
#pragma unroll
      for (int k = 0; k < 4; ++k) { see(a[k].x); see(a[k].y); see(a[k].z); see(a[k].w); }
    }
    for (; i < n; i += (long long)step * 256) { const float4 a = p[i]; see(a.x); see(a.y); see(a.z); see(a.w); }
    if (first == 0 && threadIdx.x < (int)(rows * E - 4 * n)) see(src[4 * n + threadIdx.x]);
  } else {
    for (long long r = (long long)first * 8 + (threadIdx.x >> 5); r < rows; r += (long long)step * 8) {
      const float* p = src + (is_x ? s.row_of[r] : r) * E;
      for (long long e = threadIdx.x & 31; e < E; e += 32) see(p[e]);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0 && m) atomicMax(is_x ? &s.scalars->amax_x : &s.scalars->amax_w, m);
}

// v = 2^e (scaled value), the largest scaled value in [2^14, 2^15): fp16 holds it, and halves down to 2^-24 of an ulp each
__device__ __forceinline__ int scale_exponent(unsigned amax) {
  if (amax == 0) return 0;
  const int e = (int)(amax >> 23) - 127;
  return (e < -100 ? -100 : e) - 14;
}

// A warp per row.  x: compact rows, and zeros behind them to the end of the last tile of rows.
__global__ void __launch_bounds__(256) split_kernel(const float* __restrict__ x, const float* __restrict__ w, long long M, long long V, long long E,
                                                    long long pitch, LmSaved s, LmSplit xs, LmSplit ws, int products, float T, int blocks_x) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const int l = threadIdx.x & 31;
  const bool is_x = (int)blockIdx.x < blocks_x;
  const int ex = scale_exponent(s.scalars->amax_x), ew = scale_exponent(s.scalars->amax_w);
  if (blockIdx.x == 0 && threadIdx.x == 0) s.scalars->logit2 = ldexpf(1.4426950408889634f / T, ex + ew);
  const long long count = s.scalars->count;
  const long long up_to = (count + LM_TILE - 1) / LM_TILE * LM_TILE;
  const long long rows = is_x ? (up_to < M ? up_to : M) : V;
  const int first = is_x ? blockIdx.x : blockIdx.x - blocks_x, step = is_x ? blocks_x : gridDim.x - blocks_x;
  const float scale = ldexpf(1.0f, -(is_x ? ex : ew));
  const LmSplit d = is_x ? xs : ws;
  const bool vec = ((uintptr_t)(is_x ? x : w) & 15) == 0 && E % 4 == 0;
  auto halves = [&](float v, unsigned short& hi, unsigned short& lo) {
    const float f = v * scale;
    const __half h = __float2half_rn(f);
    hi = __half_as_ushort(h);
    lo = __half_as_ushort(__float2half_rn(f - __half2float(h)));
  };
  for (long long i = (long long)first * 8 + (threadIdx.x >> 5); i < rows; i += (long long)step * 8) {
    // w from its end: the tail of it is still in L2 from the pass before
    const long long r = is_x ? i : rows - 1 - i;
    const bool zero = is_x && r >= count;
    const float* src = is_x ? x + (zero ? 0ll : (long long)s.row_of[r]) * E : w + r * E;
    uint16_t* hi = d.hi + r * pitch;
    uint16_t* lo = d.lo + r * pitch;
    if (vec) {
#pragma unroll 4
      for (long long e = 4 * l; e < E; e += 128) {
        const float4 a = zero ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(src + e);
        ushort4 h, o;
        halves(a.x, h.x, o.x); halves(a.y, h.y, o.y); halves(a.z, h.z, o.z); halves(a.w, h.w, o.w);
        *reinterpret_cast<ushort4*>(hi + e) = h;
        if (products == 3) *reinterpret_cast<ushort4*>(lo + e) = o;
      }
    } else {
      for (long long e = l; e < E; e += 32) {
        unsigned short h, o;
        halves(zero ? 0.0f : src[e], h, o);
        hi[e] = h;
        if (products == 3) lo[e] = o;
      }
    }
  }
}

// ---- rows ------------------------------------------------------------------------------------------

// The rows' losses added up by one block, in 64 bits and in a fixed order.
template <int THREADS>
__device__ __forceinline__ void sum_losses(float* loss, const float* row_loss, long long M, int count, int mean) {
  __shared__ double sums[THREADS / 32];
  double a = 0.0;
  for (long long r = threadIdx.x; r < M; r += THREADS) a += __ldcg(row_loss + r);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < THREADS / 32; ++k) a += sums[k];
    if (mean && count > 0) a /= (double)count;
    *loss = (float)a;
  }
}

// After the products: (m, s) of the rows that count from their tiles', and their losses from the targets' logits.  32 rows a block, the
// tiles shared out over 32 warps, so that a warp reads whole lines; then a warp per row.  The last block to end adds the losses up.
__global__ void __launch_bounds__(1024) join_tiles_kernel(const float2* __restrict__ partial, int parts, const float* __restrict__ target_z,
                                                          float* __restrict__ row_loss, float* __restrict__ loss, long long M, int K, float T, int mean,
                                                          LmSaved s, unsigned long long* ticket) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  __shared__ float2 red[32][33];
  __shared__ int last;
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31, count = s.scalars->count;
  const long long i = (long long)blockIdx.x * 32 + l;
  float m = -INFINITY, sum = 0.0f;                            // m in units of log 2
  if (i < count) {
#pragma unroll 4
    for (int j = w; j < parts; j += 32) {
      const float2 b = partial[(long long)j * M + i];
      const float top = fmaxf(m, b.x);
      if (top == -INFINITY) { sum += b.y; continue; }         // nothing but words that do not exist; or a NaN, which counts
      sum = sum * gt_ex2(m - top) + b.y * gt_ex2(b.x - top);
      m = top;
    }
  }
  red[w][l] = make_float2(m, sum);
  __syncthreads();
  // warp w joins row w's 32 shares, in an order that is the same every time
  const float2 mine = red[l][w];
  const float top = warp_max(mine.x);
  sum = warp_sum(top == -INFINITY ? mine.y : mine.y * gt_ex2(mine.x - top));
  const long long r = (long long)blockIdx.x * 32 + w;
  if (r < count) {
    const long long t = s.row_of[r];
    const float log_s = logf(sum);
    float cross = 0.0f;
    for (int k = l; k < K; k += 32) {
      if (s.ids[t * K + k] == LM_UNUSED) break;
      const float q = s.q[t * K + k];
      if (q != 0.0f) cross += q * ((target_z[r * K + k] - top) * 0.6931471805599453f - log_s);
    }
    cross = warp_sum(cross);
    if (l == 0) {
      s.stats[r] = make_float2(top, sum);
      row_loss[t] = T * T * (s.konst[t] - cross);
    }
  }
  if (!loss) return;
  __threadfence();
  __syncthreads();
  unsigned none;
  if (threadIdx.x == 0) last = lm_count_out(ticket, gridDim.x, 0, &none);
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum_losses<1024>(loss, row_loss, M, count, mean);
}

// After the few rows' products (distillation): the same, a block per row; the parts are blocks' and by row, and the targets' logits are
// taken straight from x and w.
__global__ void __launch_bounds__(256) join_blocks_kernel(float* __restrict__ row_loss, float* __restrict__ loss, const float* __restrict__ x,
                                                          const float* __restrict__ w, long long M, int E, int K, float T, int mean,
                                                          const float2* __restrict__ partial, int parts, LmSaved s, unsigned long long* ticket) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  __shared__ float part[8];
  __shared__ float2 joined[8];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
  const long long t = blockIdx.x;
  float m = -INFINITY, sum = 0.0f;
  auto add = [&](float2 b) {
    const float top = fmaxf(m, b.x);
    if (top == -INFINITY) { sum += b.y; return; }
    sum = sum * gt_ex2(m - top) + b.y * gt_ex2(b.x - top);
    m = top;
  };
  for (int j = threadIdx.x; j < parts; j += 256) add(partial[(long long)j * M + t]);
  const float warp_top = warp_max(m);
  sum = warp_sum(warp_top == -INFINITY ? sum : sum * gt_ex2(m - warp_top));
  if (l == 0) joined[warp] = make_float2(warp_top, sum);
  __syncthreads();
  m = -INFINITY; sum = 0.0f;
  for (int k = 0; k < 8; ++k) add(joined[k]);
  if (threadIdx.x == 0) s.stats[t] = make_float2(m, sum);
  const bool live = s.weight[t] != 0.0f;
  float cross = 0.0f;
  if (live) {
    const float log_s = logf(sum), top = m * 0.6931471805599453f;
    const float* xr = x + t * E;
    const bool vec = ((uintptr_t)x & 15) == 0 && ((uintptr_t)w & 15) == 0 && E % 4 == 0;
    constexpr int AT_ONCE = 4;                                // targets whose words are read together
    for (int k0 = warp * AT_ONCE; k0 < K; k0 += 8 * AT_ONCE) {
      const float* wr[AT_ONCE];
      float q[AT_ONCE], z[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int id = k0 + k < K ? s.ids[t * K + k0 + k] : LM_UNUSED;
        q[k] = id != LM_UNUSED ? s.q[t * K + k0 + k] : 0.0f;
        wr[k] = w + (long long)(id != LM_UNUSED ? id : 0) * E;
        z[k] = 0.0f;
      }
      if (vec) {
#pragma unroll 2
        for (int e = 4 * l; e < E; e += 128) {
          const float4 a = *reinterpret_cast<const float4*>(xr + e);
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            const float4 b = *reinterpret_cast<const float4*>(wr[k] + e);
            z[k] = fmaf(a.x, b.x, z[k]); z[k] = fmaf(a.y, b.y, z[k]); z[k] = fmaf(a.z, b.z, z[k]); z[k] = fmaf(a.w, b.w, z[k]);
          }
        }
      } else {
#pragma unroll 4
        for (int e = l; e < E; e += 32) {
          const float a = xr[e];
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) z[k] = fmaf(a, wr[k][e], z[k]);
        }
      }
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const float sum = warp_sum(z[k]) / T;
        if (q[k] != 0.0f) cross += q[k] * ((sum - top) - log_s);
      }
    }
  }
  if (l == 0) part[warp] = cross;
  __syncthreads();
  cross = 0.0f;
  for (int k = 0; k < 8; ++k) cross += part[k];
  if (live && threadIdx.x == 0) row_loss[t] = T * T * (s.konst[t] - cross);
  if (!loss) return;
  __threadfence();
  __syncthreads();
  unsigned none;
  if (threadIdx.x == 0) last = lm_count_out(ticket, gridDim.x, 0, &none);
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum_losses<256>(loss, row_loss, M, s.scalars->count, mean);
}

// Before the backward walk.  Block 0: what the rows' gradients are multiplied by.  The halves of G hold 2^14 u (p - q), u = 1, or with
// a gradient per row that row's share of a power of two P above the largest; the rest goes into the products' own factors.  It
// also clears the steps' counters.  The other blocks (if any): zeros for dx of the rows that do not count, a warp per row.
__global__ void __launch_bounds__(1024) begin_backward_kernel(const float* __restrict__ upstream, int reduction, float T, LmSaved s, int* counters,
                                                              int steps, float* __restrict__ dx, long long M, long long E) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  if (blockIdx.x > 0) {
    for (long long t = (long long)(blockIdx.x - 1) * 32 + (threadIdx.x >> 5); t < M; t += (long long)(gridDim.x - 1) * 32)
      if (s.weight[t] == 0.0f)
        for (long long e = threadIdx.x & 31; e < E; e += 32) dx[t * E + e] = 0.0f;
    return;
  }
  __shared__ unsigned part[32];
  const int n = s.scalars->count;
  for (int i = threadIdx.x; i < steps; i += 1024) counters[i] = 0;
  float P = 1.0f;
  if (reduction == GT_REDUCE_NONE) {
    unsigned m = 0;
    for (int i = threadIdx.x; i < n; i += 1024) {
      const unsigned b = __float_as_uint(upstream[s.row_of[i]]) & 0x7fffffffu;
      if (b < 0x7f800000u && b > m) m = b;
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xffffffffu, part[threadIdx.x & 31]);
    if (m) { int e = (int)(m >> 23) - 126; P = ldexpf(1.0f, e < -100 ? -100 : e > 127 ? 127 : e); }
  }
  for (int i = threadIdx.x; i < n; i += 1024) {
    const float u = (reduction == GT_REDUCE_NONE ? upstream[s.row_of[i]] / P : 1.0f) * 16384.0f;
    s.factor[i] = make_float2(u / s.stats[i].y, u);
  }
  if (threadIdx.x == 0) {
    float c = reduction == GT_REDUCE_NONE ? P : upstream[0];
    if (reduction == GT_REDUCE_MEAN && n > 0) c /= (float)n;
    c *= T;
    s.scalars->dx = ldexpf(c, scale_exponent(s.scalars->amax_w) - 14);
    s.scalars->dw = ldexpf(c, scale_exponent(s.scalars->amax_x) - 14);
  }
}

// to (+)= the shares of a piece, in order: (n_shares, M, E).  A block per row and 256 columns; dx: the rows that count, elsewhere all M.
__global__ void __launch_bounds__(256) add_shares_kernel(float* __restrict__ to, const float* __restrict__ shares, int n_shares, long long M, long long E,
                                                         int add, const int* __restrict__ row_of, const int* __restrict__ count) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const long long i = blockIdx.x;
  if (count && i >= *count) return;
  const long long e = (long long)blockIdx.y * 256 + threadIdx.x;
  if (e >= E) return;
  float* out = to + (row_of ? (long long)row_of[i] : i) * E + e;
  float a = add ? *out : 0.0f;
#pragma unroll 8
  for (int j = 0; j < n_shares; ++j) a += shares[((long long)j * M + i) * E + e];
  *out = a;
}

bool bad_width(long long E) { return E <= 0 || E >= (1 << 24); }

bool bad_precision(int p) { return p != GT_PREC_TF32 && p != GT_PREC_TF32X3 && p != GT_PREC_FP32; }

// How a linear form's work is cut up, and where everything lies.
struct Linear {
  LmSaved s;
  LmProblem p;
  float* row_loss;
  float* dx_part;                  // few rows
  bool few_rows;
  int pieces;
  size_t saved_bytes, scratch_bytes;
};
Linear linear_layout(gt_ctx* ctx, void* saved, void* scratch, long long M, long long V, long long E, long long K, int precision) {
  Linear l;
  memset(&l, 0, sizeof(l));
  LmProblem& p = l.p;
  p.M = M; p.V = V; p.E = E; p.K = (int)K;
  l.few_rows = gt_lm_few_rows(M, V, E);
  if (l.few_rows) {
    LmCarve c = {(char*)saved, 0}, f = {(char*)scratch, 0};
    l.s = lm_saved(c, M, K);
    l.saved_bytes = c.at;
    LmCarve b = f;
    l.row_loss = f.take<float>(M);
    p.partial = f.take<float2>((size_t)gt_lm_rows_parts(ctx, M, V, false) * M);
    l.dx_part = b.take<float>((size_t)gt_lm_rows_parts(ctx, M, V, true) * M * E);
    l.scratch_bytes = f.at > b.at ? f.at : b.at;
    return l;
  }
  p.products = precision == GT_PREC_TF32 ? 1 : 3;
  p.pitch_e = (E + 7) / 8 * 8;
  // Words of a piece: what PIECE_BYTES hold of G for M rows (two pieces of it exist at a time), in whole tiles.
  p.words = PIECE_BYTES / 4 / M / LM_TILE * LM_TILE;
  if (p.words < LM_TILE) p.words = LM_TILE;
  if (p.words > V) p.words = V;
  p.pitch_v = (p.words + 7) / 8 * 8;
  l.pieces = (int)((V + p.words - 1) / p.words);
  p.dx_split = lm_shares((p.words + LM_KBLOCK - 1) / LM_KBLOCK, lm_step_stages(p, p.words, l.pieces > 1 ? p.words : 0), ctx->sm_count / 2);
  // dW's shares, step by step: the most that a step needs (full pieces beside a full one, beside the last one; the last one alone)
  long long dw_rows = 0;
  for (long long piece = l.pieces > 3 ? l.pieces - 3 : 0; piece < l.pieces; ++piece) {
    const long long n = lm_dw_split(ctx, p, lm_piece_words(p, piece), lm_piece_words(p, piece + 1)) * lm_piece_words(p, piece);
    if (n > lm_piece_words(p, piece) && n > dw_rows) dw_rows = n;
  }

  LmCarve c = {(char*)saved, 0};
  l.s = lm_saved(c, M, K);
  p.x.hi = c.take<uint16_t>(M * p.pitch_e);
  p.w.hi = c.take<uint16_t>(V * p.pitch_e);
  if (p.products == 3) { p.x.lo = c.take<uint16_t>(M * p.pitch_e); p.w.lo = c.take<uint16_t>(V * p.pitch_e); }
  l.saved_bytes = c.at;

  LmCarve f = {(char*)scratch, 0};                       // the forward pass and the backward pass use it in turn
  p.counters = f.take<int>(l.pieces + 1);
  LmCarve b = f;
  l.row_loss = f.take<float>(M);
  p.partial = f.take<float2>((V + LM_TILE - 1) / LM_TILE * 2 * M);
  p.target_z = f.take<float>(M * K);
  for (int i = 0; i < (l.pieces > 1 ? 2 : 1); ++i) {
    p.g[i].hi = b.take<uint16_t>(M * p.pitch_v);
    if (p.products == 3) p.g[i].lo = b.take<uint16_t>(M * p.pitch_v);
  }
  if (p.dx_split > 1) p.dx_partial = b.take<float>(p.dx_split * M * E);
  if (dw_rows > 0) p.dw_partial = b.take<float>(dw_rows * E);
  l.scratch_bytes = f.at > b.at ? f.at : b.at;
  p.scalars = l.s.scalars; p.row_of = l.s.row_of; p.stats = l.s.stats; p.factor = l.s.factor; p.ids = l.s.ids; p.q = l.s.q;
  return l;
}

LmRows rows_problem(const Linear& l, const float* x, const float* w, long long M, long long V, long long E, long long K, float T, int reduction) {
  LmRows r;
  memset(&r, 0, sizeof(r));
  r.M = (int)M; r.V = (int)V; r.E = (int)E; r.K = (int)K;
  r.x = x; r.w = w; r.T = T; r.s = l.s; r.partial = l.p.partial; r.reduction = reduction;
  return r;
}

int prepare_linear(gt_ctx* ctx, const LmSaved& s, int* counters, float* row_loss, const float* targets, float ignore, const float* ids,
                   const float* teacher, long long M, long long V, long long K, float T) {
  if (targets) {
    GT_CUDA_OK(ctx, gt_launch_overlapped(hard_targets_kernel, dim3(1), dim3(1024), 0, ctx->stream, targets, M, V, ignore, s, row_loss, counters, ctx->d_status));
  } else {
    int rc = gt_lm_top_targets(ctx, s, row_loss, ids, teacher, M, V, K, T);
    if (rc != GT_OK) return rc;
    GT_CUDA_OK(ctx, gt_launch_overlapped(compact_rows_kernel, dim3(1), dim3(1024), 0, ctx->stream, M, s, counters));
  }
  ctx->launches += 1;
  return GT_OK;
}

int linear_forward(gt_ctx* ctx, float* loss, void* saved, void* scratch, const float* x, const float* w, const float* targets, float ignore,
                   const float* ids, const float* teacher, int64_t M, int64_t V, int64_t E, int64_t K, float T, int reduction, int precision) {
  const Linear l = linear_layout(ctx, saved, scratch, M, V, E, K, precision);
  const LmSaved& s = l.s;
  float* rows = reduction == GT_REDUCE_NONE ? loss : l.row_loss;
  float* sum = reduction == GT_REDUCE_NONE ? nullptr : loss;
  const int mean = reduction == GT_REDUCE_MEAN;
  if (l.few_rows) {
    LmRows r = rows_problem(l, x, w, M, V, E, K, T, reduction);
    r.parts = gt_lm_rows_parts(ctx, M, V, false);
    r.ticket = lm_ticket(ctx);
    if (!targets) {
      int rc = gt_lm_top_targets(ctx, s, rows, ids, teacher, M, V, K, T);
      if (rc == GT_OK) rc = gt_lm_rows_forward(ctx, r);
      if (rc != GT_OK) return rc;
      GT_CUDA_OK(ctx, gt_launch_overlapped(join_blocks_kernel, dim3((unsigned)M), dim3(256), 0, ctx->stream, rows, sum, x, w, M, (int)E, (int)K, T, mean, l.p.partial,
                                           r.parts, s, lm_ticket(ctx)));
      ctx->launches += 1;
      return GT_OK;
    }
    r.targets = targets; r.ignore = ignore;
    r.row_loss = rows;
    r.loss = sum;
    return gt_lm_rows_forward(ctx, r);
  }
  int rc = prepare_linear(ctx, s, l.p.counters, rows, targets, ignore, ids, teacher, M, V, K, T);
  if (rc != GT_OK) return rc;
  const long long most = 8ll * ctx->sm_count;
  auto blocks = [&](long long n) { return (int)((n + 7) / 8 < most ? (n + 7) / 8 : most); };
  const int bx = blocks(M), bw = blocks(V);
  GT_CUDA_OK(ctx, gt_launch_overlapped(largest_kernel, dim3((unsigned)(bx + bw)), dim3(256), 0, ctx->stream, x, w, V, E, s, bx));
  GT_CUDA_OK(ctx, gt_launch_overlapped(split_kernel, dim3((unsigned)(bx + bw)), dim3(256), 0, ctx->stream, x, w, M, V, E, l.p.pitch_e, s, l.p.x, l.p.w, l.p.products, T, bx));
  ctx->launches += 2;
  rc = gt_lm_stats(ctx, l.p);
  if (rc != GT_OK) return rc;
  GT_CUDA_OK(ctx, gt_launch_overlapped(join_tiles_kernel, dim3((unsigned)((M + 31) / 32)), dim3(1024), 0, ctx->stream, l.p.partial,
                                       (int)((V + LM_TILE - 1) / LM_TILE * 2), l.p.target_z, rows, sum, M, (int)K, T, mean, s, lm_ticket(ctx)));
  ctx->launches += 1;
  return GT_OK;
}

}  // namespace

int gt_lm_top_targets(gt_ctx* ctx, const LmSaved& s, float* row_loss, const float* ids, const float* teacher, long long M, long long V, long long K,
                      float T) {
  GT_CUDA_OK(ctx, gt_launch_overlapped(top_targets_kernel, dim3((unsigned)((M + 3) / 4)), dim3(128), (size_t)4 * 2 * K * 4, ctx->stream, ids, teacher, M, V, (int)K, 1.0f / T, s, row_loss, lm_ticket(ctx), ctx->d_status));
  ctx->launches += 1;
  return GT_OK;
}

extern "C" int gt_linear_loss_sizes(gt_ctx* ctx, int64_t M, int64_t V, int64_t E, int64_t K, int precision, size_t* saved, size_t* scratch) {
  if (!ctx || !saved || !scratch || lm_bad_sizes(M, V, K) || bad_width(E) || bad_precision(precision)) return GT_ERR_INVALID_ARG;
  const Linear l = linear_layout(ctx, nullptr, nullptr, M, V, E, K, precision);
  *saved = l.saved_bytes;
  *scratch = l.scratch_bytes;
  return GT_OK;
}

extern "C" int gt_linear_cross_entropy(gt_ctx* ctx, float* loss, void* saved, void* scratch, const float* x, const float* w, const float* targets,
                                       int64_t M, int64_t V, int64_t E, float ignore_index, int reduction, int precision) {
  if (!ctx || !loss || !saved || !scratch || !x || !w || !targets || lm_bad_sizes(M, V, 1) || bad_width(E) || lm_bad_reduction(reduction) ||
      bad_precision(precision)) return GT_ERR_INVALID_ARG;
  return linear_forward(ctx, loss, saved, scratch, x, w, targets, ignore_index, nullptr, nullptr, M, V, E, 1, 1.0f, reduction, precision);
}

extern "C" int gt_linear_topk_distillation(gt_ctx* ctx, float* loss, void* saved, void* scratch, const float* x, const float* w, const float* ids,
                                           const float* teacher, int64_t M, int64_t V, int64_t E, int64_t K, float temperature, int reduction,
                                           int precision) {
  if (!ctx || !loss || !saved || !scratch || !x || !w || !ids || !teacher || lm_bad_sizes(M, V, K) || bad_width(E) || lm_bad_reduction(reduction) ||
      lm_bad_temperature(temperature) || bad_precision(precision)) return GT_ERR_INVALID_ARG;
  return linear_forward(ctx, loss, saved, scratch, x, w, nullptr, 0.0f, ids, teacher, M, V, E, K, temperature, reduction, precision);
}

extern "C" int gt_linear_loss_backward(gt_ctx* ctx, float* dx, float* dw, void* saved, void* scratch, const float* x, const float* w,
                                       const float* upstream, int64_t M, int64_t V, int64_t E, int64_t K, float temperature, int reduction,
                                       int precision, int acc_dx, int acc_dw) {
  if (!ctx || !saved || !scratch || !x || !w || !upstream || lm_bad_sizes(M, V, K) || bad_width(E) || lm_bad_reduction(reduction) ||
      lm_bad_temperature(temperature) || bad_precision(precision)) return GT_ERR_INVALID_ARG;
  if (!dx && !dw) return GT_OK;
  Linear l = linear_layout(ctx, saved, scratch, M, V, E, K, precision);
  if (l.few_rows) {
    LmRows r = rows_problem(l, x, w, M, V, E, K, temperature, reduction);
    r.parts = gt_lm_rows_parts(ctx, M, V, true);
    r.upstream = upstream; r.dw = dw; r.acc_dw = acc_dw;
    r.dx_part = dx ? l.dx_part : nullptr;
    return gt_lm_rows_backward(ctx, r, dx, acc_dx);
  }
  LmProblem& p = l.p;
  p.dx = dx; p.dw = dw; p.acc_dx = acc_dx; p.acc_dw = acc_dw;
  const long long zero_blocks = dx && !acc_dx ? ((M + 31) / 32 < ctx->sm_count ? (M + 31) / 32 : ctx->sm_count) : 0;
  GT_CUDA_OK(ctx, gt_launch_overlapped(begin_backward_kernel, dim3((unsigned)(1 + zero_blocks)), dim3(1024), 0, ctx->stream, upstream, reduction, temperature, l.s, p.counters, l.pieces + 1, dx, M, E));
  ctx->launches += 1;
  for (int piece = 0; piece <= l.pieces; ++piece) {
    int rc = gt_lm_step(ctx, p, piece);
    if (rc != GT_OK) return rc;
    if (piece > 0 && dx && p.dx_split > 1) {
      GT_CUDA_OK(ctx, gt_launch_overlapped(add_shares_kernel, dim3((unsigned)M, (unsigned)((E + 255) / 256)), dim3(256), 0, ctx->stream, dx, p.dx_partial, p.dx_split, M, E, acc_dx || piece > 1,
                                           l.s.row_of, &l.s.scalars->count));
      ctx->launches += 1;
    }
    const long long words = lm_piece_words(p, piece - 1);
    const int dw_split = lm_dw_split(ctx, p, words, lm_piece_words(p, piece));
    if (dw && dw_split > 1) {
      GT_CUDA_OK(ctx, gt_launch_overlapped(add_shares_kernel, dim3((unsigned)words, (unsigned)((E + 255) / 256)), dim3(256), 0, ctx->stream, dw + (long long)(piece - 1) * p.words * E, p.dw_partial,
                                           dw_split, words, E, acc_dw, (const int*)nullptr, (const int*)nullptr));
      ctx->launches += 1;
    }
  }
  return GT_OK;
}
