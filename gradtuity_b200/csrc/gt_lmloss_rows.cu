// The linear losses (gt_lmloss.cu) for few rows, or for little work, in 32-bit multiply-adds: what a row or a few cost is reading W
// (and writing dW), and a small problem is launches and latencies; the tensor-core path pays for splitting W into halves first,
// and for tiles of 256 rows.
//
// One row: a warp per word, in registers for all that is done with it.  More: a block of eight warps takes 32 words at a time.  The E columns are shared out over the lanes of CW warps (1, 2, 4 or 8), C columns
// each, and the words over the 8 / CW groups of such warps; MT rows of x stay in registers.  Every lane multiplies its columns of a
// few words with its columns of the rows, the 32 lanes add up by exchanging halves (one exchange per value instead of five), and
// the warps' sums meet in shared memory.  So W is read once, straight from memory in whole lines, and no operand passes through
// shared memory.  Loads are never guarded: addresses past the end are pulled back, and what comes of them is not used.
// Forward: running maximum and sum of each row; the last block to end joins the blocks' and, for cross entropy, takes the losses.
// Backward: the logits again, G = c (p - q), then from the same words dx += G w (in registers, one partial sum per block, added up
// in the blocks' order by a second kernel) and dW = G^T x, written straight out.
// More than MT rows: the rows' tiles one after the other, adding to dW.

#include "gt_lmloss.h"

namespace {

constexpr int THREADS = 256, WARPS = 8, WORDS = 32;

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

// N values per lane, a power of two up to 64, summed over the lanes: afterwards lane l holds the sums max(1, N / 32) l .. (N >= 32),
// or the sum l N / 32 (N < 32).
template <int N>
__device__ __forceinline__ void lanes_sum(float (&v)[N]) {
  const int lane = threadIdx.x & 31;
  int n = N;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (n > 1) {
      n >>= 1;
      const bool up = (lane & o) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < n) {
          const float send = up ? v[i] : v[i + n], keep = up ? v[i + n] : v[i];
          v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
      }
    } else {
      v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    }
  }
}

// Words loaded at a time, and multiplied at a time.
template <int MT, int C> struct Words {
  static constexpr int SUM = MT == 4 ? 8 : 4;
  static constexpr int LOAD = MT == 16 && C <= 2 ? 8 : SUM;
};

struct Rows {
  LmRows r;
  int* status;
};

// Where a thread stands: its group of warps, its first column, its group's words among the block's.
struct Place {
  int part, group, col0, word0, words;
};
template <int C>
__device__ __forceinline__ Place place_of(int cw) {
  const int warp = threadIdx.x >> 5;
  Place p;
  p.part = warp & (cw - 1);
  p.group = warp / cw;
  p.col0 = p.part * 32 * C + (threadIdx.x & 31);
  p.words = WORDS * cw / WARPS;
  p.word0 = p.group * p.words;
  return p;
}

// The block's logits of its words and MT rows: each warp leaves its columns' share in red[row][word].
template <int MT, int C>
__device__ __forceinline__ void dots(const float (&x)[MT][C], const float* __restrict__ w, long long v0, int V, int E, const Place& at, float* red) {
  constexpr int WS = Words<MT, C>::SUM, WL = Words<MT, C>::LOAD, N = WS * MT;
  static_assert(N >= 32, "every lane holds a sum");
  const int lane = threadIdx.x & 31;
  const float* col[C];
#pragma unroll
  for (int c = 0; c < C; ++c) col[c] = w + min(at.col0 + 32 * c, E - 1);        // x is 0 past the last column
#pragma unroll 1
  for (int s = 0; s < at.words; s += WL) {
    float b[WL][C];
#pragma unroll
    for (int i = 0; i < WL; ++i) {
      const long long v = min(v0 + at.word0 + s + i, (long long)V - 1) * E;
#pragma unroll
      for (int c = 0; c < C; ++c) b[i][c] = col[c][v];
    }
#pragma unroll
    for (int h = 0; h < WL; h += WS) {
      float a[N];
#pragma unroll
      for (int i = 0; i < WS; ++i)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          float t = x[m][0] * b[h + i][0];
#pragma unroll
          for (int c = 1; c < C; ++c) t = fmaf(x[m][c], b[h + i][c], t);
          a[i * MT + m] = t;
        }
      lanes_sum<N>(a);
#pragma unroll
      for (int j = 0; j < N / 32; ++j) {
        const int k = lane * (N / 32) + j, word = s + h + k / MT;                // which sum this lane holds
        if (word < at.words) red[(k % MT) * WORDS + at.word0 + word] = a[j];
      }
    }
  }
}

template <int MT, int C>
__device__ __forceinline__ void load_rows(float (&x)[MT][C], const float* __restrict__ src, int m0, int M, int E, int col0, const float* weight) {
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const bool row = m0 + m < M && (weight == nullptr || weight[m0 + m] != 0.0f);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int col = col0 + 32 * c;
      x[m][c] = row && col < E ? src[(long long)(m0 + m) * E + col] : 0.0f;
    }
  }
}

// Row t's (m log2 e, s) from the blocks' partial ones, by `lanes` lanes of a warp that stand together.
__device__ __forceinline__ float2 join_parts(const float2* partial, int parts, long long M, long long t, int l, int lanes) {
  float m = -INFINITY, s = 0.0f;
#pragma unroll 8
  for (int j = l; j < parts; j += lanes) {
    const float2 b = __ldcg(partial + (long long)j * M + t);
    const float top = fmaxf(m, b.x);
    if (top == -INFINITY) { s += b.y; continue; }
    s = s * gt_ex2(m - top) + b.y * gt_ex2(b.x - top);
    m = top;
  }
  float top = m;
  for (int o = lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  s = top == -INFINITY ? s : s * gt_ex2(m - top);
  for (int o = lanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return make_float2(top, s);
}

template <int MT, int C>
__global__ void __launch_bounds__(THREADS) few_rows_forward_kernel(const Rows a) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const LmRows& p = a.r;
  __shared__ float red[2][WARPS][MT * WORDS];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Place at = place_of<C>(p.cw);
  const int m0 = blockIdx.y * MT;
  float x[MT][C];
  load_rows<MT, C>(x, p.x, m0, p.M, p.E, at.col0, nullptr);
  constexpr int ROWS = (MT + WARPS - 1) / WARPS;                // rows whose maximum and sum a warp keeps
  float m[ROWS], s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) { m[i] = -INFINITY; s[i] = 0.0f; }
  const float l2 = 1.4426950408889634f / p.T;
  int buf = 0;
  for (long long v0 = (long long)blockIdx.x * WORDS; v0 < p.V; v0 += (long long)gridDim.x * WORDS, buf ^= 1) {
    dots<MT, C>(x, p.w, v0, p.V, p.E, at, red[buf][at.part]);
    __syncthreads();                                            // the other buffer is free: its readers passed this barrier
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = warp + i * WARPS;
      if (r < MT) {
        float z = 0.0f;
        for (int k = 0; k < p.cw; ++k) z += red[buf][k][r * WORDS + lane];
        z = v0 + lane < p.V ? z * l2 : -INFINITY;
        const float top = fmaxf(m[i], warp_max(z));
        if (top != -INFINITY) {
          s[i] = s[i] * gt_ex2(m[i] - top) + warp_sum(gt_ex2(z - top));
          m[i] = top;
        } else {
          s[i] += warp_sum(z == -INFINITY ? 0.0f : z);          // a NaN is no maximum, but it counts
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = warp + i * WARPS;
    if (r < MT && m0 + r < p.M && lane == 0) p.partial[(long long)blockIdx.x * p.M + m0 + r] = make_float2(m[i], s[i]);
  }
  if (!p.targets) return;                                       // distillation: the rows' kernels do the rest

  // ---- cross entropy: the last block takes the losses
  __threadfence();
  __syncthreads();
  unsigned none;
  if (threadIdx.x == 0) last = lm_count_out(p.ticket, gridDim.x * gridDim.y, 0, &none);
  __syncthreads();
  if (!last) return;
  __threadfence();
  // a row by a warp, or by eight lanes where rows are short: four rows a warp then, with their loads in flight together
  const int lanes = p.E <= 256 ? 8 : 32, l = lane & (lanes - 1), per_block = THREADS / lanes;
  double total = 0.0;
  int n = 0;
  for (int t0 = 0; t0 < p.M; t0 += per_block) {
    const int t = t0 + threadIdx.x / lanes;
    const bool row = t < p.M;
    const float f = row ? p.targets[t] : p.ignore;
    const bool in_range = f >= 0.0f && f < (float)p.V, used = f != p.ignore && in_range;
    const float* xr = p.x + (long long)(used ? t : 0) * p.E;
    const float* wr = p.w + (long long)(used ? (int)f : 0) * p.E;
    float z = 0.0f;
#pragma unroll 24
    for (int e = l; e < p.E; e += lanes) z = fmaf(xr[e], wr[e], z);
    const float2 st = join_parts(p.partial, gridDim.x, p.M, row ? t : 0, l, lanes);
    for (int o = lanes / 2; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (!row || l != 0) continue;
    float loss = 0.0f;
    if (used) {
      loss = logf(st.y) - (z - st.x * 0.6931471805599453f);
      p.s.stats[t] = st;
      total += loss;
      ++n;
    }
    if (f != p.ignore && !in_range) atomicExch(a.status, GT_ERR_INVALID_ARG);
    p.s.ids[t] = used ? (int)f : LM_UNUSED;
    p.s.q[t] = used ? 1.0f : 0.0f;
    p.s.weight[t] = used ? 1.0f : 0.0f;
    if (p.row_loss) p.row_loss[t] = loss;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  __shared__ double totals[WARPS];
  __shared__ int counts[WARPS];
  if (lane == 0) { totals[warp] = total; counts[warp] = n; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < WARPS; ++k) { total += totals[k]; n += counts[k]; }
    p.s.scalars->count = n;
    if (p.loss) *p.loss = (float)(p.reduction == GT_REDUCE_MEAN && n > 0 ? total / n : total);
  }
}

template <int MT, int C>
__global__ void __launch_bounds__(THREADS) few_rows_backward_kernel(const Rows a) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const LmRows& p = a.r;
  // the warps' shares of the logits; at the end, dx of half the groups of warps (4 x 32 columns a lane a warp, 4 warps)
  __shared__ float pool[MT * 512 > WARPS * MT * WORDS ? MT * 512 : WARPS * MT * WORDS];
  float (*const red)[MT * WORDS] = reinterpret_cast<float (*)[MT * WORDS]>(pool);
  __shared__ __align__(16) float gs[WORDS * MT];                // G, word by word
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Place at = place_of<C>(p.cw);
  const float l2 = 1.4426950408889634f / p.T;
  constexpr int ROWS = (MT + WARPS - 1) / WARPS;
  for (int m0 = 0; m0 < p.M; m0 += MT) {
    float x[MT][C], dx[MT][C];
    load_rows<MT, C>(x, p.x, m0, p.M, p.E, at.col0, p.s.weight);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < C; ++c) dx[m][c] = 0.0f;
    // the rows whose G this warp makes
    float top[ROWS], f[ROWS], cq[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int t = m0 + warp + i * WARPS;
      top[i] = 0.0f; f[i] = 0.0f; cq[i] = 0.0f;
      if (warp + i * WARPS < MT && t < p.M && p.s.weight[t] != 0.0f) {
        float c = p.T * (p.reduction == GT_REDUCE_NONE ? p.upstream[t] : p.upstream[0]);
        if (p.reduction == GT_REDUCE_MEAN) c /= (float)p.s.scalars->count;
        const float2 st = p.s.stats[t];
        top[i] = st.x; f[i] = c / st.y; cq[i] = c;
      }
    }
    for (long long v0 = (long long)blockIdx.x * WORDS; v0 < p.V; v0 += (long long)gridDim.x * WORDS) {
      dots<MT, C>(x, p.w, v0, p.V, p.E, at, red[at.part]);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = warp + i * WARPS;
        if (r < MT) {
          float z = 0.0f;
          for (int k = 0; k < p.cw; ++k) z += red[k][r * WORDS + lane];
          const int t = m0 + r, v = (int)v0 + lane;
          float g = 0.0f;
          if (t < p.M && p.s.weight[t] != 0.0f && v < p.V) {
            g = f[i] * gt_ex2(z * l2 - top[i]);
            const int* ids = p.s.ids + (long long)t * p.K;
            int lo = 0, hi = p.K;                               // the row's targets at this word
            while (lo < hi) { const int mid = (lo + hi) >> 1; if (ids[mid] < v) lo = mid + 1; else hi = mid; }
            for (; lo < p.K && ids[lo] == v; ++lo) g -= cq[i] * p.s.q[(long long)t * p.K + lo];
          }
          gs[lane * MT + r] = g;
        }
      }
      __syncthreads();
      const int words = min(at.words, (int)min((long long)WORDS, p.V - v0) - at.word0);
      const bool add = p.acc_dw || m0 > 0;
      constexpr int GROUP = 4;                                  // words whose loads go out together, ahead of the stores
#pragma unroll 1
      for (int i0 = 0; i0 < words; i0 += GROUP) {
        float b[GROUP][C], d[GROUP][C];
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
          const long long row = (v0 + at.word0 + min(i0 + i, words - 1)) * p.E;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const int col = min(at.col0 + 32 * c, p.E - 1);
            b[i][c] = p.dx_part ? __ldg(p.w + row + col) : 0.0f;      // read a moment ago: in L1
            d[i][c] = add && p.dw ? p.dw[row + col] : 0.0f;
          }
        }
#pragma unroll
        for (int i = 0; i < GROUP; ++i) {
          if (i0 + i >= words) break;
          const float* gi = gs + (at.word0 + i0 + i) * MT;
#pragma unroll
          for (int m = 0; m < MT; m += 4) {
            float g[4];
            *reinterpret_cast<float4*>(g) = *reinterpret_cast<const float4*>(gi + m);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
              for (int c = 0; c < C; ++c) {
                dx[m + k][c] = fmaf(g[k], b[i][c], dx[m + k][c]);
                d[i][c] = fmaf(g[k], x[m + k][c], d[i][c]);
              }
          }
        }
        if (p.dw) {
#pragma unroll
          for (int i = 0; i < GROUP; ++i)
#pragma unroll
            for (int c = 0; c < C; ++c)
              if (i0 + i < words && at.col0 + 32 * c < p.E) p.dw[(v0 + at.word0 + i0 + i) * p.E + at.col0 + 32 * c] = d[i][c];
        }
      }
      // gs is written again behind the next block's first barrier; red behind this block's second one
    }
    if (p.dx_part) {
      // the groups' sums, halving their number each time: the order is the same every time
      const int cols = p.cw * 32 * C, mine = at.part * 32 * C + lane;
      for (int half = WARPS / p.cw / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (at.group >= half && at.group < 2 * half) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < C; ++c) pool[((at.group - half) * MT + m) * cols + mine + 32 * c] = dx[m][c];
        }
        __syncthreads();
        if (at.group < half) {
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int c = 0; c < C; ++c) dx[m][c] += pool[(at.group * MT + m) * cols + mine + 32 * c];
        }
      }
      if (at.group == 0) {
        float* to = p.dx_part + ((long long)blockIdx.x * p.M + m0) * p.E;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const int col = at.col0 + 32 * c;
            if (m0 + m < p.M && col < p.E) to[(long long)m * p.E + col] = dx[m][c];
          }
      }
      __syncthreads();
    }
  }
}

// ---- one row ------------------------------------------------------------------------------------------
// A warp takes whole words, two at a time: loads, dot product and, in the backward pass, dx += g w and dW = g x need no other warp, so
// nothing waits but for memory.  NC: 128 columns each, four a lane; side by side for 16-byte loads (VEC), else 32 apart.
template <int NC, bool VEC>
struct Row {
  float v[NC][4];
  static __device__ __forceinline__ int column(int i, int j) { return i * 128 + (VEC ? 4 * (threadIdx.x & 31) + j : 32 * j + (threadIdx.x & 31)); }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = 0.0f;
  }
  __device__ __forceinline__ void load(const float* __restrict__ src, int E) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      if (VEC) {
        const int col = column(i, 0);
        const float4 a = col < E ? *reinterpret_cast<const float4*>(src + col) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[i][0] = a.x; v[i][1] = a.y; v[i][2] = a.z; v[i][3] = a.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = column(i, j) < E ? src[column(i, j)] : 0.0f;
      }
    }
  }
  __device__ __forceinline__ float dot(const Row& o) const {
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) z = fmaf(v[i][j], o.v[i][j], z);
    return z;
  }
};

template <int NC, bool VEC>
__global__ void __launch_bounds__(THREADS) one_row_forward_kernel(const Rows a) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const LmRows& p = a.r;
  __shared__ float zs[WARPS];
  __shared__ float2 ms[WARPS];
  __shared__ int last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float l2 = 1.4426950408889634f / p.T;
  Row<NC, VEC> x;
  x.load(p.x, p.E);
  float m = -INFINITY, s = 0.0f;
  auto add = [&](float2 b) {
    const float top = fmaxf(m, b.x);
    if (top == -INFINITY) { s += b.y; return; }                 // a NaN is no maximum, but it counts
    s = s * gt_ex2(m - top) + b.y * gt_ex2(b.x - top);
    m = top;
  };
  const int stride = gridDim.x * WARPS;
  for (int v = blockIdx.x * WARPS + warp; v < p.V; v += 2 * stride) {
    const bool two = v + stride < p.V;
    Row<NC, VEC> w0, w1;
    w0.load(p.w + (long long)v * p.E, p.E);
    w1.load(p.w + (long long)(two ? v + stride : v) * p.E, p.E);
    const float z0 = warp_sum(x.dot(w0)) * l2, z1 = warp_sum(x.dot(w1)) * l2;
    add(make_float2(z0, z0 == z0 ? 1.0f : z0));
    if (two) add(make_float2(z1, z1 == z1 ? 1.0f : z1));
  }
  if (lane == 0) ms[warp] = make_float2(m, s);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < WARPS; ++k) add(ms[k]);
    p.partial[blockIdx.x] = make_float2(m, s);
  }
  if (!p.targets) return;                                       // distillation: the rows' kernels do the rest
  unsigned none;
  if (threadIdx.x == 0) last = lm_count_out(p.ticket, gridDim.x, 0, &none);
  __syncthreads();
  if (!last) return;
  __threadfence();
  const float f = p.targets[0];
  const bool in_range = f >= 0.0f && f < (float)p.V, used = f != p.ignore && in_range;
  const float* wr = p.w + (long long)(used ? (int)f : 0) * p.E;
  float z = 0.0f;
#pragma unroll 4
  for (int e = threadIdx.x; e < p.E; e += THREADS) z = fmaf(p.x[e], wr[e], z);
  m = -INFINITY; s = 0.0f;
#pragma unroll 4
  for (int j = threadIdx.x; j < (int)gridDim.x; j += THREADS) add(__ldcg(p.partial + j));
  const float top = warp_max(m);
  s = warp_sum(top == -INFINITY ? s : s * gt_ex2(m - top));
  z = warp_sum(z);
  if (lane == 0) { zs[warp] = z; ms[warp] = make_float2(top, s); }
  __syncthreads();
  if (threadIdx.x != 0) return;
  m = top;
  for (int k = 1; k < WARPS; ++k) { z += zs[k]; add(ms[k]); }
  const float loss = used ? logf(s) - (z - m * 0.6931471805599453f) : 0.0f;
  if (f != p.ignore && !in_range) atomicExch(a.status, GT_ERR_INVALID_ARG);
  p.s.stats[0] = make_float2(m, s);
  p.s.ids[0] = used ? (int)f : LM_UNUSED;
  p.s.q[0] = p.s.weight[0] = used ? 1.0f : 0.0f;
  p.s.scalars->count = used ? 1 : 0;
  if (p.row_loss) p.row_loss[0] = loss;
  if (p.loss) *p.loss = loss;
}

template <int NC, bool VEC>
__global__ void __launch_bounds__(THREADS) one_row_backward_kernel(const Rows a) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  const LmRows& p = a.r;
  __shared__ float sums[WARPS][NC * 128];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float l2 = 1.4426950408889634f / p.T;
  const bool live = p.s.weight[0] != 0.0f;
  const float c = live ? p.T * p.upstream[0] : 0.0f;            // one row: sum, mean and the row itself are the same
  const float2 st = live ? p.s.stats[0] : make_float2(0.0f, 1.0f);
  const float f = c / st.y;
  Row<NC, VEC> x, dx;
  dx.clear();
  if (live) x.load(p.x, p.E); else x.clear();
  const int first = p.s.ids[0];
  auto word = [&](const Row<NC, VEC>& w, int v, float z) {
    float g = live ? f * gt_ex2(z * l2 - st.x) : 0.0f;
    if (v == first || (p.K > 1 && live)) {                      // the row's targets at this word
      int lo = 0, hi = p.K;
      while (lo < hi) { const int mid = (lo + hi) >> 1; if (p.s.ids[mid] < v) lo = mid + 1; else hi = mid; }
      for (; lo < p.K && p.s.ids[lo] == v; ++lo) g -= c * p.s.q[lo];
    }
    float* to = p.dw + (long long)v * p.E;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int col = Row<NC, VEC>::column(i, 0);
      float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.dw && p.acc_dw) {
        if (VEC) {
          if (col < p.E) *reinterpret_cast<float4*>(d) = *reinterpret_cast<const float4*>(to + col);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) if (Row<NC, VEC>::column(i, j) < p.E) d[j] = to[Row<NC, VEC>::column(i, j)];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        dx.v[i][j] = fmaf(g, w.v[i][j], dx.v[i][j]);
        d[j] = fmaf(g, x.v[i][j], d[j]);
      }
      if (!p.dw) continue;
      if (VEC) {
        if (col < p.E) *reinterpret_cast<float4*>(to + col) = *reinterpret_cast<float4*>(d);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (Row<NC, VEC>::column(i, j) < p.E) to[Row<NC, VEC>::column(i, j)] = d[j];
      }
    }
  };
  const int stride = gridDim.x * WARPS;
  for (int v = blockIdx.x * WARPS + warp; v < p.V; v += 2 * stride) {
    const bool two = v + stride < p.V;
    Row<NC, VEC> w0, w1;
    w0.load(p.w + (long long)v * p.E, p.E);
    w1.load(p.w + (long long)(two ? v + stride : v) * p.E, p.E);
    const float z0 = warp_sum(x.dot(w0)), z1 = warp_sum(x.dot(w1));
    word(w0, v, z0);
    if (two) word(w1, v + stride, z1);
  }
  if (!p.dx_part) return;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[warp][Row<NC, VEC>::column(i, j)] = dx.v[i][j];
  __syncthreads();
  for (int e = threadIdx.x; e < p.E; e += THREADS) {
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) t += sums[k][e];
    p.dx_part[(long long)blockIdx.x * p.E + e] = t;
  }
}

// dx (+)= the blocks' shares: 32 columns of a row per block, a warp takes every 32nd share, and the warps are added in order.
__global__ void __launch_bounds__(1024) few_rows_dx_kernel(float* __restrict__ dx, const float* __restrict__ part, int parts, long long M, int E, int add) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  __shared__ float sums[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.x * 32 + lane;
  const long long t = blockIdx.y;
  float s = 0.0f;
  if (col < E) {
#pragma unroll 8
    for (int j = warp; j < parts; j += 32) s += part[((long long)j * M + t) * E + col];
  }
  sums[warp][lane] = s;
  __syncthreads();
  s = warp_sum(sums[lane][warp]);                               // the 32 warps' sums of column `warp`
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < E) dx[t * E + mine] = add ? dx[t * E + mine] + s : s;
}

template <int MT, int C>
int launch_as(gt_ctx* ctx, const Rows& a, bool backward) {
  const LmRows& p = a.r;
  if (backward) GT_CUDA_OK(ctx, gt_launch_overlapped(few_rows_backward_kernel<MT, C>, dim3((unsigned)p.parts), dim3(THREADS), 0, ctx->stream, a));
  else GT_CUDA_OK(ctx, gt_launch_overlapped(few_rows_forward_kernel<MT, C>, dim3((unsigned)p.parts, (unsigned)((p.M + MT - 1) / MT)), dim3(THREADS), 0, ctx->stream, a));
  ctx->launches += 1;
  return GT_OK;
}
template <int NC>
int launch_one(gt_ctx* ctx, const Rows& a, bool backward) {
  const LmRows& p = a.r;
  const bool vec = p.E % 4 == 0 && (((uintptr_t)p.x | (uintptr_t)p.w | (uintptr_t)p.dw) & 15) == 0;
  void (*kernel)(const Rows) = backward ? (vec ? one_row_backward_kernel<NC, true> : one_row_backward_kernel<NC, false>)
                                        : (vec ? one_row_forward_kernel<NC, true> : one_row_forward_kernel<NC, false>);
  GT_CUDA_OK(ctx, gt_launch_overlapped(kernel, dim3((unsigned)p.parts), dim3(THREADS), 0, ctx->stream, a));
  ctx->launches += 1;
  return GT_OK;
}
template <int MT>
int launch_for(gt_ctx* ctx, const Rows& a, bool backward) {
  switch (a.r.c) {
    case 1: return launch_as<MT, 1>(ctx, a, backward);
    case 2: return launch_as<MT, 2>(ctx, a, backward);
    case 3: return launch_as<MT, 3>(ctx, a, backward);
    default: return launch_as<MT, 4>(ctx, a, backward);
  }
}
int launch(gt_ctx* ctx, const LmRows& p, bool backward) {
  Rows a = {p, ctx->d_status};
  // As many columns a lane as there are, up to four: adding up over lanes and warps costs the same for one column as for four.
  const int wide = (p.E + 127) / 128;
  a.r.cw = wide <= 1 ? 1 : wide <= 2 ? 2 : wide <= 4 ? 4 : 8;
  a.r.c = (p.E + 32 * a.r.cw - 1) / (32 * a.r.cw);
  if (p.M == 1) {
    switch ((p.E + 127) / 128) {
      case 1: return launch_one<1>(ctx, a, backward);
      case 2: return launch_one<2>(ctx, a, backward);
      case 3: return launch_one<3>(ctx, a, backward);
      case 4: return launch_one<4>(ctx, a, backward);
      case 5: return launch_one<5>(ctx, a, backward);
      case 6: return launch_one<6>(ctx, a, backward);
      case 7: return launch_one<7>(ctx, a, backward);
      default: return launch_one<8>(ctx, a, backward);
    }
  }
  if (p.M <= 4) return launch_for<4>(ctx, a, backward);
  return launch_for<16>(ctx, a, backward);
}

}  // namespace

// Measured against the tensor-core path, with gradients, us (this / that): 8 x 768 x 50257 359 / 366, 16 x 768 x 50257 370 / 366,
// 16 x 256 x 8000 77 / 106, 64 x 128 x 4000 76 / 81, 64 x 256 x 4000 78 / 82, 64 x 512 x 4000 135 / 91, 128 x 128 x 4000 112 / 81.
bool gt_lm_few_rows(long long M, long long V, long long E) {
  if (E > 1024) return false;
  return M <= 16 || (M <= 64 && M * V * E <= LM_ROWS_WORK);
}

int gt_lm_rows_parts(gt_ctx* ctx, long long M, long long V, bool backward) {
  const long long words = M == 1 ? 2 * WARPS : WORDS, blocks = (V + words - 1) / words, tiles = M <= 16 ? 1 : (M + 15) / 16;
  long long most = 2ll * ctx->sm_count;                          // blocks an SM; one row of 768 x 50257: 92, 92, 95, 97 us with 2, 3, 4, 6
  if (!backward) most = (most + tiles - 1) / tiles;
  return (int)(blocks < most ? blocks : most);
}

int gt_lm_rows_forward(gt_ctx* ctx, const LmRows& p) { return launch(ctx, p, false); }

int gt_lm_rows_backward(gt_ctx* ctx, const LmRows& p, float* dx, int acc_dx) {
  int rc = launch(ctx, p, true);
  if (rc != GT_OK || !dx) return rc;
  GT_CUDA_OK(ctx, gt_launch_overlapped(few_rows_dx_kernel, dim3((unsigned)((p.E + 31) / 32), (unsigned)p.M), dim3(1024), 0, ctx->stream, dx, p.dx_part, p.parts, p.M, p.E, acc_dx));
  ctx->launches += 1;
  return GT_OK;
}
