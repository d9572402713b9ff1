// Distillation of given logits from a teacher's top logits (the formulas: gt_lmloss.cu): row kernels, bound by HBM.  A pass reads
// the (rows, C) logits once and, with gradients, writes as much: 2 x 1.65 GB for 8192 rows of 50257 words.
//
// e^((z - m) / T) is 2^(z l2 - m l2) with l2 = log2(e) / T.  Sums are in 32 bits; s and m are kept apart, so that p carries no
// rounding of a log-sum-exp.

#include "gt_lmloss.h"

namespace {

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

// A thread's running maximum m and the sum of 2^(z l2 - m l2) beside it: one multiply-add and one ex2 per logit.  m starts at
// LOW instead of -inf: words masked with -inf or with the type's lowest value then add 0 without a test.  A row whose logits are all
// at LOW or below leaves (LOW, 0); it is summed again by `row_of_low_logits`.  A NaN ends up in the sum.
constexpr float LOW = -1.0e30f;
struct Running {
  float m = LOW, m2, s = 0.0f;
  __device__ __forceinline__ explicit Running(float l2) { m2 = __fmul_rn(LOW, l2); }
  __device__ __forceinline__ void raise(float top, float l2) {
    if (top > m) { const float t2 = __fmul_rn(top, l2); s *= gt_ex2(m2 - t2); m = top; m2 = t2; }      // no fused residue: LOW l2 - LOW l2 is 0
  }
  __device__ __forceinline__ void add(float z, float l2) {
    raise(z, l2);
    s += gt_ex2(fmaf(z, l2, -m2));
  }
  __device__ __forceinline__ void add4(const float4& z, float l2) {
    raise(fmaxf(fmaxf(z.x, z.y), fmaxf(z.z, z.w)), l2);
    s += (gt_ex2(fmaf(z.x, l2, -m2)) + gt_ex2(fmaf(z.y, l2, -m2))) + (gt_ex2(fmaf(z.z, l2, -m2)) + gt_ex2(fmaf(z.w, l2, -m2)));
  }
};

// The block's (m, s) from its threads', in every thread: each warp leaves its own, and after a barrier each joins them all.
__device__ __forceinline__ void leave_stats(const Running& r, float l2, float2* red) {
  const float m = warp_max(r.m);
  const float s = warp_sum(r.s * gt_ex2(r.m2 - __fmul_rn(m, l2)));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float2(m, s);
}
__device__ __forceinline__ float2 join_stats(const float2* red, int warps, float l2) {
  const int l = threadIdx.x & 31;
  const float2 a = l < warps ? red[l] : make_float2(LOW, 0.0f);
  const float m = warp_max(a.x);
  const float s = warp_sum(a.y * gt_ex2(__fmul_rn(a.x, l2) - __fmul_rn(m, l2)));
  return make_float2(m, s);
}

// (m, s) of a row without a logit above LOW, from global memory, by the whole block: the true maximum first, then differences.  All
// words at -inf: (-inf, 0), and NaN from there on.
__device__ __noinline__ float2 row_of_low_logits(const float* z, int C, float l2, float2* red, int warps) {
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  float m = -INFINITY, s = 0.0f;
  for (int j = threadIdx.x; j < C; j += blockDim.x) m = fmaxf(m, z[j]);
  m = warp_max(m);
  __syncthreads();
  if (l == 0) red[w].x = m;
  __syncthreads();
  m = warp_max(l < warps ? red[l].x : -INFINITY);
  if (m != -INFINITY)
    for (int j = threadIdx.x; j < C; j += blockDim.x) s += gt_ex2((z[j] - m) * l2);
  s = warp_sum(s);
  __syncthreads();
  if (l == 0) red[w].y = s;
  __syncthreads();
  s = warp_sum(l < warps ? red[l].y : 0.0f);
  return make_float2(m, s);
}

// The first of K sorted ids that is not below `id`.
__device__ __forceinline__ int lower(const int* ids, int K, int id) {
  int lo = 0, hi = K;
  while (lo < hi) { const int mid = (lo + hi) >> 1; if (ids[mid] < id) lo = mid + 1; else hi = mid; }
  return lo;
}

struct Rows {
  const float* z; long long ld;            // logits
  float* g; long long ld_g;                // their gradient (null: none wanted)
  long long B; int C, K;
  float T, l2;                             // l2 = log2(e) / T
  LmSaved s;
  float* row_loss;
  float* loss;                             // null: the rows' losses are what is asked for
  const float* upstream;                   // backward only; forward gradients are for an upstream gradient of 1
  int reduction, accumulate;
  unsigned long long* ticket;
};

__device__ __forceinline__ float row_factor(const Rows& p, long long t) {
  float c = p.T;
  if (p.upstream) c *= p.reduction == GT_REDUCE_NONE ? p.upstream[t] : p.upstream[0];
  if (p.reduction == GT_REDUCE_MEAN) c /= (float)p.s.scalars->count;
  return c;
}

// The last block to end adds the rows' losses up, in 64 bits and in a fixed order.
__device__ __forceinline__ void finish(const Rows& p, double* red) {
  __shared__ int last;
  __syncthreads();
  unsigned none;
  if (threadIdx.x == 0) last = lm_count_out(p.ticket, gridDim.x, 0, &none);
  __syncthreads();
  if (!last) return;
  double a = 0.0;
  for (long long t = threadIdx.x; t < p.B; t += blockDim.x) a += __ldcg(p.row_loss + t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < (int)blockDim.x / 32; ++w) a += red[w];
    const int n = p.s.scalars->count;
    if (p.reduction == GT_REDUCE_MEAN && n > 0) a /= (double)n;
    *p.loss = (float)a;
  }
}

// ---- rows straight from global memory ------------------------------------------------------------------
// A block per row: short rows, rows in any alignment, the forward pass alone, and the backward pass (BACKWARD: m and s are known).
// With a gradient the second reading of a row finds it in L2.  16-byte accesses between the row's first and last aligned
// address, single floats at the ends.
constexpr int STREAM_THREADS = 512;

template <bool BACKWARD>
__global__ void __launch_bounds__(STREAM_THREADS) distill_rows_kernel(const Rows p) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  __shared__ float2 red[STREAM_THREADS / 32];
  __shared__ double sums[STREAM_THREADS / 32];
  const long long t = blockIdx.x;
  const int tid = threadIdx.x;
  const float* z = p.z + t * p.ld;
  float* g = p.g ? p.g + t * p.ld_g : nullptr;
  const int* ids = p.s.ids + t * p.K;
  const float* q = p.s.q + t * p.K;
  const int head = min(p.C, (int)((16 - ((uintptr_t)z & 15)) & 15) / 4), body = (p.C - head) / 4, tail0 = head + 4 * body;
  const float4* z4 = reinterpret_cast<const float4*>(z + head);
  const bool counts = p.s.weight[t] != 0.0f;
  if (counts) {
    float2 st;
    if (BACKWARD) {
      st = p.s.stats[t];
    } else {
      Running r(p.l2);
#pragma unroll 4
      for (int j = tid; j < body; j += STREAM_THREADS) r.add4(z4[j], p.l2);
      if (tid < head) r.add(z[tid], p.l2);
      if (tail0 + tid < p.C && tid < 4) r.add(z[tail0 + tid], p.l2);
      leave_stats(r, p.l2, red);
      __syncthreads();
      st = join_stats(red, STREAM_THREADS / 32, p.l2);
      if (st.x == LOW && st.y == 0.0f) st = row_of_low_logits(z, p.C, p.l2, red, STREAM_THREADS / 32);
      if (tid < 32) {
        const float log_s = logf(st.y);
        float cross = 0.0f;
        for (int k = tid; k < p.K; k += 32) {
          const float qk = q[k];
          if (qk != 0.0f) cross += qk * ((z[ids[k]] - st.x) / p.T - log_s);
        }
        cross = warp_sum(cross);
        if (tid == 0) {
          p.s.stats[t] = st;
          p.row_loss[t] = p.T * p.T * (p.s.konst[t] - cross);
        }
      }
    }
    if (g) {
      const float c = row_factor(p, t), f = c / st.y, m = st.x;
      if ((((uintptr_t)g ^ (uintptr_t)z) & 15) == 0) {
        float4* g4 = reinterpret_cast<float4*>(g + head);
#pragma unroll 4
        for (int j = tid; j < body; j += STREAM_THREADS) {
          const float4 x = z4[j];
          float4 v = make_float4(f * gt_ex2((x.x - m) * p.l2), f * gt_ex2((x.y - m) * p.l2), f * gt_ex2((x.z - m) * p.l2), f * gt_ex2((x.w - m) * p.l2));
          if (p.accumulate) { const float4 o = g4[j]; v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w; }
          g4[j] = v;
        }
        const int j = tid < head ? tid : tid < 8 && tid >= 4 && tail0 + tid - 4 < p.C ? tail0 + tid - 4 : -1;
        if (j >= 0) g[j] = f * gt_ex2((z[j] - m) * p.l2) + (p.accumulate ? g[j] : 0.0f);
      } else {
        for (int j = tid; j < p.C; j += STREAM_THREADS) g[j] = f * gt_ex2((z[j] - m) * p.l2) + (p.accumulate ? g[j] : 0.0f);
      }
      __syncthreads();
      for (int k = tid; k < p.K; k += STREAM_THREADS) {
        const int id = ids[k];
        if (id == LM_UNUSED || (k > 0 && ids[k - 1] == id)) continue;       // the first of a run of equal ids takes them all
        float sum = 0.0f;
        for (int j = k; j < p.K && ids[j] == id; ++j) sum += q[j];
        g[id] -= c * sum;
      }
    }
  } else if (g && !p.accumulate) {
    for (int j = tid; j < p.C; j += STREAM_THREADS) g[j] = 0.0f;
  }
  if (!BACKWARD && p.loss) finish(p, sums);
}

// ---- long rows, loss and gradient in one pass over HBM ---------------------------------------------------
// A block per SM takes rows in turn and holds the row in shared memory between the two passes.  The bulk-copy engine brings it in
// as chunks, a barrier each, so that the first pass starts on chunk 0 while the last is in flight; the second pass writes the
// gradient over it and the engine takes it out, chunk by chunk; a chunk of the next row is asked for as soon as the store of the
// same chunk has been read out.  The row's up to three floats before its first 16-byte boundary and behind its last one are
// read and written singly, so that any pitch will do.
// Targets: thread k has the row's k-th, and a bit per word says that one lies there.  Between the passes the thread reads its
// word's logit and writes its gradient; the second pass leaves words with a bit alone, so neither waits for the other.  (With
// the second pass searching the sorted ids instead, 8192 x 50257 took 564 us with one target a row, 675 us with 32.)
constexpr int ROW_THREADS = 1024;
constexpr int ROW_MAX_CHUNKS = 14;
constexpr int ROW_MAX_TOP = 256;
constexpr int ROW_MIN_C = 4096, ROW_MAX_C = 53248;
constexpr int ROW_MAP_WORDS = ROW_MAX_C / 32 + 1;

__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded: after about a second the block gives up, raises the status word and every thread leaves its loops.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status) {
  if (bar_test(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (bar_test(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > 2000000000LL) { *abort_flag = 1; atomicExch(status, GT_ERR_TIMEOUT); return false; }
  }
}

__global__ void __launch_bounds__(ROW_THREADS, 1) distill_row_in_smem_kernel(const Rows p, int nchunks, int q4, int* status) {
  gt_let_next_kernel_start();
  gt_wait_for_previous_kernel();
  extern __shared__ __align__(128) uint8_t row_smem[];
  __shared__ float2 red[32];
  __shared__ double sums[32];
  __shared__ unsigned map[2][ROW_MAP_WORDS];
  __shared__ int top_id[2][ROW_MAX_TOP];
  __shared__ float top_q[2][ROW_MAX_TOP], cross_part[ROW_MAX_TOP / 32];
  __shared__ __align__(8) unsigned long long bars[ROW_MAX_CHUNKS];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  float4* const row4 = reinterpret_cast<float4*>(row_smem);
  const uint32_t row_addr = (uint32_t)__cvta_generic_to_shared(row_smem);
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
  const int tid = threadIdx.x, K = p.K;
  for (int i = tid; i < 2 * ROW_MAP_WORDS; i += ROW_THREADS) (&map[0][0])[i] = 0;
  if (tid < 2 * ROW_MAX_TOP) (&top_id[0][0])[tid] = LM_UNUSED;
  if (tid == 0) {
    for (int c = 0; c < ROW_MAX_CHUNKS; ++c) asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar0 + 8 * c), "r"(1) : "memory");
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  // floats before the first 16-byte boundary, and whole 16-byte units from there
  auto head_of = [&](long long row) { return (int)((16 - ((uintptr_t)(p.z + row * p.ld) & 15)) & 15) / 4; };
  auto request = [&](long long row, int c) {
    const int head = head_of(row), n4 = (p.C - head) >> 2;
    const int u0 = c * q4, u1 = min(u0 + q4, n4);
    const uint32_t bytes = (uint32_t)(u1 - u0) * 16u;
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar0 + 8 * c), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(row_addr + (uint32_t)u0 * 16u), "l"(p.z + row * p.ld + head + (long long)u0 * 4), "r"(bytes), "r"(bar0 + 8 * c) : "memory");
  };
  long long row = blockIdx.x;
  if (tid == 0 && row < p.B)
    for (int c = 0; c < nchunks; ++c) request(row, c);
  bool ok = true;
  uint32_t failed_parity = 0;
  for (int it = 0; ok && row < p.B; row += gridDim.x, ++it) {
    const uint32_t parity = (uint32_t)(it & 1);
    const int head = head_of(row), n4 = (p.C - head) >> 2, tail0 = head + 4 * n4;
    const float* z = p.z + row * p.ld;
    float* g = p.g + row * p.ld_g;
    // asked for now, needed after the first pass: this row's targets, and the single floats at its ends
    const int my_id = tid < K ? p.s.ids[row * K + tid] : LM_UNUSED;
    const float my_q = tid < K ? p.s.q[row * K + tid] : 0.0f;
    const float weight = p.s.weight[row], konst = p.s.konst[row], c_row = row_factor(p, row);
    const int edge = tid < head ? tid : tid >= 4 && tid < 8 && tail0 + tid - 4 < p.C ? tail0 + tid - 4 : -1;
    const float edge_z = edge >= 0 ? z[edge] : 0.0f;
    // ---- pass 1: running maximum and sum, chunk by chunk as they arrive
    Running r(p.l2);
    for (int c = 0; c < nchunks; ++c) {
      if (!bar_wait(bar0 + 8 * c, parity, abort_flag, status)) { ok = false; break; }       // leaves the chunk loop only
      const int u1 = min((c + 1) * q4, n4);
      for (int u = c * q4 + tid; u < u1; u += ROW_THREADS) r.add4(row4[u], p.l2);
    }
    if (edge >= 0) r.add(edge_z, p.l2);
    // the targets' bits (counted from `head`), and those of the row before, which everybody is done with, off the other map
    unsigned* const bits = map[it & 1];
    const bool inside = my_id != LM_UNUSED && my_id >= head && my_id < tail0;
    if (tid < K) {
      const int old = top_id[(it & 1) ^ 1][tid], old_head = it > 0 ? head_of(row - gridDim.x) : 0;
      if (old != LM_UNUSED && old >= old_head) map[(it & 1) ^ 1][(old - old_head) >> 5] = 0;
      top_id[it & 1][tid] = my_id;
      top_q[it & 1][tid] = my_q;
      if (inside) atomicOr(&bits[(my_id - head) >> 5], 1u << ((my_id - head) & 31));
    }
    leave_stats(r, p.l2, red);
    if (!__syncthreads_and(ok)) { ok = false; failed_parity = parity; break; }
    float2 st = join_stats(red, 32, p.l2);
    if (st.x == LOW && st.y == 0.0f) st = row_of_low_logits(z, p.C, p.l2, red, 32);
    const float c = c_row, m = st.x;
    const bool live = weight != 0.0f;
    // 2^(z l2 - m2) f in the second pass with the m2 of the first, whose rounding cancels in f = c / s; differences for logits
    // whose product with l2 might overflow
    const float m2 = __fmul_rn(m, p.l2), f = c / st.y;
    const bool far = !(fabsf(m) < -LOW);
    auto grad_of = [&](float x) { return f * gt_ex2(far ? (x - m) * p.l2 : fmaf(x, p.l2, -m2)); };
    const int* ids = top_id[it & 1];
    const float* qs = top_q[it & 1];
    float* const row_f = reinterpret_cast<float*>(row_smem);
    if (tid < ROW_MAX_TOP) {                                    // whole warps
      float cross = 0.0f;
      if (my_id != LM_UNUSED && (tid == 0 || ids[tid - 1] != my_id)) {       // the first of a run of equal ids takes them all
        float sum = my_q;
        for (int k = tid + 1; k < K && ids[k] == my_id; ++k) sum += qs[k];
        const float x = inside ? row_f[my_id - head] : z[my_id];
        if (sum != 0.0f) cross = sum * ((x - m) / p.T - logf(st.y));
        const float e = live ? grad_of(x) - c * sum : 0.0f;
        if (inside) row_f[my_id - head] = e; else g[my_id] = e;
      }
      cross = warp_sum(cross);
      if ((tid & 31) == 0) cross_part[tid >> 5] = cross;
    }
    // ---- pass 2: the gradient over the row, in place; each chunk leaves as soon as the whole block has written it
    if (edge >= 0) {
      const int k = lower(ids, K, edge);
      if (k == K || ids[k] != edge) g[edge] = live ? grad_of(edge_z) : 0.0f;
    }
    const long long next = row + gridDim.x;
    for (int c2 = 0; c2 < nchunks; ++c2) {
      const int u0 = c2 * q4, u1 = min(u0 + q4, n4);
      for (int u = u0 + tid; u < u1; u += ROW_THREADS) {
        const float4 x = row4[u];
        const unsigned taken = bits[u >> 3] >> (4 * (u & 7)) & 15u;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (live && !far) v = make_float4(f * gt_ex2(fmaf(x.x, p.l2, -m2)), f * gt_ex2(fmaf(x.y, p.l2, -m2)), f * gt_ex2(fmaf(x.z, p.l2, -m2)),
                                          f * gt_ex2(fmaf(x.w, p.l2, -m2)));
        else if (live) v = make_float4(grad_of(x.x), grad_of(x.y), grad_of(x.z), grad_of(x.w));
        if (taken == 0) { row4[u] = v; continue; }
        if (!(taken & 1u)) row_f[4 * u] = v.x;
        if (!(taken & 2u)) row_f[4 * u + 1] = v.y;
        if (!(taken & 4u)) row_f[4 * u + 2] = v.z;
        if (!(taken & 8u)) row_f[4 * u + 3] = v.w;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncthreads();
      if (tid == 0) {
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                     ::"l"(g + head + (long long)u0 * 4), "r"(row_addr + (uint32_t)u0 * 16u), "r"((uint32_t)(u1 - u0) * 16u) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        // chunk c2 - 1 of the next row may come in once its store has been read out of shared memory: it was issued a chunk ago
        if (c2 >= 1 && next < p.B) {
          asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          request(next, c2 - 1);
        }
      }
    }
    if (tid == 0 && next < p.B) {
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
      request(next, nchunks - 1);
    }
    // the loss; a barrier of the second pass lies behind cross_part, another before it is written again
    if (tid == 0 && live) {
      float cross = 0.0f;
      for (int w = 0; w < ROW_MAX_TOP / 32; ++w) cross += cross_part[w];
      p.s.stats[row] = st;
      p.row_loss[row] = p.T * p.T * (konst - cross);
    }
  }
  if (tid == 0) {
    if (!ok) {     // giving up: let the copies of the row that was being waited for land (bounded) before shared memory is released
      const long long t0 = clock64();
      for (int c = 0; c < nchunks; ++c)
        while (!bar_test(bar0 + 8 * c, failed_parity) && clock64() - t0 < 2000000000LL) {}
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  finish(p, sums);
}

}  // namespace

extern "C" int gt_topk_distillation_sizes(gt_ctx* ctx, int64_t B, int64_t C, int64_t K, size_t* saved) {
  if (!ctx || !saved || lm_bad_sizes(B, C, K)) return GT_ERR_INVALID_ARG;
  *saved = lm_saved(nullptr, B, K).bytes + lm_up256(sizeof(float) * B);
  return GT_OK;
}

extern "C" int gt_topk_distillation(gt_ctx* ctx, float* loss, void* saved, float* dlogits, int64_t ld_dlogits, const float* logits,
                                    int64_t ld_logits, const float* ids, const float* teacher, int64_t B, int64_t C, int64_t K, float temperature,
                                    int reduction) {
  if (!ctx || !loss || !saved || !logits || !ids || !teacher || lm_bad_sizes(B, C, K) || ld_logits < C || lm_bad_reduction(reduction) ||
      lm_bad_temperature(temperature) || (dlogits && (ld_dlogits < C || reduction == GT_REDUCE_NONE))) return GT_ERR_INVALID_ARG;
  Rows p;
  memset(&p, 0, sizeof(p));
  p.z = logits; p.ld = ld_logits; p.g = dlogits; p.ld_g = ld_dlogits;
  p.B = B; p.C = (int)C; p.K = (int)K; p.T = temperature; p.l2 = 1.4426950408889634f / temperature;
  p.s = lm_saved(saved, B, K);
  p.row_loss = reduction == GT_REDUCE_NONE ? loss : (float*)((char*)saved + p.s.bytes);
  p.loss = reduction == GT_REDUCE_NONE ? nullptr : loss;
  p.reduction = reduction;
  p.ticket = lm_ticket(ctx);
  int rc = gt_lm_top_targets(ctx, p.s, p.row_loss, ids, teacher, B, C, K, temperature);
  if (rc != GT_OK) return rc;
  // The row in shared memory: with a gradient, for rows long enough to be worth a block of 1024 threads and short enough to fit
  // (53248 words beside the targets), where logits and gradient lie alike with respect to 16 bytes.
  if (dlogits && C >= ROW_MIN_C && C <= ROW_MAX_C && K <= ROW_MAX_TOP && (((uintptr_t)logits ^ (uintptr_t)dlogits) & 15) == 0 &&
      (ld_logits - ld_dlogits) % 4 == 0 && ((uintptr_t)logits & 3) == 0) {
    GT_SMEM_OPT_IN(ctx, distill_row_in_smem_kernel, (ROW_MAX_C + 3) / 4 * 16);
    const int units = (int)((C + 3) / 4);
    // chunks of about 40 KB, eight of a shorter row: see gt_cross_entropy_fused
    int chunks = units >= 5120 ? (units + 1280) / 2560 : 8;
    if (chunks < 2) chunks = 2;
    if (chunks > ROW_MAX_CHUNKS) chunks = ROW_MAX_CHUNKS;
    const int grid = (int)(B < ctx->sm_count ? B : ctx->sm_count);
    GT_CUDA_OK(ctx, gt_launch_overlapped(distill_row_in_smem_kernel, dim3(grid), dim3(ROW_THREADS), (size_t)units * 16, ctx->stream, p, chunks, (units + chunks - 1) / chunks, ctx->d_status));
  } else {
    GT_CUDA_OK(ctx, gt_launch_overlapped(distill_rows_kernel<false>, dim3((unsigned)B), dim3(STREAM_THREADS), 0, ctx->stream, p));
  }
  ctx->launches += 1;
  return GT_OK;
}

extern "C" int gt_topk_distillation_backward(gt_ctx* ctx, float* dlogits, int64_t ld_dlogits, void* saved, const float* logits, int64_t ld_logits,
                                             const float* upstream, int64_t B, int64_t C, int64_t K, float temperature, int reduction,
                                             int accumulate) {
  if (!ctx || !dlogits || !saved || !logits || !upstream || lm_bad_sizes(B, C, K) || ld_logits < C || ld_dlogits < C || lm_bad_reduction(reduction) ||
      lm_bad_temperature(temperature)) return GT_ERR_INVALID_ARG;
  Rows p;
  memset(&p, 0, sizeof(p));
  p.z = logits; p.ld = ld_logits; p.g = dlogits; p.ld_g = ld_dlogits;
  p.B = B; p.C = (int)C; p.K = (int)K; p.T = temperature; p.l2 = 1.4426950408889634f / temperature;
  p.s = lm_saved(saved, B, K);
  p.upstream = upstream; p.reduction = reduction; p.accumulate = accumulate;
  GT_CUDA_OK(ctx, gt_launch_overlapped(distill_rows_kernel<true>, dim3((unsigned)B), dim3(STREAM_THREADS), 0, ctx->stream, p));
  ctx->launches += 1;
  return GT_OK;
}
