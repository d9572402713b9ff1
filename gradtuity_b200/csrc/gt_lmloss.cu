// Losses of the language-model head with sparse targets, and their gradients.
//
// For token t and word v, z_tv = logit_tv / T (T = 1 for cross entropy; the linear forms compute logit = x W^T themselves):
//     p_tv = exp(z_tv - m_t) / s_t,  m_t = max_v z_tv,  s_t = sum_v exp(z_tv - m_t)
//     loss_t = T^2 sum_k q_tk (log q_tk - (z_t,id_tk - m_t - log s_t))
//     d loss_t / d logit_tv = T (p_tv - sum of the q_tk with id_tk = v)
// The targets of a row are (id, q) pairs sorted by id: one pair with q = 1 for cross entropy; for distillation the softmax of
// the teacher's top logits / T over the entries in use.  A row without any target in use has weight 0: no loss, no gradient.
// m and s are kept apart instead of as m + log s: p then carries no rounding of a sum of that size.
//
// Linear forms: the (tokens x words) logits are never kept.  Both directions walk over pieces of the vocabulary; the backward
// computes a piece's logits again, turns them into the logits' gradient G in place, and multiplies:
//     dx += G W_piece,   dW_piece = G^T x.

#include <math.h>

#include "gt_internal.h"

namespace {

constexpr int TOP_MAX = 1024;                       // targets of a row: they are sorted in shared memory
constexpr int UNUSED = 0x7fffffff;                  // id of a place that is not in use; sorts behind every word
constexpr long long PIECE_BYTES = 64ll << 20;       // what one piece of logits may occupy

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

// (maximum, sum of exponentials relative to it); an empty part is (-inf, 0).  A maximum of -inf on both sides stays (-inf, 0):
// every exponential is then 0, which the caller sees as a sum of 0.
struct MaxSum { float m, s; };
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s};
  return {m, a.s * expf(a.m - m) + b.s * expf(b.m - m)};
}
__device__ __forceinline__ MaxSum warp_join(MaxSum a) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    MaxSum b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, a.s, o);
    // the same order of the two operands on both lanes, so that all lanes hold the same bits
    a = (threadIdx.x & o) ? join(b, a) : join(a, b);
  }
  return a;
}

// What the forward pass leaves for the backward pass, in one block of memory.
struct Saved {
  int* count;       // rows that count
  float2* stats;    // (m, s) per row
  float* weight;    // 1, or 0 for a row that does not count
  float* konst;     // sum of q log q per row
  int* ids;         // (M, K), ascending, UNUSED at the end
  float* q;         // (M, K), 0 where unused
  size_t bytes;
};
size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
Saved saved_layout(void* base, long long M, long long K) {
  Saved s;
  char* p = (char*)base;
  size_t at = 0;
  auto take = [&](size_t n) { char* r = p + at; at += up256(n); return r; };
  s.count = (int*)take(sizeof(int));
  s.stats = (float2*)take(sizeof(float2) * M);
  s.weight = (float*)take(sizeof(float) * M);
  s.konst = (float*)take(sizeof(float) * M);
  s.ids = (int*)take(sizeof(int) * M * K);
  s.q = (float*)take(sizeof(float) * M * K);
  s.bytes = at;
  return s;
}

// ---- targets -------------------------------------------------------------------------------------

// Cross entropy: one target of q = 1 per row.  An id outside the vocabulary sets the status word.
__global__ void __launch_bounds__(256) hard_targets_kernel(const float* __restrict__ targets, long long M, long long V, float ignore,
                                                           Saved s, int* status) {
  const long long t = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  bool used = false;
  if (t < M) {
    const float f = targets[t];
    const bool in_range = f >= 0.0f && f < (float)V;
    used = f != ignore && in_range;
    if (f != ignore && !in_range) atomicExch(status, GT_ERR_INVALID_ARG);
    s.ids[t] = used ? (int)f : UNUSED;
    s.q[t] = used ? 1.0f : 0.0f;
    s.weight[t] = used ? 1.0f : 0.0f;
    s.konst[t] = 0.0f;
  }
  const int n = __syncthreads_count(used);
  if (threadIdx.x == 0 && n) atomicAdd(s.count, n);        // whole numbers: the order does not matter
}

// Distillation: a warp per row.  q = softmax(teacher / T) over the places in use (id >= 0, logit above -inf), sorted by id by
// counting, for each place, the places that go before it (K^2 comparisons, K is tens to a few hundred).
__global__ void __launch_bounds__(128) top_targets_kernel(const float* __restrict__ ids, const float* __restrict__ teacher, long long M,
                                                          long long V, int K, float inv_T, Saved s, int* status) {
  extern __shared__ float smem[];
  const int w = threadIdx.x >> 5, l = threadIdx.x & 31;
  int* key = reinterpret_cast<int*>(smem) + (size_t)w * 2 * K;
  float* val = reinterpret_cast<float*>(key + K);
  __shared__ int counted[4];
  const long long t = (long long)blockIdx.x * 4 + w;
  float mx = -INFINITY;
  bool any = false;
  if (t < M) {
    for (int k = l; k < K; k += 32) {
      const float f = ids[t * K + k], v = teacher[t * K + k];
      bool used = !(f < 0.0f) && v > -INFINITY;
      if (used && !(f < (float)V)) { atomicExch(status, GT_ERR_INVALID_ARG); used = false; }
      key[k] = used ? (int)f : UNUSED;
      val[k] = used ? v : -INFINITY;
      if (used) { any = true; mx = fmaxf(mx, v); }
    }
    any = __any_sync(0xffffffffu, any);
    mx = warp_max(mx);
    __syncwarp();
    float sum = 0.0f;
    for (int k = l; k < K; k += 32)
      if (key[k] != UNUSED) sum += expf((val[k] - mx) * inv_T);
    sum = warp_sum(sum);
    const float log_sum = logf(sum), inv = 1.0f / sum;
    float konst = 0.0f;
    for (int k = l; k < K; k += 32) {
      const int id = key[k];
      int before = 0;
      for (int j = 0; j < K; ++j) {
        const int o = key[j];
        before += (o < id) || (o == id && j < k);
      }
      float q = 0.0f;
      if (id != UNUSED) {
        const float u = (val[k] - mx) * inv_T;
        q = expf(u) * inv;
        if (q != 0.0f) konst += q * (u - log_sum);          // 0 log 0 = 0
      }
      s.ids[t * K + before] = id;
      s.q[t * K + before] = q;
    }
    konst = warp_sum(konst);
    if (l == 0) { s.weight[t] = any ? 1.0f : 0.0f; s.konst[t] = konst; }
  }
  if (l == 0) counted[w] = any;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int n = counted[0] + counted[1] + counted[2] + counted[3];
    if (n) atomicAdd(s.count, n);
  }
}

// ---- rows ------------------------------------------------------------------------------------------

// (m, s) of a row of `n` values scaled by `scale`, joined with what `stats` holds when `carry`.  A block per row.
__global__ void __launch_bounds__(256) row_stats_kernel(const float* __restrict__ z, long long ld, long long n, float scale, float2* __restrict__ stats,
                                                        int carry) {
  __shared__ MaxSum part[8];
  const long long t = blockIdx.x;
  const float* zr = z + t * ld;
  MaxSum a = {-INFINITY, 0.0f};
  for (long long j = threadIdx.x; j < n; j += blockDim.x) {
    const float v = zr[j] * scale;
    if (v > a.m) { a.s = a.s * expf(a.m - v) + 1.0f; a.m = v; }
    else if (v != -INFINITY) { a.s += expf(v - a.m); }
  }
  a = warp_join(a);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    MaxSum r = carry ? MaxSum{stats[t].x, stats[t].y} : MaxSum{-INFINITY, 0.0f};
    for (int w = 0; w < 8; ++w) r = join(r, part[w]);
    stats[t] = make_float2(r.m, r.s);
  }
}

// z -> the gradient of the loss with respect to the logits, in place or to another place: g = c (p - q), where c holds the row's
// weight, T, the upstream gradient and 1 / n.  The columns are words [v0, v0 + n).  A block per row.
__global__ void __launch_bounds__(256) row_grad_kernel(float* __restrict__ g, long long ld_g, const float* z, long long ld, long long v0, long long n,
                                                       float scale, float T, Saved s, int K, const float* __restrict__ upstream, int reduction,
                                                       int accumulate) {
  const long long t = blockIdx.x;
  const float* zr = z + t * ld;
  float* gr = g + t * ld_g;
  float c = s.weight[t] * T;
  if (c != 0.0f) {
    c *= reduction == GT_REDUCE_NONE ? upstream[t] : upstream[0];
    if (reduction == GT_REDUCE_MEAN) c /= (float)*s.count;
  }
  if (s.weight[t] == 0.0f) {
    if (!accumulate) for (long long j = threadIdx.x; j < n; j += blockDim.x) gr[j] = 0.0f;
    return;
  }
  const float2 st = s.stats[t];
  const float m = st.x, cs = c / st.y;
  for (long long j = threadIdx.x; j < n; j += blockDim.x) {
    const float v = cs * expf(zr[j] * scale - m);
    gr[j] = accumulate ? gr[j] + v : v;
  }
  __syncthreads();
  const int* ids = s.ids + t * K;
  const float* q = s.q + t * K;
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const long long id = ids[k];
    if (id < v0 || id >= v0 + n || (k > 0 && ids[k - 1] == id)) continue;     // the first of a run of equal ids takes them all
    float sum = 0.0f;
    for (int j = k; j < K && ids[j] == id; ++j) sum += q[j];
    gr[id - v0] -= c * sum;
  }
}

// loss_t from the row's statistics and the logits of its targets: a warp per row.  x given: logits are x_t . w_id, in fp32.
__global__ void __launch_bounds__(256) row_loss_kernel(float* __restrict__ row_loss, const float* __restrict__ logits, long long ld,
                                                       const float* __restrict__ x, const float* __restrict__ w, long long M, long long E, int K,
                                                       float scale, float T, Saved s) {
  const long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int l = threadIdx.x & 31;
  if (t >= M) return;
  if (s.weight[t] == 0.0f) {
    if (l == 0) row_loss[t] = 0.0f;
    return;
  }
  const float2 st = s.stats[t];
  const float log_s = logf(st.y);
  float cross = 0.0f;
  for (int k = 0; k < K; ++k) {
    const int id = s.ids[t * K + k];
    if (id == UNUSED) break;
    const float q = s.q[t * K + k];
    if (q == 0.0f) continue;
    float z = 0.0f;
    if (x) {
      for (long long e = l; e < E; e += 32) z = fmaf(x[t * E + e], w[(long long)id * E + e], z);
      z = warp_sum(z);
    } else {
      z = logits[t * ld + id];
    }
    cross += q * ((z * scale - st.x) - log_s);
  }
  if (l == 0) row_loss[t] = T * T * (s.konst[t] - cross);
}

// Sum or mean of the rows' losses in 64 bits, in a fixed order: one block.
__global__ void __launch_bounds__(1024) reduce_loss_kernel(float* __restrict__ loss, const float* __restrict__ row_loss, long long M, const int* count,
                                                           int mean) {
  __shared__ double part[32];
  double a = 0.0;
  for (long long t = threadIdx.x; t < M; t += 1024) a += row_loss[t];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 32; ++w) a += part[w];
    if (mean && *count > 0) a /= (double)*count;
    *loss = (float)a;
  }
}

bool bad_sizes(long long M, long long V, long long K) {
  return M <= 0 || V <= 0 || K <= 0 || M > 0x7fffffff || V >= (1ll << 24) || K > TOP_MAX;    // ids are float-encoded: exact below 2^24
}
bool bad_temperature(float T) { return !(T > 0.0f) || isinf(T); }
bool bad_reduction(int r) { return r != GT_REDUCE_NONE && r != GT_REDUCE_MEAN && r != GT_REDUCE_SUM; }

bool bad_precision(int p) { return p != GT_PREC_TF32 && p != GT_PREC_TF32X3 && p != GT_PREC_FP32; }

// words of a piece: what the byte limit allows for M rows, in whole multiples of 256
long long piece_words(long long M, long long V) {
  long long n = PIECE_BYTES / 4 / M / 256 * 256;
  if (n < 256) n = 256;
  return n < V ? n : V;
}
long long piece_pitch(long long words) { return (words + 3) / 4 * 4; }

int prepare_targets(gt_ctx* ctx, const Saved& s, const float* targets, float ignore, const float* ids, const float* teacher, long long M, long long V,
                    long long K, float T) {
  GT_CUDA_OK(ctx, cudaMemsetAsync(s.count, 0, sizeof(int), ctx->stream));
  if (targets) {
    hard_targets_kernel<<<(unsigned)((M + 255) / 256), 256, 0, ctx->stream>>>(targets, M, V, ignore, s, ctx->d_status);
  } else {
    top_targets_kernel<<<(unsigned)((M + 3) / 4), 128, (size_t)4 * 2 * K * 4, ctx->stream>>>(ids, teacher, M, V, (int)K, 1.0f / T, s, ctx->d_status);
  }
  GT_CUDA_OK(ctx, cudaGetLastError());
  ctx->launches += 1;
  return GT_OK;
}

int finish_loss(gt_ctx* ctx, float* loss, float* row_loss, const float* logits, long long ld, const float* x, const float* w, long long M, long long E,
                long long K, float T, int reduction, const Saved& s) {
  float* rows = reduction == GT_REDUCE_NONE ? loss : row_loss;
  row_loss_kernel<<<(unsigned)((M + 7) / 8), 256, 0, ctx->stream>>>(rows, logits, ld, x, w, M, E, (int)K, 1.0f / T, T, s);
  if (reduction != GT_REDUCE_NONE)
    reduce_loss_kernel<<<1, 1024, 0, ctx->stream>>>(loss, rows, M, s.count, reduction == GT_REDUCE_MEAN);
  GT_CUDA_OK(ctx, cudaGetLastError());
  ctx->launches += reduction == GT_REDUCE_NONE ? 1 : 2;
  return GT_OK;
}

int linear_forward(gt_ctx* ctx, float* loss, void* saved, void* scratch, const float* x, const float* w, const float* targets, float ignore,
                   const float* ids, const float* teacher, int64_t M, int64_t V, int64_t E, int64_t K, float T, int reduction, int precision) {
  const Saved s = saved_layout(saved, M, K);
  int rc = prepare_targets(ctx, s, targets, ignore, ids, teacher, M, V, K, T);
  if (rc != GT_OK) return rc;
  float* row_loss = (float*)scratch;
  float* z = (float*)((char*)scratch + up256(sizeof(float) * M));
  const long long step = piece_words(M, V), pitch = piece_pitch(step);
  for (long long v0 = 0; v0 < V; v0 += step) {
    const long long n = V - v0 < step ? V - v0 : step;
    rc = gt_gemm(ctx, GT_LAYOUT_NT, M, n, E, x, E, w + v0 * E, E, z, pitch, nullptr, nullptr, 1.0f, 0, GT_EPI_NONE, precision, nullptr);
    if (rc != GT_OK) return rc;
    row_stats_kernel<<<(unsigned)M, 256, 0, ctx->stream>>>(z, pitch, n, 1.0f / T, s.stats, v0 > 0);
    GT_CUDA_OK(ctx, cudaGetLastError());
    ctx->launches += 1;
  }
  return finish_loss(ctx, loss, row_loss, nullptr, 0, x, w, M, E, K, T, reduction, s);
}

}  // namespace

extern "C" int gt_linear_loss_sizes(gt_ctx* ctx, int64_t M, int64_t V, int64_t E, int64_t K, int precision, size_t* saved, size_t* scratch) {
  if (!ctx || !saved || !scratch || E <= 0 || bad_sizes(M, V, K) || bad_precision(precision)) return GT_ERR_INVALID_ARG;
  *saved = saved_layout(nullptr, M, K).bytes;
  *scratch = up256(sizeof(float) * M) + sizeof(float) * M * piece_pitch(piece_words(M, V));
  return GT_OK;
}

extern "C" int gt_linear_cross_entropy(gt_ctx* ctx, float* loss, void* saved, void* scratch, const float* x, const float* w, const float* targets,
                                       int64_t M, int64_t V, int64_t E, float ignore_index, int reduction, int precision) {
  if (!ctx || !loss || !saved || !scratch || !x || !w || !targets || E <= 0 || bad_sizes(M, V, 1) || bad_reduction(reduction) || bad_precision(precision)) return GT_ERR_INVALID_ARG;
  return linear_forward(ctx, loss, saved, scratch, x, w, targets, ignore_index, nullptr, nullptr, M, V, E, 1, 1.0f, reduction, precision);
}

extern "C" int gt_linear_topk_distillation(gt_ctx* ctx, float* loss, void* saved, void* scratch, const float* x, const float* w, const float* ids,
                                           const float* teacher, int64_t M, int64_t V, int64_t E, int64_t K, float temperature, int reduction,
                                           int precision) {
  if (!ctx || !loss || !saved || !scratch || !x || !w || !ids || !teacher || E <= 0 || bad_sizes(M, V, K) || bad_reduction(reduction) ||
      bad_temperature(temperature) || bad_precision(precision)) return GT_ERR_INVALID_ARG;
  return linear_forward(ctx, loss, saved, scratch, x, w, nullptr, 0.0f, ids, teacher, M, V, E, K, temperature, reduction, precision);
}

extern "C" int gt_linear_loss_backward(gt_ctx* ctx, float* dx, float* dw, void* saved, void* scratch, const float* x, const float* w,
                                       const float* upstream, int64_t M, int64_t V, int64_t E, int64_t K, float temperature, int reduction,
                                       int precision, int acc_dx, int acc_dw) {
  if (!ctx || !saved || !scratch || !x || !w || !upstream || E <= 0 || bad_sizes(M, V, K) || bad_reduction(reduction) || bad_temperature(temperature) ||
      bad_precision(precision)) return GT_ERR_INVALID_ARG;
  const Saved s = saved_layout(saved, M, K);
  float* z = (float*)((char*)scratch + up256(sizeof(float) * M));
  const long long step = piece_words(M, V), pitch = piece_pitch(step);
  for (long long v0 = 0; v0 < V; v0 += step) {
    const long long n = V - v0 < step ? V - v0 : step;
    int rc = gt_gemm(ctx, GT_LAYOUT_NT, M, n, E, x, E, w + v0 * E, E, z, pitch, nullptr, nullptr, 1.0f, 0, GT_EPI_NONE, precision, nullptr);
    if (rc != GT_OK) return rc;
    row_grad_kernel<<<(unsigned)M, 256, 0, ctx->stream>>>(z, pitch, z, pitch, v0, n, 1.0f / temperature, temperature, s, (int)K, upstream, reduction, 0);
    GT_CUDA_OK(ctx, cudaGetLastError());
    ctx->launches += 1;
    if (dx) {
      rc = gt_gemm(ctx, GT_LAYOUT_NN, M, E, n, z, pitch, w + v0 * E, E, dx, E, nullptr, nullptr, 1.0f, acc_dx || v0 > 0, GT_EPI_NONE, precision, nullptr);
      if (rc != GT_OK) return rc;
    }
    if (dw) {
      rc = gt_gemm(ctx, GT_LAYOUT_TN, n, E, M, z, pitch, x, E, dw + v0 * E, E, nullptr, nullptr, 1.0f, acc_dw, GT_EPI_NONE, precision, nullptr);
      if (rc != GT_OK) return rc;
    }
  }
  return GT_OK;
}

extern "C" int gt_topk_distillation_sizes(gt_ctx* ctx, int64_t B, int64_t C, int64_t K, size_t* saved) {
  if (!ctx || !saved || bad_sizes(B, C, K)) return GT_ERR_INVALID_ARG;
  *saved = saved_layout(nullptr, B, K).bytes + up256(sizeof(float) * B);
  return GT_OK;
}

extern "C" int gt_topk_distillation(gt_ctx* ctx, float* loss, void* saved, const float* logits, int64_t ld_logits, const float* ids,
                                    const float* teacher, int64_t B, int64_t C, int64_t K, float temperature, int reduction) {
  if (!ctx || !loss || !saved || !logits || !ids || !teacher || bad_sizes(B, C, K) || ld_logits < C || bad_reduction(reduction) ||
      bad_temperature(temperature)) return GT_ERR_INVALID_ARG;
  const Saved s = saved_layout(saved, B, K);
  int rc = prepare_targets(ctx, s, nullptr, 0.0f, ids, teacher, B, C, K, temperature);
  if (rc != GT_OK) return rc;
  row_stats_kernel<<<(unsigned)B, 256, 0, ctx->stream>>>(logits, ld_logits, C, 1.0f / temperature, s.stats, 0);
  GT_CUDA_OK(ctx, cudaGetLastError());
  ctx->launches += 1;
  return finish_loss(ctx, loss, (float*)((char*)saved + s.bytes), logits, ld_logits, nullptr, nullptr, B, 0, K, temperature, reduction, s);
}

extern "C" int gt_topk_distillation_backward(gt_ctx* ctx, float* dlogits, int64_t ld_dlogits, void* saved, const float* logits, int64_t ld_logits,
                                             const float* upstream, int64_t B, int64_t C, int64_t K, float temperature, int reduction,
                                             int accumulate) {
  if (!ctx || !dlogits || !saved || !logits || !upstream || bad_sizes(B, C, K) || ld_logits < C || ld_dlogits < C || bad_reduction(reduction) ||
      bad_temperature(temperature)) return GT_ERR_INVALID_ARG;
  const Saved s = saved_layout(saved, B, K);
  row_grad_kernel<<<(unsigned)B, 256, 0, ctx->stream>>>(dlogits, ld_dlogits, logits, ld_logits, 0, C, 1.0f / temperature, temperature, s, (int)K,
                                                        upstream, reduction, accumulate);
  GT_CUDA_OK(ctx, cudaGetLastError());
  ctx->launches += 1;
  return GT_OK;
}
