// The products of the linear losses (gt_lmloss.cu) on the tensor cores: logits with their running maximum and sum, the
// logits' gradient G, dx = G W and dW = G^T x.
//
// Mathematics.  A 32-bit operand is split into two halves of 11 bits each, v = 2^e (hi + lo), with one power of two for the whole
// matrix (its largest value lands in [2^14, 2^15), so lo keeps its bits down to 2^-38 of that), and a product is
//     hi hi' + hi lo' + lo hi'      (what is dropped, lo lo', is 2^-22 of the operands)
// by fp16 tensor-core instructions, which run at twice the rate of tf32 and read half the bytes.  With products == 1 only hi hi'
// is taken: the operand rounding of tf32.
// The tensor cores add into their 32-bit accumulators by cutting off, not rounding (measured: a sum of K = 512 terms of one
// sign comes out 1.5e-6 too small).  So no accumulator stays there for long: after two or three stages (128 or 192 of K) the
// epilogue warps add it to their registers, rounding to nearest, while the next one fills the other half of tensor memory.
//
// Work.  One kernel, persistent, a pair of CTAs (cta_group::2) per 256 x 256 tile, handed out by a counter: the units of a launch
// differ in length by a factor of ten, and the long ones come first, so that the short ones fill the end:
//     dW tile     256 words x 256 of E, over all rows            A = G^T (MN-major), B = x  (MN-major)
//     dx tile     256 rows x 256 of E, over a piece of the words  A = G   (K-major),  B = W  (MN-major)
//     G tile      256 rows x 256 words, over E                    A = x   (K-major),  B = W  (K-major)
// A launch computes dW and dx of one piece and, beside them, G of the next one.
// Warps per CTA: a producer (TMA), the issuer of the MMAs (leader CTA), eight epilogue warps, of which each holds 32 rows x 128
// columns, 128 registers a thread.

#include "gt_lmloss.h"
#include "gt_umma_common.cuh"

namespace {

constexpr int THREADS = 320;
constexpr int TILE = LM_TILE, HALF = 128, BK = LM_KBLOCK;
constexpr int OPERAND_BYTES = HALF * BK * 2;                    // one half-precision operand of one CTA and stage: 16 KB
constexpr int RING_BYTES = 3 * 4 * OPERAND_BYTES;               // three stages of hi and lo, or six of hi
constexpr int MAX_STAGES = 6;
constexpr int STAGE_TILE = 4096;                                // per epilogue warp
constexpr int SLOTS = 4;                                        // units handed out ahead
constexpr int SMEM_BYTES = RING_BYTES + 8 * STAGE_TILE + 1024 + 1024;
static_assert(SMEM_BYTES <= 232448, "exceeds the 227 KB of shared memory a CTA may use");

enum Kind { STATS, GRAD, DX, DW };

struct Params {
  LmScalars* scalars;
  int* counter;
  int* status;
  const int* row_of;
  const float2* stats;
  const float2* factor;
  const int* ids;
  const float* q;
  float2* partial;
  float* target_z;
  float* dx; float* dw;
  float* dx_partial; float* dw_partial;
  long long E;
  int M, V, K;
  int products, sub_z, sub_mul;   // stages between two roundings to nearest: of the logits, of dx and dW
  int forward;                    // 1: STATS units over all words, nothing else
  int words_grad, v0_grad;        // piece of the G units (0 words: none)
  int words_mul, v0_mul;          // piece of the dx and dW units (0: none)
  int dx_split, dw_split, acc_dx, acc_dw, want_dx, want_dw;
  int vec_dx, vec_dw;
};

struct Unit {
  int kind;
  int m0, n0;                     // tile origin
  int kb_lo, kb_hi;               // stages
  int share;                      // of a dx or dW tile
};

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Unit u of the launch.  `rows`: rows that count.  Returns false past the last one.
__device__ __forceinline__ bool unit_of(const Params& p, int rows, int u, Unit& t) {
  const int tiles_m = ceil_div(rows, TILE), tiles_e = ceil_div((int)p.E, TILE);
  t.share = 0;
  if (p.want_dw && p.words_mul) {
    const int n = ceil_div(p.words_mul, TILE) * tiles_e * p.dw_split;
    if (u < n) {
      const int kb = ceil_div(rows, BK), per = ceil_div(kb, p.dw_split);
      t.kind = DW; t.share = u % p.dw_split; u /= p.dw_split;
      t.m0 = u / tiles_e * TILE; t.n0 = u % tiles_e * TILE;
      t.kb_lo = min(kb, t.share * per); t.kb_hi = min(kb, t.kb_lo + per);
      return true;
    }
    u -= n;
  }
  if (p.want_dx && p.words_mul) {
    const int n = tiles_m * tiles_e * p.dx_split;
    if (u < n) {
      const int kb = ceil_div(p.words_mul, BK), per = ceil_div(kb, p.dx_split);
      t.kind = DX; t.share = u % p.dx_split; u /= p.dx_split;
      t.m0 = u / tiles_e * TILE; t.n0 = u % tiles_e * TILE;
      t.kb_lo = min(kb, t.share * per); t.kb_hi = min(kb, t.kb_lo + per);
      return true;
    }
    u -= n;
  }
  const int words = p.forward ? p.V : p.words_grad;
  const int n = tiles_m * ceil_div(words, TILE);
  if (u >= n) return false;
  // rows fastest: the pairs at work share a few tiles of W, and x stays in L2
  t.kind = p.forward ? STATS : GRAD; t.m0 = u % tiles_m * TILE; t.n0 = u / tiles_m * TILE;
  t.kb_lo = 0; t.kb_hi = ceil_div((int)p.E, BK);
  return true;
}

// Instruction descriptor, kind::f16: D = fp32, A and B = fp16, M = 256 over the pair, N = 256.
__host__ __device__ constexpr uint32_t idesc_f16(bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
}
__device__ __forceinline__ void mma_f16_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n"
      ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 16 k elements further: 32 bytes along a K-major row, or two groups of 8 k rows of 128 bytes
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, bool mn, int kk) {
  return mn ? make_smem_desc(addr + kk * 2048, 8192, 1024, 2) : make_smem_desc(addr + kk * 32, 16, 1024, 2);
}
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"((uint64_t)map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int v) { asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {        // a in the low half
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float half_to_float(uint16_t h) { float f; asm("cvt.f32.f16 %0, %1;" : "=f"(f) : "h"(h)); return f; }
__device__ __forceinline__ uint16_t float_to_half(float f) { uint16_t h; asm("cvt.rn.f16.f32 %0, %1;" : "=h"(h) : "f"(f)); return h; }

// Adds without reading, so that nothing waits: one unit of a launch adds to an element, there is no order to depend on.
__device__ __forceinline__ void add_to(float* p, float a) { asm volatile("red.global.add.f32 [%0], %1;" ::"l"(p), "f"(a) : "memory"); }
__device__ __forceinline__ void add_to(float* p, const float4& a) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(a.x), "f"(a.y), "f"(a.z), "f"(a.w) : "memory");
}

// Arrival that passes on no data of this thread's.  (A releasing one of cluster scope first waits for the thread's stores to global
// memory; an epilogue warp has a whole tile of them on their way.)
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

struct Maps {
  CUtensorMap x[2], w[2], g_mul[2], g_out[2];        // hi, lo
};

__global__ void __launch_bounds__(THREADS, 1) lm_pair_kernel(const __grid_constant__ Maps maps, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* base = smem_raw + (ring - smem_u32(smem_raw));
  uint8_t* staging = base + RING_BYTES;
  uint8_t* ctrl = staging + 8 * STAGE_TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ctrl);
  const uint32_t bar_full = smem_u32(bars);                     // [stage], leader's: the bytes of both CTAs
  const uint32_t bar_empty = bar_full + 8 * MAX_STAGES;         // [stage], each CTA's own
  const uint32_t bar_tfull = bar_empty + 8 * MAX_STAGES;        // [2], each CTA's own
  const uint32_t bar_tempty = bar_tfull + 16;                   // [2], leader's: 8 warps x 2 CTAs
  const uint32_t bar_sfull = bar_tempty + 16;                   // [slot], each CTA's own: a unit has been handed out
  const uint32_t bar_sempty = bar_sfull + 8 * SLOTS;            // [slot], leader's: everybody has read it
  const uint32_t bar_drain = bar_sempty + 8 * SLOTS;
  volatile int* slots = reinterpret_cast<volatile int*>(ctrl + 512);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 512 + 4 * SLOTS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();                      // 0: leader

  if (threadIdx.x == 0) {
    for (int s = 0; s < MAX_STAGES; ++s) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(bar_tfull + 8 * a, 1); mbar_init(bar_tempty + 8 * a, 16); }
    for (int s = 0; s < SLOTS; ++s) { mbar_init(bar_sfull + 8 * s, 1); mbar_init(bar_sempty + 8 * s, 18); }   // 16 warps, the MMA thread, the other producer
    mbar_init(bar_drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  gt_let_next_kernel_start();
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  gt_wait_for_previous_kernel();
  const int rows = *(volatile int*)&p.scalars->count;
  const int stages = p.products == 3 ? 3 : 6;
  const uint32_t stage_bytes = p.products == 3 ? 4 * OPERAND_BYTES : 2 * OPERAND_BYTES;
  const uint32_t b_at = stage_bytes / 2;                        // A hi (, A lo), B hi (, B lo)
  const uint32_t leader_full = map_to_cta(bar_full, 0), leader_tempty = map_to_cta(bar_tempty, 0), leader_sempty = map_to_cta(bar_sempty, 0);

  // The next unit, for everybody but the leader's producer: waits for the slot, reads it, hands the slot back.
  int slot = 0; uint32_t slot_ph = 0;
  auto take_unit = [&](bool whole_warp, int& u) -> bool {
    const bool got = mbar_wait_cluster(bar_sfull + 8 * slot, slot_ph, abort_flag, p.status);
    if (whole_warp ? !__all_sync(0xffffffffu, got) : !got) return false;
    if (whole_warp) {
      u = __shfl_sync(0xffffffffu, lane == 0 ? slots[slot] : 0, 0);       // lane 0 has read the slot when it hands it back
      if (lane == 0) mbar_arrive_cluster_relaxed(leader_sempty + 8 * slot);
    } else {
      u = slots[slot];
      mbar_arrive_cluster(leader_sempty + 8 * slot);
    }
    if (++slot == SLOTS) { slot = 0; slot_ph ^= 1u; }
    return true;
  };

  if (warp == 0) {
    // ------------------------------ producer (one per CTA) ------------------------------
    if (lane == 0) {
      const uint32_t peer_sfull = map_to_cta(bar_sfull, 1), own_sfull = map_to_cta(bar_sfull, 0);
      const uint32_t peer_slots = map_to_cta(smem_u32((const void*)slots), 1);
      int s = 0; uint32_t ph = 0;
      long long issued = 0;
      bool ok = true;
      int next = rank == 0 ? atomicAdd(p.counter, 1) : 0;
      while (ok) {
        int u;
        Unit t;
        if (rank == 0) {
          u = next;
          if (!mbar_wait_cluster(bar_sempty + 8 * slot, slot_ph ^ 1u, abort_flag, p.status)) { ok = false; break; }
          slots[slot] = u;
          st_cluster(peer_slots + 4 * slot, u);
          mbar_arrive_cluster(own_sfull + 8 * slot);
          mbar_arrive_cluster(peer_sfull + 8 * slot);
          if (++slot == SLOTS) { slot = 0; slot_ph ^= 1u; }
        } else if (!take_unit(false, u)) { ok = false; break; }
        if (!unit_of(p, rows, u, t)) break;
        // The next unit is asked for near this one's end: its number is back in time, and a pair in a long unit does not sit on
        // work that others could do (asked for at the start, a pass over 8192 x 768 x 50257 took 7.95 ms instead of 6.91).
        const int ask = max(t.kb_lo, t.kb_hi - 2);
        if (rank == 0 && t.kb_lo >= t.kb_hi) next = atomicAdd(p.counter, 1);
        const CUtensorMap* ma = t.kind == DX || t.kind == DW ? maps.g_mul : maps.x;
        const CUtensorMap* mb = t.kind == DW ? maps.x : maps.w;
        const bool a_mn = t.kind == DW, b_mn = t.kind == DX || t.kind == DW;
        const int a0 = t.m0 + (int)rank * HALF;                 // this CTA's half of the tile's rows, and of its columns
        int b0 = t.n0 + (int)rank * HALF;
        int bk = 0;                                             // where k = 0 lies in B
        if (t.kind == GRAD) b0 += p.v0_grad;
        if (t.kind == DX) bk = p.v0_mul;
        for (int kb = t.kb_lo; kb < t.kb_hi; ++kb) {
          if (!mbar_wait_cluster(bar_empty + 8 * s, ph ^ 1u, abort_flag, p.status)) { ok = false; break; }
          if (rank == 0) {
            mbar_expect_tx(bar_full + 8 * s, 2 * stage_bytes);
            if (kb == ask) next = atomicAdd(p.counter, 1);
          }
          const uint32_t full = leader_full + 8 * s;
          const uint32_t st = ring + s * stage_bytes;
          const int k0 = kb * BK;
          // boxes of 64 x 64: two cover 128 rows of 64 k (K-major), or 64 k rows of twice 64 columns (MN-major)
          const int ax = a_mn ? a0 : k0, ay = a_mn ? k0 : a0, bx = b_mn ? b0 : k0, by = b_mn ? k0 + bk : b0;
          for (int h = 0; h < (p.products == 3 ? 2 : 1); ++h) {
            const uint32_t sa = st + h * OPERAND_BYTES, sb = st + b_at + h * OPERAND_BYTES;
            tma_load_2d_pair(sa, ma + h, full, ax, ay);
            tma_load_2d_pair(sa + 8192, ma + h, full, a_mn ? ax + 64 : ax, a_mn ? ay : ay + 64);
            tma_load_2d_pair(sb, mb + h, full, bx, by);
            tma_load_2d_pair(sb + 8192, mb + h, full, b_mn ? bx + 64 : bx, b_mn ? by : by + 64);
          }
          ++issued;
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
      }
      if (!ok && rank == 0) {       // giving up: the loads already issued complete on these barriers; give them time to land
        for (long long i = issued > stages ? issued - stages : 0; i < issued; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(bar_full + 8 * (int)(i % stages), (uint32_t)((i / stages) & 1)) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------ MMA issuer (leader CTA only) ------------------------------
    if (lane == 0 && rank == 0) {
      const uint32_t peer_empty = map_to_cta(bar_empty, 1), peer_tfull = map_to_cta(bar_tfull, 1);
      const uint32_t own_empty = map_to_cta(bar_empty, 0), own_tfull = map_to_cta(bar_tfull, 0);
      int s = 0; uint32_t ph = 0;
      int acc = 0; uint32_t aph = 0;
      bool ok = true, any_issued = false;
      int u;
      Unit t;
      while (ok) {
        if (!take_unit(false, u)) { ok = false; break; }
        if (!unit_of(p, rows, u, t)) break;
        const bool a_mn = t.kind == DW, b_mn = t.kind == DX || t.kind == DW;
        const uint32_t idesc = idesc_f16(a_mn, b_mn);
        for (int kb = t.kb_lo; ok && kb < t.kb_hi;) {
          if (!mbar_wait_cluster(bar_tempty + 8 * acc, aph ^ 1u, abort_flag, p.status)) { ok = false; break; }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + (uint32_t)(acc * TILE);
          const int end = min(t.kb_hi, kb + (t.kind <= GRAD ? p.sub_z : p.sub_mul));
          uint32_t started = 0;
          for (; kb < end; ++kb) {
            if (!mbar_wait_cluster(bar_full + 8 * s, ph, abort_flag, p.status)) { ok = false; break; }
            tc_fence_after();
            const uint32_t sa = ring + s * stage_bytes, sb = sa + b_at;
            if (p.products == 3) {       // the small products first, while the accumulator is small
#pragma unroll
              for (int kk = 0; kk < BK / 16; ++kk) {
                mma_f16_pair(d_tmem, operand_desc(sa + OPERAND_BYTES, a_mn, kk), operand_desc(sb, b_mn, kk), idesc, started);
                started = 1;
                mma_f16_pair(d_tmem, operand_desc(sa, a_mn, kk), operand_desc(sb + OPERAND_BYTES, b_mn, kk), idesc, 1u);
              }
            }
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk) {
              mma_f16_pair(d_tmem, operand_desc(sa, a_mn, kk), operand_desc(sb, b_mn, kk), idesc, started);
              started = 1;
            }
            any_issued = true;
            tc_commit_pair(own_empty + 8 * s);
            tc_commit_pair(peer_empty + 8 * s);
            if (++s == stages) { s = 0; ph ^= 1u; }
          }
          if (!ok) break;
          tc_commit_pair(own_tfull + 8 * acc);
          tc_commit_pair(peer_tfull + 8 * acc);
          if (++acc == 2) { acc = 0; aph ^= 1u; }
        }
      }
      if (!ok && any_issued) {
        tc_commit_pair(map_to_cta(bar_drain, 0));
        const long long t0 = clock64();
        while (!mbar_try_wait(bar_drain, 0) && clock64() - t0 < WAIT_LIMIT_CYCLES) {}
      }
    }
  } else {
    // ------------------------------ epilogue: warp e holds rows 32 q .. + 31, columns 128 half .. + 127 ------------------------------
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * HALF);
    uint8_t* tile = staging + (warp - 2) * STAGE_TILE;
    const uint32_t tile_u32 = smem_u32(tile);
    const float logit2 = p.scalars->logit2;
    int acc = 0; uint32_t aph = 0;
    bool ok = true;
    int u;
    Unit t;
    while (ok) {
      if (!take_unit(true, u)) break;
      if (!unit_of(p, rows, u, t)) break;
      const int row = t.m0 + (int)rank * HALF + quarter * 32 + lane;      // row of the tile's matrix: a compact row, or a word (dW)
      const int col0 = t.n0 + half * HALF;
      // what the row needs, asked for before the accumulators are waited for
      float2 st = make_float2(0.0f, 1.0f), fac = make_float2(0.0f, 0.0f);
      const int* ids = nullptr; const float* q = nullptr;
      int k = 0, next_id = 0x7fffffff;
      if (t.kind == DX) st.x = p.scalars->dx;
      if (t.kind == DW) st.x = p.scalars->dw;
      if (t.kind <= GRAD && row < rows) {
        if (t.kind == GRAD) { st = p.stats[row]; fac = p.factor[row]; }
        const long long r = p.row_of[row];
        ids = p.ids + r * p.K; q = p.q + r * p.K;
        const int first = (t.kind == GRAD ? p.v0_grad : 0) + col0;                     // first target at or behind this warp's columns
        int lo = 0, hi = p.K;
        while (lo < hi) { const int mid = (lo + hi) >> 1; if (ids[mid] < first) lo = mid + 1; else hi = mid; }
        k = lo;
        if (k < p.K) next_id = ids[k];
      }
      float v[128];
      if (t.kb_lo >= t.kb_hi) {
#pragma unroll
        for (int i = 0; i < 128; ++i) v[i] = 0.0f;
      }
      const int sub = t.kind <= GRAD ? p.sub_z : p.sub_mul;
      for (int kb = t.kb_lo; kb < t.kb_hi; kb += sub) {
        const bool got = mbar_wait_cluster(bar_tfull + 8 * acc, aph, abort_flag, p.status);
        if (!__all_sync(0xffffffffu, got)) { ok = false; break; }
        tc_fence_after();
        const uint32_t at = lane_base + (uint32_t)(acc * TILE);
        if (kb == t.kb_lo) {
#pragma unroll
          for (int c = 0; c < 4; ++c) tc_ld32(at + 32 * c, v + 32 * c);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c) {                         // 16 at a time: 168 registers are what a thread may have
            float w[16];
            tc_ld16(at + 16 * c, w);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) v[16 * c + i] += w[i];
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(leader_tempty + 8 * acc);      // the loads are complete (wait::ld)
        if (++acc == 2) { acc = 0; aph ^= 1u; }
      }
      if (!ok) break;

      if (t.kind == STATS) {
        const int left = p.V - col0;                            // columns of this half that are words
        // The targets among these words: a lane puts its row through the staging tile (its own part of it, swizzled) to pick from
        // it by index.  The loss takes the targets' logits from here rather than from an exact product: what the additions in
        // tensor memory cut off is then in both sides of z - log sum e^z.
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int word0 = col0 + 32 * c;
          if (!__any_sync(0xffffffffu, next_id < word0 + 32)) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(tile + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                make_float4(v[32 * c + 4 * j], v[32 * c + 4 * j + 1], v[32 * c + 4 * j + 2], v[32 * c + 4 * j + 3]);
          while (next_id < word0 + 32) {
            const int n = next_id - word0;
            p.target_z[(long long)row * p.K + k] = logit2 * *reinterpret_cast<const float*>(tile + lane * 128 + (((n >> 2) ^ (lane & 7)) << 4) + (n & 3) * 4);
            next_id = ++k < p.K ? ids[k] : 0x7fffffff;
          }
          __syncwarp();
        }
        float2 out = make_float2(-INFINITY, 0.0f);
        if (left > 0) {
          if (left < HALF) {
#pragma unroll
            for (int i = 0; i < 128; ++i) if (i >= left) v[i] = -INFINITY;
          }
          float mx = v[0];
#pragma unroll
          for (int i = 1; i < 128; ++i) mx = fmaxf(mx, v[i]);
          const float m2 = mx * logit2;
          float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
#pragma unroll
          for (int i = 0; i < 128; i += 4) {
            s0 += gt_ex2(fmaf(v[i], logit2, -m2)); s1 += gt_ex2(fmaf(v[i + 1], logit2, -m2));
            s2 += gt_ex2(fmaf(v[i + 2], logit2, -m2)); s3 += gt_ex2(fmaf(v[i + 3], logit2, -m2));
          }
          out = make_float2(m2, (s0 + s1) + (s2 + s3));
        }
        if (row < rows) p.partial[(long long)(t.n0 / HALF + half) * p.M + row] = out;
      } else if (t.kind == GRAD) {
        const bool live = row < rows;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int first = col0 + 32 * c;                      // within the piece
          if (first >= p.words_grad) break;
#pragma unroll
          for (int n = 32 * c; n < 32 * c + 32; n += 2) {       // in place: the halves of two columns take their registers
            float g0 = fac.x * gt_ex2(fmaf(v[n], logit2, -st.x)), g1 = fac.x * gt_ex2(fmaf(v[n + 1], logit2, -st.x));
            if (!live) { g0 = 0.0f; g1 = 0.0f; }
            const uint32_t hi = pack_half2(g0, g1);
            v[n] = __uint_as_float(hi);
            v[n + 1] = __uint_as_float(pack_half2(g0 - half_to_float((uint16_t)hi), g1 - half_to_float((uint16_t)(hi >> 16))));
          }
          if (lane == 0) tma_store_wait_read<0>();              // the staging tile is free again
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {                         // 8 columns: 16 bytes of hi, 16 of lo
            const int at = lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4);        // 64-byte swizzle
            const float* b = v + 32 * c + 8 * j;
            *reinterpret_cast<float4*>(tile + at) = make_float4(b[0], b[2], b[4], b[6]);
            *reinterpret_cast<float4*>(tile + 2048 + at) = make_float4(b[1], b[3], b[5], b[7]);
          }
          const int word0 = p.v0_grad + first;
          while (next_id < word0 + 32) {                        // this row's targets among these words
            const int n = next_id - word0;
            const int at = lane * 64 + (((n >> 3) ^ ((lane >> 1) & 3)) << 4) + (n & 7) * 2;
            uint16_t* ph = reinterpret_cast<uint16_t*>(tile + at);
            uint16_t* pl = reinterpret_cast<uint16_t*>(tile + 2048 + at);
            const float g = (half_to_float(*ph) + half_to_float(*pl)) - fac.y * q[k];
            const uint16_t h = float_to_half(g);
            *ph = h;
            *pl = float_to_half(g - half_to_float(h));
            next_id = ++k < p.K ? ids[k] : 0x7fffffff;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            const int r0 = t.m0 + (int)rank * HALF + quarter * 32;
            if (r0 < p.M) {
              tma_store_2d(&maps.g_out[0], tile_u32, first, r0);
              if (p.products == 3) tma_store_2d(&maps.g_out[1], tile_u32 + 2048, first, r0);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          }
        }
      } else {
        // dx or dW: 32 x 32 blocks through shared memory, so that a warp writes whole lines
        const bool is_dw = t.kind == DW;
        const float alpha = st.x;
        const bool share = (is_dw ? p.dw_split : p.dx_split) > 1;
        const bool add = share ? false : is_dw ? p.acc_dw != 0 : (p.acc_dx != 0 || p.v0_mul > 0);
        const bool vec = (share || (is_dw ? p.vec_dw : p.vec_dx) != 0) && p.E % 4 == 0;
        const int row_base = t.m0 + (int)rank * HALF + quarter * 32;
        const int row_end = is_dw ? p.words_mul : rows;
        float* out = is_dw ? (share ? p.dw_partial + (long long)t.share * p.words_mul * p.E : p.dw + (long long)p.v0_mul * p.E)
                           : (share ? p.dx_partial + (long long)t.share * p.M * p.E : p.dx);
        const bool linear = is_dw || share;
        float* const line = out + (long long)(row_base + (lane >> 3)) * p.E + 4 * (lane & 7);
        const int lines = row_end - row_base - (lane >> 3);
        int mine = row_base + lane;                             // lane l knows where row l goes
        if (!is_dw && !share && mine < row_end) mine = p.row_of[mine];
        if (lane == 0) tma_store_wait_read<0>();                // a G unit may have used the staging tile before
        __syncwarp();
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int first = col0 + 32 * c;
          if (first >= (int)p.E || row_base >= row_end) break;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<float4*>(tile + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                make_float4(alpha * v[32 * c + 4 * j], alpha * v[32 * c + 4 * j + 1], alpha * v[32 * c + 4 * j + 2], alpha * v[32 * c + 4 * j + 3]);
          __syncwarp();
          if (vec && linear) {                                  // rows one after the other: a pointer that moves on
            float* dst = line + first;
            const bool inside = first + 4 * (lane & 7) < (int)p.E;
#pragma unroll
            for (int it = 0; it < 8; ++it, dst += 4 * p.E) {
              const int r = it * 4 + (lane >> 3);
              if (inside && 4 * it < lines) {
                const float4 a = *reinterpret_cast<const float4*>(tile + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                if (add) add_to(dst, a);
                else *reinterpret_cast<float4*>(dst) = a;
              }
            }
          } else if (vec) {
            const int j = lane & 7, col = first + 4 * j;
#pragma unroll
            for (int it = 0; it < 8; ++it) {
              const int r = it * 4 + (lane >> 3);
              const int to = __shfl_sync(0xffffffffu, mine, r);
              if (row_base + r < row_end && col < (int)p.E) {
                const float4 a = *reinterpret_cast<const float4*>(tile + r * 128 + ((j ^ (r & 7)) << 4));
                float* dst = out + (long long)to * p.E + col;
                if (add) add_to(dst, a);
                else *reinterpret_cast<float4*>(dst) = a;
              }
            }
          } else {
#pragma unroll 4
            for (int r = 0; r < 32; ++r) {
              const int to = __shfl_sync(0xffffffffu, mine, r);
              if (row_base + r < row_end && first + lane < (int)p.E) {
                const float a = *reinterpret_cast<const float*>(tile + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                float* dst = out + (long long)to * p.E + first + lane;
                if (add) add_to(dst, a);
                else *dst = a;
              }
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync_all();                    // nobody leaves while the peer may still signal or read this CTA
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
  }
}

// ---- host ------------------------------------------------------------------------------------------

int encode_half(gt_ctx* ctx, CUtensorMap* map, const uint16_t* ptr, long long cols, long long rows, long long pitch, int box_cols, int box_rows,
                CUtensorMapSwizzle swizzle) {
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)pitch * 2ull};
  cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = ctx->encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, (void*)ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    GT_FAIL(ctx, GT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d): ptr=%p cols=%lld rows=%lld pitch=%lld box=(%d,%d)", (int)r, (const void*)ptr, cols,
            rows, pitch, box_cols, box_rows);
  return GT_OK;
}

int encode_pair(gt_ctx* ctx, CUtensorMap* maps, const LmSplit& s, const LmProblem& p, long long cols, long long rows, long long pitch, int box_cols,
                int box_rows, CUtensorMapSwizzle swizzle) {
  int rc = encode_half(ctx, &maps[0], s.hi, cols, rows, pitch, box_cols, box_rows, swizzle);
  if (rc == GT_OK) rc = encode_half(ctx, &maps[1], p.products == 3 ? s.lo : s.hi, cols, rows, pitch, box_cols, box_rows, swizzle);
  return rc;
}

void launch_config(cudaLaunchConfig_t* cfg, cudaLaunchAttribute* attr, int pairs, cudaStream_t stream) {
  memset(cfg, 0, sizeof(*cfg));
  cfg->gridDim = dim3(2u * (unsigned)pairs, 1, 1);
  cfg->blockDim = dim3(THREADS, 1, 1);
  cfg->dynamicSmemBytes = SMEM_BYTES;
  cfg->stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = gt_pdl_enabled() ? 1 : 0;
  cfg->attrs = attr;
  cfg->numAttrs = 2;
}

Params common_params(gt_ctx* ctx, const LmProblem& p) {
  Params a;
  memset(&a, 0, sizeof(a));
  a.scalars = p.scalars; a.status = ctx->d_status; a.row_of = p.row_of;
  a.stats = p.stats; a.factor = p.factor; a.ids = p.ids; a.q = p.q; a.K = p.K;
  a.partial = p.partial; a.target_z = p.target_z;
  a.E = p.E; a.M = (int)p.M; a.V = (int)p.V;
  a.products = p.products;
  // Between two roundings to nearest: 128 or 192 of K with three products (24, 36 additions), 512 with one, whose operands are rounded
  // to 11 bits anyway.  Every hand-over costs the tensor cores about 450 cycles.  8192 x 768 x 50257 with gradients, by stages of
  // 64 between two hand-overs, time and error of dx against 64 bits: 2: 6.91 ms, 3.0e-7; 3: 6.46 ms, 4.3e-7; 4: 6.46 ms,
  // 5.8e-7; 6: 6.31 ms, 8.6e-7.  The logits have the smaller number: the loss subtracts the targets' from them in 32 bits, so
  // their bias stays in it.  It is the same one forward and backward: p is a quotient of the two, and the bias cancels.
  a.sub_z = p.products == 3 ? 2 : 8;
  a.sub_mul = p.products == 3 ? 3 : 8;
  a.dx_split = a.dw_split = 1;
  return a;
}

int launch(gt_ctx* ctx, const Maps& maps, const Params& a, long long units) {
  GT_SMEM_OPT_IN(ctx, lm_pair_kernel, SMEM_BYTES);
  int pairs = gt_lm_pairs(ctx);
  if (pairs <= 0) GT_FAIL(ctx, GT_ERR_UNSUPPORTED, "no pair of CTAs of the loss kernel fits on this device");
  if (pairs > units) pairs = (int)units;
  cudaLaunchConfig_t cfg; cudaLaunchAttribute attr[2];
  launch_config(&cfg, attr, pairs, ctx->stream);
  GT_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, lm_pair_kernel, maps, a));
  ctx->launches += 1;
  return GT_OK;
}

long long tiles(long long n) { return (n + TILE - 1) / TILE; }

}  // namespace

int gt_lm_pairs(gt_ctx* ctx) {
  static int cached[64];
  static bool known[64];
  if (ctx->device < 0 || ctx->device >= 64) return 0;
  if (!known[ctx->device]) {
    int n = 0;
    cudaLaunchConfig_t cfg; cudaLaunchAttribute attr[2];
    launch_config(&cfg, attr, ctx->sm_count / 2, ctx->stream);
    cfg.numAttrs = 1;                    // the question concerns the cluster's shape only
    if (cudaFuncSetAttribute(lm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, lm_pair_kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
    cached[ctx->device] = n;
    known[ctx->device] = true;
  }
  return cached[ctx->device];
}

int gt_lm_stats(gt_ctx* ctx, const LmProblem& p) {
  Maps maps;
  memset(&maps, 0, sizeof(maps));
  int rc = encode_pair(ctx, maps.x, p.x, p, p.E, p.M, p.pitch_e, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == GT_OK) rc = encode_pair(ctx, maps.w, p.w, p, p.E, p.V, p.pitch_e, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc != GT_OK) return rc;
  Params a = common_params(ctx, p);
  a.forward = 1;
  a.counter = p.counters;
  return launch(ctx, maps, a, tiles(p.M) * tiles(p.V));
}

int gt_lm_step(gt_ctx* ctx, const LmProblem& p, int piece) {
  Maps maps;
  memset(&maps, 0, sizeof(maps));
  Params a = common_params(ctx, p);
a.words_grad = (int)lm_piece_words(p, piece); a.v0_grad = (int)(piece * p.words);
  a.words_mul = (int)lm_piece_words(p, piece - 1); a.v0_mul = (int)((piece - 1) * p.words);
  int rc = encode_pair(ctx, maps.x, p.x, p, p.E, p.M, p.pitch_e, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == GT_OK) rc = encode_pair(ctx, maps.w, p.w, p, p.E, p.V, p.pitch_e, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == GT_OK && a.words_mul)
    rc = encode_pair(ctx, maps.g_mul, p.g[(piece + 1) & 1], p, a.words_mul, p.M, p.pitch_v, 64, 64, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc == GT_OK && a.words_grad)
    rc = encode_pair(ctx, maps.g_out, p.g[piece & 1], p, a.words_grad, p.M, p.pitch_v, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc != GT_OK) return rc;
  a.counter = p.counters + piece;
  a.dx = p.dx; a.dw = p.dw; a.acc_dx = p.acc_dx; a.acc_dw = p.acc_dw;
  a.want_dx = p.dx != nullptr; a.want_dw = p.dw != nullptr;
  a.dx_split = p.dx_split; a.dx_partial = p.dx_partial;
  a.dw_split = lm_dw_split(ctx, p, a.words_mul, a.words_grad); a.dw_partial = p.dw_partial;
  a.vec_dx = ((uintptr_t)p.dx & 15) == 0 && p.E % 4 == 0;
  a.vec_dw = ((uintptr_t)p.dw & 15) == 0 && p.E % 4 == 0;
  const long long units = tiles(a.words_mul) * tiles(p.E) * a.dw_split * (p.dw != nullptr) +
                          (a.words_mul ? tiles(p.M) * tiles(p.E) * p.dx_split * (p.dx != nullptr) : 0) + tiles(p.M) * tiles(a.words_grad);
  return launch(ctx, maps, a, units);
}
