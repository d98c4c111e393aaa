// attn.key_mass: how much softmax weight a window of queries gives to every cached row.
//
// For the T queries of a sequence (its last T tokens, query t seeing the rows 0 .. ctx - T + t) and the G query heads of
// a KV head, with s_ti = q_t . k_i * scale and lse_t = log sum_i exp(s_ti):
//   key_mass_i (+)= sum_t sum_g exp(s_tgi - lse_tg).
// Two passes over the scores: the first finds lse of every query row, the second adds up columns.  The scores of a pass
// are not kept: T G values a row are more bytes than the row itself as soon as T G > D / 2.
//
// Bound, for long windows: the tensor pipe and the special-function unit alike (a 128 x 128 tile of D = 256 is 1024
// cycles of MMA and 1024 of exponentials), for short ones the launches and one tile's latency.
//
// Both passes are the same pipeline: a warp of TMA loads, a warp that issues tcgen05.mma (M = N = 128,
// fp32 accumulators in tensor memory, four of them), and four groups of four warps that read one each in turn.
// Pass 1 holds a block of query rows (lanes) and streams 128-key tiles (columns): a thread owns a query row and keeps
// its running maximum and sum.  Pass 2 holds a 128-key tile (lanes) and streams the blocks of query rows that see it: a
// thread owns a key and adds up exp2(s - lse).  So every reduction runs along a thread's own columns, every sum has one
// owner and a fixed order, and nothing is exchanged but the groups' partial sums.
// The groups' arithmetic is what takes longest to keep up: four warps per scheduler hide its latency, two numbers go to
// an fma or add (f32x2), tiles that every row sees whole have a path without a mask.  (Graph replays of one
// input.  Two groups, a mask for every tile, one number at a time: 273 us instead of 245 for 2047 queries over 8192 rows.
// The held operand in tensor memory and three groups: 239, but 44 instead of 37 for 32 queries over four prompts at a tile
// per CTA in pass 2, whose one load per item it exposes.  Several tiles per CTA have since made 30 of the 37.)
//
// A block holds the (token, head) pairs of floor(128 / G) tokens, fetched as one 3-D box; the keys come straight from the
// pages where the cache is bf16 and its pages hold whole swizzle atoms (8 rows), else from a bf16 copy made first.
#include <cuda.h>
#include "abi.h"
#include "attn_pages.cuh"
#include "kv_formats.cuh"
#include "tc_host.h"
#include "tc_ptx.cuh"

namespace q35 {

constexpr int KM_TILE = 128;    // query rows per block, keys per tile
constexpr int KM_GROUPS = 4;    // groups of four warps that read accumulators
constexpr int KM_THREADS = 128 + 128 * KM_GROUPS;  // TMA, MMA, two spare warps, the groups
constexpr int KM_ACC = KM_GROUPS;  // accumulators of 128 columns, all of tensor memory.  A group always reads the same one:
                                // it waits for the next phase of that one's barrier and cannot take an older for it
constexpr int KM_ITEMS = 16;    // most tiles of a CTA in pass 2
constexpr float KM_LOG2E = 1.4426950408889634f;

struct MassArgs {
  PageTable t;
  const int* qo_indptr;        // [B + 1]
  const float* kv_scale;       // E4M3
  const float* sm_scale;       // optional [1]
  float* key_mass;             // [pages, P, HKV]
  float2* part;                // workspace [splits][T_total HQ]: maximum and sum of a query row over a range of keys
  int T_total, HQ, HKV, G, D, splits, accumulate, e4m3;
  int tokens;                  // tokens per block of query rows
  int box_rows;                // rows per TMA box of keys
  int copied;                  // keys come from the bf16 copy [HKV, n_indices P, D]
};

// the window of sequence b: tokens q0 .. q0 + T - 1 of q, the first of them at position `first`; T = 0 if there is none, and
// `refused` if what the table says is no window of this sequence: recorded, and its weights stay as they are
struct Window { int q0, T, first; bool refused; };
__device__ __forceinline__ Window window_of(const MassArgs& a, int b, const SeqPages& sp) {
  const int q0 = a.qo_indptr[b], q1 = a.qo_indptr[b + 1];
  if (q0 < 0 || q1 < q0 || q1 > a.T_total || q1 - q0 > sp.ctx) {  // the cache must hold the window's own rows
    atomicOr(a.t.status, DS_BAD_TOKEN);
    return {0, 0, 0, true};
  }
  return {q0, q1 - q0, sp.ctx - (q1 - q0), false};
}

__device__ __forceinline__ float mass_scale(const MassArgs& a, int kvh) {
  const float k_mul = !a.e4m3 ? 1.f : a.kv_scale ? a.kv_scale[kvh] : 0.125f;
  return (a.sm_scale ? a.sm_scale[0] : rsqrtf(float(a.D))) * KM_LOG2E * k_mul;
}

// ---- the pipeline's own PTX -----------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
// D[tmem] (+)= A[smem] B[smem], bf16 with fp32 accumulation.  Instruction descriptor: [4,6) 1 = fp32 result, [7,10) and
// [10,13) 1 = bf16 A and B, [17,23) N >> 3, [24,29) M >> 4
constexpr uint32_t KM_IDESC = 1u << 4 | 1u << 7 | 1u << 10 | uint32_t(KM_TILE >> 3) << 17 | uint32_t(KM_TILE >> 4) << 24;
__device__ __forceinline__ void tc_mma_bf16(uint32_t d, uint64_t ad, uint64_t bd, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(ad), "l"(bd), "r"(KM_IDESC), "r"(accumulate) : "memory");
}
// this warp's 32 lanes x 32 consecutive columns of fp32 accumulators
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr) : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// two fp32 numbers to an instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(v));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(x), "l"(y), "l"(z));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(x), "l"(y));
  return d;
}
__device__ __forceinline__ uint64_t ex2_pair(uint64_t v) {
  const float2 x = halves(v);
  return pair(ex2(x.x), ex2(x.y));
}

template <int D>
struct MassCfg {
  static constexpr int PANELS = D / 64;                  // 64 channels = the 128 bytes of a swizzled row
  static constexpr int PANEL = KM_TILE * 128;
  static constexpr int OPERAND = PANELS * PANEL;         // a block or tile: 64 KB at D = 256
  static constexpr int STAGES = D == 256 ? 2 : 4;
  static constexpr int SMEM = 1024 + (1 + STAGES) * OPERAND;
};

// What a CTA works on: a block of query rows (pass 1) or a tile of keys (pass 2) of one (sequence, KV head), and the n
// tiles or blocks from `begin` on that it meets; the first of them is the CTA's t0-th.
struct MassItem {
  int b, index, kvh, begin, n, t0;
  SeqPages sp;
  Window w;
  float scale;
};

template <int D, bool SUM>
__global__ void __launch_bounds__(KM_THREADS, 1)
    mass_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const MassArgs a) {
  using C = MassCfg<D>;
  using namespace tc;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * C::STAGES + 2 * KM_ACC + 2];
  __shared__ uint32_t s_tmem;
  __shared__ MassItem s_item[KM_ITEMS];
  __shared__ __align__(16) float s_lse[KM_GROUPS][2][KM_TILE];  // [group][turn]: minus the lse of the block's query rows
  __shared__ int s_see[KM_GROUPS][2][KM_TILE];                  // and the last key that each of them sees
  __shared__ float s_sum[2][KM_GROUPS][KM_TILE];                // the groups' maxima and sums (pass 2: sums, by turns)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t sbase = (smem_u32(smem_raw) + 1023u) & ~1023u;  // swizzled tiles start on 1024 bytes
  const uint32_t held = sbase, ring = sbase + C::OPERAND;
  const uint32_t bars = smem_u32(s_bar);
  auto full = [&](int s) { return bars + 8 * s; };
  auto empty = [&](int s) { return bars + 8 * (C::STAGES + s); };
  auto acc_full = [&](int i) { return bars + 8 * (2 * C::STAGES + i); };
  auto acc_empty = [&](int i) { return bars + 8 * (2 * C::STAGES + KM_ACC + i); };
  const uint32_t held_full = bars + 8 * (2 * C::STAGES + 2 * KM_ACC), held_empty = held_full + 8;
  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (int i = 0; i < KM_ACC; ++i) { mbar_init(acc_full(i), 1); mbar_init(acc_empty(i), 128); }
    mbar_init(held_full, 1);
    mbar_init(held_empty, 1);
    fence_barrier_init();
    tma_prefetch_desc(&qmap);
    tma_prefetch_desc(&kmap);
  }
  pdl_wait();
  pdl_launch();
  // the CTA's items, one warp to each: pass 1 has one per CTA, pass 2 every gridDim.x-th
  if (warp < (SUM ? KM_ITEMS : 1)) {
    MassItem it{};
    const int64_t number = blockIdx.x + int64_t(warp) * gridDim.x;
    it.b = -1;
    if (number < int64_t(INT_MAX)) {
      const int2 at = find_item(a.t.B, int(number) / a.HKV, [&](int b) {
        const SeqPages sp = seq_pages(a.t, b);
        if (SUM) return (sp.ctx + KM_TILE - 1) / KM_TILE;
        const int T = window_of(a, b, sp).T;
        return (T + a.tokens - 1) / a.tokens;
      });
      it.b = at.x;
      it.index = at.y;
    }
    if (it.b >= 0) {
      it.kvh = int(number) % a.HKV;
      it.sp = seq_pages(a.t, it.b);
      it.w = window_of(a, it.b, it.sp);
      it.scale = mass_scale(a, it.kvh);
      const Window w = it.w;
      const int blocks = (w.T + a.tokens - 1) / a.tokens;
      if (SUM) {
        it.begin = min(blocks, max(0, it.index * KM_TILE - w.first) / a.tokens);  // the first that sees the tile's first key
        it.n = blocks - it.begin;
      } else {
        it.index = blocks - 1 - it.index;  // the blocks that see most come first
        const int last = min(w.T, (it.index + 1) * a.tokens) - 1, tiles = (w.first + last) / KM_TILE + 1;
        const int per = (tiles + a.splits - 1) / a.splits;
        it.begin = min(tiles, int(blockIdx.y) * per);
        it.n = min(tiles, it.begin + per) - it.begin;
      }
    }
    if (lane == 0) s_item[warp] = it;
  }
  // blocks of a.tokens tokens leave the last rows of an operand untouched: zeros there, so that nothing old is NaN
  const int block_rows = a.tokens * a.G;
  if (block_rows < KM_TILE) {
    const int first_op = SUM ? 1 : 0, n_op = SUM ? C::STAGES : 1, per = (KM_TILE - block_rows) * 8;  // 16-byte pieces
    for (int i = tid; i < n_op * C::PANELS * per; i += KM_THREADS) {
      const int panel = i / per, at = i % per;
      asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};"
                   ::"r"(sbase + first_op * C::OPERAND + panel * C::PANEL + block_rows * 128 + at * 16), "r"(0u));
    }
    fence_proxy_async();
  }
  __syncthreads();
  if (s_item[0].b < 0) return;  // fewer items than the grid's bound
  int items = 1;
  while (SUM && items < KM_ITEMS && s_item[items].b >= 0) ++items;
  if (tid == 0)
    for (int k = 1; k < items; ++k) s_item[k].t0 = s_item[k - 1].t0 + s_item[k - 1].n;
  if (warp == 2) { tmem_alloc(smem_u32(&s_tmem), KM_ACC * KM_TILE); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&s_tmem);

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA
    const int boxes = KM_TILE / a.box_rows;
    // lane l: the row of the tensor map where box l of a tile starts, -1 = behind the end of the sequence
    auto box_at = [&](const MassItem& it, int tile) -> int {
      const int pos = tile * KM_TILE + lane * a.box_rows;
      if (lane >= boxes || pos >= it.sp.ctx) return -1;
      if (a.copied) return it.kvh * (a.t.n_indices * a.t.P) + it.sp.first * a.t.P + pos;
      const int e = a.t.page_of(pos), id = page_at(a.t, it.sp.first + e);
      return (id < 0 ? 0 : id) * 2 * a.t.P + (pos - e * a.t.P);
    };
    auto load_keys = [&](const MassItem& it, int y, uint32_t dst, uint32_t bar) {
      const int x0 = a.copied ? 0 : it.kvh * D;
      const int there = __popc(__ballot_sync(0xffffffffu, y >= 0));
      if (lane == 0) mbar_expect_tx(bar, there * a.box_rows * 128 * C::PANELS);
      __syncwarp();
      for (int i0 = 0; i0 < there * C::PANELS; i0 += 32) {
        const int i = i0 + lane, row = __shfl_sync(0xffffffffu, y, (i / C::PANELS) & 31);
        if (i < there * C::PANELS)
          tma_load_2d(dst + (i % C::PANELS) * C::PANEL + (i / C::PANELS) * a.box_rows * 128, &kmap, bar,
                      x0 + (i % C::PANELS) * 64, row);
      }
    };
    auto load_block = [&](const MassItem& it, int blk, uint32_t dst, uint32_t bar) {
      if (lane == 0) mbar_expect_tx(bar, block_rows * 128 * C::PANELS);
      __syncwarp();
      if (lane < C::PANELS)
        tma_load_3d(dst + lane * C::PANEL, &qmap, bar, lane * 64, it.kvh * a.G, it.w.q0 + blk * a.tokens);
    };
    int t = 0, holds = 0;
    bool ok = true;
    int y_held = SUM ? box_at(s_item[0], s_item[0].index) : 0;  // looked up an item ahead
    for (int k = 0; ok && k < items; ++k) {
      const MassItem it = s_item[k];
      const int y_now = y_held;
      if (SUM && k + 1 < items) y_held = box_at(s_item[k + 1], s_item[k + 1].index);
      if (SUM && it.n == 0) continue;  // a sequence without a window
      if (SUM && !mbar_wait(held_empty, (holds & 1) ^ 1)) {
        atomicOr(a.t.status, DS_WAIT_TIMEOUT | 0x10);
        break;
      }
      if (SUM) load_keys(it, y_now, held, held_full);
      else load_block(it, it.index, held, held_full);
      ++holds;
      int y = SUM ? 0 : box_at(it, it.begin);
      for (int j = 0; j < it.n; ++j, ++t) {
        const int s = t % C::STAGES, next = !SUM && j + 1 < it.n ? box_at(it, it.begin + j + 1) : -1;
        if (!mbar_wait(empty(s), (t / C::STAGES & 1) ^ 1)) {
          atomicOr(a.t.status, DS_WAIT_TIMEOUT | 0x10);
          ok = false;
          break;
        }
        if (SUM) load_block(it, it.begin + j, ring + s * C::OPERAND, full(s));
        else load_keys(it, y, ring + s * C::OPERAND, full(s));
        y = next;
      }
    }
    // no load is on its way when the block ends, whichever wait ran out
    if (holds) mbar_wait(held_full, (holds - 1) & 1);
    for (int k = max(0, t - C::STAGES); k < t; ++k) mbar_wait(full(k % C::STAGES), k / C::STAGES & 1);
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (elect_one()) {
      // descriptors once: an offset in bytes / 16 is added to their address field (one thread issues all, instruction by
      // instruction: building a descriptor per MMA took longer than the MMA)
      const uint64_t held_desc = smem_desc(held, 16, 1024, 2), ring_desc = smem_desc(ring, 16, 1024, 2);
      int t = 0, holds = 0;
      bool ok = true;
      for (int k = 0; ok && k < items; ++k) {
        const int n = s_item[k].n;
        if (SUM && n == 0) continue;
        if (!mbar_wait(held_full, holds++ & 1)) {
          atomicOr(a.t.status, DS_WAIT_TIMEOUT | 0x40);
          break;
        }
        for (int j = 0; j < n; ++j, ++t) {
          const int s = t % C::STAGES, i = t % KM_ACC;
          if (!mbar_wait(acc_empty(i), (t / KM_ACC & 1) ^ 1)) {
            atomicOr(a.t.status, DS_WAIT_TIMEOUT | 0x20);
            ok = false;
            break;
          }
          if (!mbar_wait(full(s), t / C::STAGES & 1)) {
            atomicOr(a.t.status, DS_WAIT_TIMEOUT | 0x40);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t streamed = ring_desc + s * (C::OPERAND / 16);
#pragma unroll
          for (int p = 0; p < C::PANELS; ++p)
#pragma unroll
            for (int c = 0; c < 4; ++c)  // 16 channels = 32 bytes of a panel's rows
              tc_mma_bf16(tmem + i * KM_TILE, held_desc + (p * C::PANEL + c * 32) / 16,
                          streamed + (p * C::PANEL + c * 32) / 16, (p | c) != 0);
          tc_commit(empty(s));
          tc_commit(acc_full(i));
        }
        if (SUM && ok && k + 1 < items) tc_commit(held_empty);
      }
      // nor a product
      for (int k = max(0, t - KM_ACC); k < t; ++k) mbar_wait(acc_full(k % KM_ACC), k / KM_ACC & 1);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- accumulators: group g takes every fourth one
    const int g = (warp - 4) / 4, row = (warp & 3) * 32 + lane;
    const uint32_t quarter = tmem + (uint32_t((warp & 3) * 32) << 16);
    // false once a wait has run out (for the whole warp alike); the group's barriers are met all the same
    bool alive = true;
    auto wait_acc = [&](int t) {
      if (alive && !__all_sync(0xffffffffu, mbar_wait(acc_full(t % KM_ACC), t / KM_ACC & 1))) {
        atomicOr(a.t.status, DS_WAIT_TIMEOUT | 0x100);
        alive = false;
      }
      tc_fence_after();
      return alive;
    };
    auto done = [&](int t) {
      tc_fence_before();
      mbar_arrive(acc_empty(t % KM_ACC));
    };
    if constexpr (!SUM) {
      const MassItem it = s_item[0];
      const Window w = it.w;
      const int item = it.index, begin = it.begin, n = it.n;
      const float scale = it.scale;
      const int tok = item * a.tokens + row / a.G;
      const bool real = row < block_rows && tok < w.T;
      const int see = w.first + tok, see_min = w.first + item * a.tokens;
      float m = -INFINITY, l = 0.f;
      const uint64_t scale2 = pair(scale, scale);
      for (int t = g; t < n; t += KM_GROUPS) {
        const int k0 = (begin + t) * KM_TILE;
        const bool masked = k0 + KM_TILE - 1 > see_min;  // some row of the block does not see all of the tile
        if (!wait_acc(t)) break;
#pragma unroll 1
        for (int c0 = 0; c0 < KM_TILE; c0 += 32) {
          float v[32];
          tmem_ld_x32(quarter + t % KM_ACC * KM_TILE + c0, v);
          if (c0 == KM_TILE - 32) done(t);
          if (masked) {
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              v[i] = k0 + c0 + i > see ? -INFINITY : v[i] * scale;
              top = fmaxf(top, v[i]);
            }
            const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn;
            l *= ex2(m - base);
#pragma unroll
            for (int i = 0; i < 32; ++i) l += ex2(v[i] - base);
            m = mn;
          } else {
            float hi[4] = {v[0], v[1], v[2], v[3]}, lo[4] = {v[0], v[1], v[2], v[3]};
            if (scale >= 0.f) {
#pragma unroll
              for (int i = 4; i < 32; ++i) hi[i & 3] = fmaxf(hi[i & 3], v[i]);
            } else {
#pragma unroll
              for (int i = 4; i < 32; ++i) lo[i & 3] = fminf(lo[i & 3], v[i]);
            }
            const float top = scale * (scale >= 0.f ? fmaxf(fmaxf(hi[0], hi[1]), fmaxf(hi[2], hi[3]))
                                                    : fminf(fminf(lo[0], lo[1]), fminf(lo[2], lo[3])));
            const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn;
            const uint64_t off = pair(-base, -base);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              sum[i >> 1 & 1] = add2(sum[i >> 1 & 1], ex2_pair(fma2(pair(v[i], v[i + 1]), scale2, off)));
            const float2 s2 = halves(add2(sum[0], sum[1]));
            l = l * ex2(m - base) + (s2.x + s2.y);
            m = mn;
          }
        }
      }
      s_sum[0][g][row] = m;
      s_sum[1][g][row] = l;
      asm volatile("bar.sync %0, %1;" ::"n"(1 + KM_GROUPS), "n"(128 * KM_GROUPS) : "memory");
      if (g == 0 && real) {
#pragma unroll
        for (int i = 1; i < KM_GROUPS; ++i) m = fmaxf(m, s_sum[0][i][row]);
        const float base = m == -INFINITY ? 0.f : m;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < KM_GROUPS; ++i) l += s_sum[1][i][row] * ex2(s_sum[0][i][row] - base);
        a.part[size_t(blockIdx.y) * a.T_total * a.HQ + size_t(w.q0 + tok) * a.HQ + size_t(it.kvh) * a.G + row % a.G] =
            make_float2(m, l);
      }
    } else {
      // the column whose lse this thread finds, a turn ahead, from the key ranges' maxima and sums; a query row with no
      // weight at all (every score -inf) and a column that stands for none get an infinite one: no weight
      const size_t rows = size_t(a.T_total) * a.HQ;
      // the item that the column asked for last belongs to: where it ends, and what a column of it needs
      int ahead = -1, ahead_end = 0, ahead_tok = 0, ahead_T = 0, ahead_first = 0;
      const float2* ahead_part = nullptr;
      auto column = [&](int t, float& lse, int& see) {
        lse = -INFINITY;
        see = -1;
        while (t >= ahead_end) {
          if (++ahead >= items) return;
          const MassItem& it = s_item[ahead];
          ahead_end = it.t0 + it.n;
          ahead_tok = (it.begin - it.t0) * a.tokens + row / a.G;
          ahead_T = row < block_rows ? it.w.T : 0;
          ahead_first = it.w.first;
          ahead_part = a.part + size_t(it.w.q0) * a.HQ + size_t(it.kvh) * a.G + row % a.G;
        }
        const int tok = ahead_tok + t * a.tokens;
        if (tok >= ahead_T) return;
        see = ahead_first + tok;
        const float2* p = ahead_part + size_t(tok) * a.HQ;
        float m = -INFINITY, l = 0.f;
        for (int s0 = 0; s0 < a.splits; s0 += 8) {
          float2 x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = s0 + u < a.splits ? p[(s0 + u) * rows] : make_float2(-INFINITY, 0.f);
          float top = m;
#pragma unroll
          for (int u = 0; u < 8; ++u) top = fmaxf(top, x[u].x);
          const float base = top == -INFINITY ? 0.f : top;
          l *= ex2(m - base);
#pragma unroll
          for (int u = 0; u < 8; ++u) l += x[u].y * ex2(x[u].x - base);
          m = top;
        }
        if (l != 0.f) lse = -((m == -INFINITY ? 0.f : m) + log2f(l));
      };
      float lse;
      int see, t = g;
      column(t, lse, see);
      for (int k = 0; k < items; ++k) {
        const MassItem& it = s_item[k];
        const int key = it.index * KM_TILE + row, end = it.t0 + it.n;
        const int tok_t0 = (it.begin - it.t0) * a.tokens, T = it.w.T;
        const int sees_all = it.index * KM_TILE + KM_TILE - 1 - it.w.first;  // from this token on a query sees the whole tile
        const float scale = it.scale;
        const uint64_t scale2 = pair(scale, scale);
        float total = 0.f;
        for (; t < end; t += KM_GROUPS) {
          const int turn = t / KM_GROUPS & 1;
          s_lse[g][turn][row] = lse;
          s_see[g][turn][row] = see;
          column(t + KM_GROUPS, lse, see);
          asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
          // the block's first token does not see the whole tile, or its last one is behind the window
          const int tok0 = tok_t0 + t * a.tokens;
          const bool masked = tok0 < sees_all || tok0 + a.tokens > T;
          if (!wait_acc(t)) continue;
          uint64_t sum[2] = {0ull, 0ull};
#pragma unroll 1
          for (int c0 = 0; c0 < KM_TILE; c0 += 32) {
            float v[32];
            tmem_ld_x32(quarter + t % KM_ACC * KM_TILE + c0, v);
            if (c0 == KM_TILE - 32) done(t);
            if (masked) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (s_see[g][turn][c0 + i] >= key) total += ex2(fmaf(v[i], scale, s_lse[g][turn][c0 + i]));
            } else {
              if (c0 + 32 > block_rows) {  // the rows of zeros behind the block: their product with an infinite key is NaN
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = c0 + i < block_rows ? v[i] : 0.f;
              }
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(&s_lse[g][turn][c0 + i]);
                sum[0] = add2(sum[0], ex2_pair(fma2(pair(v[i], v[i + 1]), scale2, x.x)));
                sum[1] = add2(sum[1], ex2_pair(fma2(pair(v[i + 2], v[i + 3]), scale2, x.y)));
              }
            }
          }
          const float2 s2 = halves(add2(sum[0], sum[1]));
          total += s2.x + s2.y;
        }
        // the tile is done once all groups are; one of them, by turns, stores it while the others go on
        s_sum[k & 1][g][row] = total;
        asm volatile("bar.sync %0, %1;" ::"n"(1 + KM_GROUPS), "n"(128 * KM_GROUPS) : "memory");
        if (g == k % KM_GROUPS && key < it.sp.ctx && !it.w.refused) {
          total = s_sum[k & 1][0][row];
#pragma unroll
          for (int i = 1; i < KM_GROUPS; ++i) total += s_sum[k & 1][i][row];
          const int e = a.t.page_of(key), page = page_at(a.t, it.sp.first + e);
          if (page >= 0) {
            float* dst = a.key_mass + (size_t(page) * a.t.P + (key - e * a.t.P)) * a.HKV + it.kvh;
            if (a.accumulate) atomicAdd(dst, total);  // a page may be listed by several sequences
            else *dst = total;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, KM_ACC * KM_TILE);
}

// The K rows of every table entry as bf16 [HKV, n_indices P, D]: one-byte formats (E4M3: the codes' values, exact; int8:
// bf16(int8 * scale)), and pages that do not hold whole swizzle atoms.  One CTA per entry.
template <int KVF>
__global__ void __launch_bounds__(256) mass_copy_kernel(const PageTable t, const uint8_t* cache,
                                                        const __nv_bfloat16* row_scale, uint4* out, int HKV, int D) {
  pdl_wait();
  pdl_launch();
  const int e = blockIdx.x;
  bool bad = false;
  const int page = page_or_first(t, e, bad);  // an id that is none is recorded by the pass that meets it in a sequence
  const int cpr = D * (KVF ? 1 : 2) / 16, per_row = HKV * cpr;
  const uint4* src = reinterpret_cast<const uint4*>(cache) + size_t(page) * 2 * t.P * per_row;
  const size_t rows = size_t(t.n_indices) * t.P;
  for (int i = threadIdx.x; i < t.P * per_row; i += 256) {
    const int r = i / per_row, h = i % per_row / cpr, ch = i % cpr;
    const uint4 v = src[i];
    uint4* dst = out + ((size_t(h) * rows + size_t(e) * t.P + r) * D * 2) / 16;
    if constexpr (KVF == 0) {
      dst[ch] = v;
    } else {
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      uint32_t o[8];
      float sc = 0.f;
      if constexpr (KVF == 2) sc = __bfloat162float(row_scale[(size_t(page) * 2 * t.P + r) * HKV + h]);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if constexpr (KVF == 2) {
          o[2 * u] = cvt_s8x2_bf16x2<0, 1>(w[u] ^ 0x80808080u, sc, sc);
          o[2 * u + 1] = cvt_s8x2_bf16x2<2, 3>(w[u] ^ 0x80808080u, sc, sc);
        } else {
          const uint32_t f0 = cvt_kv<0, 1>(w[u]), f1 = cvt_kv<2, 3>(w[u]);
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&f0));
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&f1));
          o[2 * u] = pack_bf16(x.x, x.y);
          o[2 * u + 1] = pack_bf16(y.x, y.y);
        }
      }
      dst[2 * ch] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[2 * ch + 1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

template <int D>
static int launch_mass(const MassArgs& a, const CUtensorMap& qmap, const CUtensorMap& kmap, int64_t blocks, int64_t tiles,
                       cudaStream_t stream) {
  using C = MassCfg<D>;
  Q35_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(mass_kernel<D, false>), C::SMEM));
  Q35_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(mass_kernel<D, true>), C::SMEM));
  if (blocks) {
    launch_pdl(mass_kernel<D, false>, dim3(unsigned(blocks * a.HKV), unsigned(a.splits)), dim3(KM_THREADS), C::SMEM, stream,
               qmap, kmap, a);
    Q35_CUDA_LAUNCH_CHECK("attn.key_mass rows");
  }
  // Short windows: a CTA per SM takes its tiles one after the other, so that what a tile waits for (tables, first loads,
  // the last exponentials) is met while its neighbours work.  Long ones, 32 blocks of queries and more: a CTA per tile, so
  // that the lengths even out (graph replays, four prompts of up to 8192, 2 heads: 32 queries 29.8 us and 37.2, 300
  // queries 118 and 123; 2047 queries 646 and 620).
  int64_t grid = tiles * a.HKV;
  if (grid > sm_count() && blocks <= 32 * int64_t(a.t.B)) {
    const int64_t least = (grid + KM_ITEMS - 1) / KM_ITEMS;
    grid = least > sm_count() ? least : sm_count();
  }
  launch_pdl(mass_kernel<D, true>, dim3(unsigned(grid)), dim3(KM_THREADS), C::SMEM, stream, qmap, kmap, a);
  Q35_CUDA_LAUNCH_CHECK("attn.key_mass columns");
  return 0;
}

int run_attn_key_mass(Call& c) {
  const char* role = "attn.key_mass";
  KvCache kv;
  Q35_TRY(get_kv_cache(c, role, &kv));
  Tensor q, qo, scale, acc, mass, ws;
  Q35_TRY(c.get("q", M(Q35_BF16), &q));
  Q35_TRY(c.get("qo_indptr", M(Q35_I32), &qo));
  Q35_TRY(c.get("sm_scale", M(Q35_F32), &scale, false));
  Q35_TRY(c.get("accumulate", M(Q35_I32), &acc, false));
  Q35_TRY(c.get("key_mass", M(Q35_F32), &mass));
  Q35_REQUIRE(q.nd == 3, Q35_ERR_SHAPE, "%s: q [T, HQ, D]", role);
  const int64_t T = q.s[0], HQ = q.s[1], D = q.s[2], HKV = kv.HKV, P = kv.P, B = qo.numel() - 1;
  Q35_REQUIRE(kv.D == D && HQ >= 1 && HQ % HKV == 0, Q35_ERR_SHAPE, "%s: head shapes", role);
  Q35_REQUIRE(D == 64 || D == 128 || D == 256, Q35_ERR_UNSUPPORTED, "%s: head_dim must be 64/128/256", role);
  const int64_t G = HQ / HKV;
  Q35_REQUIRE(G <= KM_TILE, Q35_ERR_UNSUPPORTED, "%s: at most 128 query heads per KV head (got %lld)", role, (long long)G);
  Q35_REQUIRE(B >= 0 && mass.numel() == kv.pages * P * HKV, Q35_ERR_SHAPE, "%s: qo_indptr [B + 1], key_mass [pages, P, HKV]",
              role);
  Q35_REQUIRE(!scale.present || scale.numel() == 1, Q35_ERR_SHAPE, "%s: sm_scale [1]", role);
  MassArgs a{};
  Q35_TRY(get_page_table(c, role, B, P, kv.pages, &a.t));
  const int64_t entries = a.t.n_indices, tokens = KM_TILE / G;
  // bounds on the items: sequences add a partial one each
  const int64_t blocks = T ? T / tokens + B : 0, tiles = entries * P / KM_TILE + B;
  Q35_REQUIRE(T * HQ <= INT_MAX / 2 && B <= INT_MAX / 4 && blocks * HKV <= INT_MAX && tiles * HKV <= INT_MAX,
              Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  // rows per TMA box of keys: the largest power of two that divides a page, whole 8-row swizzle atoms
  int64_t box = KM_TILE;
  while (P % box) box /= 2;
  const bool copied = kv.fmt != 0 || box < 8 || kv.pages * 2 * P > INT_MAX;
  if (copied) box = KM_TILE;
  Q35_REQUIRE(!copied || HKV * entries * P <= INT_MAX, Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  // pass 1 gets about two CTAs per SM from ranges of keys, of at least four tiles each
  const int64_t items = blocks * HKV, per_seq = B ? tiles / B : 0;
  int64_t splits = items ? (2 * sm_count() + items - 1) / items : 1;
  if (splits > per_seq / 4) splits = per_seq / 4;
  if (splits < 1) splits = 1;
  if (splits > 32) splits = 32;
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = (off + bytes + 255) / 256 * 256; return o; };
  const int64_t o_part = take(splits * T * HQ * 8), o_copy = take(copied ? HKV * entries * P * D * 2 : 0);
  Q35_TRY(c.workspace(off, &ws));
  if (c.dry || B == 0) return 0;
  Q35_REQUIRE(aligned16(q.p), Q35_ERR_ALIGN, "%s: q must be 16-byte aligned", role);
  if (entries == 0) return 0;  // no sequence has a row
  a.qo_indptr = qo.as<int>();
  a.kv_scale = kv.kv_scale; a.e4m3 = kv.fmt == 1;
  a.sm_scale = scale.present ? scale.as<float>() : nullptr;
  a.key_mass = mass.as<float>();
  uint8_t* w = ws.as<uint8_t>();
  a.part = reinterpret_cast<float2*>(w + o_part);
  a.T_total = int(T); a.HQ = int(HQ); a.HKV = int(HKV); a.G = int(G); a.D = int(D);
  a.splits = int(splits); a.accumulate = acc.present; a.tokens = int(tokens); a.box_rows = int(box); a.copied = copied;
  CUtensorMap qmap, kmap;
  if (copied) {
    uint4* out = reinterpret_cast<uint4*>(w + o_copy);
    const uint8_t* cache = static_cast<const uint8_t*>(kv.p);
    const dim3 grid{unsigned(entries)};
    if (kv.fmt == 0)
      launch_pdl(mass_copy_kernel<0>, grid, dim3(256), 0, c.stream, a.t, cache, kv.row_scale, out, int(HKV), int(D));
    else if (kv.fmt == 1)
      launch_pdl(mass_copy_kernel<1>, grid, dim3(256), 0, c.stream, a.t, cache, kv.row_scale, out, int(HKV), int(D));
    else
      launch_pdl(mass_copy_kernel<2>, grid, dim3(256), 0, c.stream, a.t, cache, kv.row_scale, out, int(HKV), int(D));
    Q35_CUDA_LAUNCH_CHECK("attn.key_mass copy");
    const uint64_t dims[2] = {uint64_t(D), uint64_t(HKV * entries * P)}, strides[1] = {uint64_t(D * 2)};
    const uint32_t bx[2] = {64, KM_TILE};
    Q35_TRY(tc_encode_bf16(&kmap, 2, out, dims, strides, bx, "K rows"));
  } else {
    const uint64_t dims[2] = {uint64_t(HKV * D), uint64_t(kv.pages * 2 * P)}, strides[1] = {uint64_t(HKV * D * 2)};
    const uint32_t bx[2] = {64, uint32_t(box)};
    Q35_TRY(tc_encode_bf16(&kmap, 2, kv.p, dims, strides, bx, "paged_kv_cache"));
  }
  if (T) {
    const uint64_t dims[3] = {uint64_t(D), uint64_t(HQ), uint64_t(T)}, strides[2] = {uint64_t(D * 2), uint64_t(HQ * D * 2)};
    const uint32_t bx[3] = {64, uint32_t(G), uint32_t(tokens)};
    Q35_TRY(tc_encode_bf16(&qmap, 3, q.p, dims, strides, bx, "q"));
  } else {
    qmap = kmap;  // not read
  }
  if (D == 64) return launch_mass<64>(a, qmap, kmap, blocks, tiles, c.stream);
  if (D == 128) return launch_mass<128>(a, qmap, kmap, blocks, tiles, c.stream);
  return launch_mass<256>(a, qmap, kmap, blocks, tiles, c.stream);
}

}  // namespace q35
