// attn.sparse_decode: one query token per sequence over chosen pages of its cache (or all of them), optionally adding
// the softmax weight that every cached row receives to key_mass.
//
// With s_gi = q_g . k_i * scale over the rows i of the chosen pages, M_g = max_i s_gi, L_g = sum_i exp(s_gi - M_g):
//   out_g = sum_i exp(s_gi - M_g) v_i / L_g,     key_mass_i += sum_g exp(s_gi - M_g) / L_g   (g over the group's heads).
//
// Bound: HBM, K and V of the chosen rows once.  A cluster of C CTAs serves one (sequence, KV head): its chosen rows,
// laid end to end, are cut into C contiguous ranges, every CTA runs one pass with a running maximum and sum over its
// range, and the C partial results are merged through distributed shared memory -- one launch, no partials in HBM, no
// counters.  (All pages of many long rows: the flat form, equal shares per CTA and a second kernel that merges.)  Inside a
// CTA each warp takes steps of 32 rows through its own cp.async ring (16-byte chunks, XOR-swizzled rows), with no block
// barrier in the loop.  Scores are computed transposed (S^T = K Q^T, mma.m16n8k16) so that the up to 8 query heads of a KV
// head are the n = 8 side and O^T takes D / 4 registers a lane.  (Times here are graph replays, but for those of weights
// and sums, which are calls among others.)
//
// The weights need the final M and L, so each CTA parks its scores (fp32, 32 bytes per row against 4 D of K and V) in
// the workspace and turns them into weights after the merge; a row's weights are added by the one CTA that read it.
#include <cooperative_groups.h>
#include "abi.h"
#include "attn_pages.cuh"
#include "kv_formats.cuh"

namespace q35 {

namespace cg = cooperative_groups;

constexpr int SP_G = 8;          // query heads per KV head handled by one mma column block
constexpr int SP_SUB = 16;       // rows of one MMA tile; a page holds whole tiles
constexpr int SP_KEYS = 32;      // rows per warp and step
constexpr float SP_LOG2E = 1.4426950408889634f;

struct SparseArgs {
  PageTable t;
  const __nv_bfloat16* q;          // [B, HQ, D]
  const uint8_t* cache;            // [pages, 2, P, HKV, D]
  const float* kv_scale;
  const __nv_bfloat16* row_scale;
  const int* pages;                // optional [B, HKV, S]
  const float* sm_scale;           // optional [1]
  const __nv_bfloat16* k_new;      // optional [B, HKV, D]: the current token's own rows
  const __nv_bfloat16* v_new;
  const int* new_at;               // [B, 2] (page, offset) of the current token, with key_mass and k_new
  __nv_bfloat16* out;              // [B, HQ, D]
  float* key_mass;                 // optional [pages, P, HKV]
  float* scores;                   // workspace, with key_mass: 8 floats per row
  float* part_o; float* part_ml;   // workspace of the flat form: [rows + n_cta][8][D], [rows + n_cta][16]
  int HQ, HKV, G, S;
  int n_cta, chunks;               // flat form: CTAs of the first kernel, CTAs per (sequence, KV head) of the second
};

// KVF: 0 bf16, 1 E4M3, 2 int8 rows with scales.
// A warp's step is 32 rows: K, then V, each a slot of its ring of three, so that 64 rows' worth of bytes are on their way
// while one slot is in use.  32 rows (two MMA tiles) share one round of shuffles, exponentials' latency and rescaling;
// 16-row steps took 5-25 % longer.  Four warps: 192 KB of ring and one CTA per SM with 512-byte rows, two or more with
// narrower ones; eight warps per CTA were slower wherever lengths differ.
template <int D, int KVF>
struct SparseCfg {
  static constexpr bool BYTE = KVF != 0;
  static constexpr int WARPS = 4;
  static constexpr int TERMS = KVF == 1 ? 2 : 3;        // 16-bit numbers that make up a weight in the P V product
  static constexpr int SLOTS = 3;                       // half steps (32 rows of K or of V) per warp
  static constexpr int ROWB = D * (BYTE ? 1 : 2);
  static constexpr int CPR = ROWB / 16;                 // 16-byte chunks per row
  static constexpr int SWZ = (CPR < 8 ? CPR : 8) - 1;   // rows narrower than 128 bytes permute fewer chunks
  static constexpr int SLOT_BYTES = SP_KEYS * ROWB;
  static constexpr int RING = WARPS * SLOTS * SLOT_BYTES;
  static constexpr int PART = WARPS * SP_G * D * 4;     // the warps' output partials reuse the ring
  static constexpr int SMEM = RING > PART ? RING : PART;
  static constexpr int LD = SP_KEYS * CPR / 32;         // chunks per lane and half step
  // CTAs per SM: as the ring and the accumulators' registers (up to 255, 170, 128 a thread) allow
  static constexpr int CTAS = D == 256 ? (BYTE ? 2 : 1) : D == 128 ? (BYTE ? 3 : 2) : 4;
};

// key_mass += weights of the rows k_begin .. k_end - 1 of a (sequence, KV head), from their scores and the heads' final
// maxima and inverse sums; `lifted`: how many times the sums are larger than what a score stands for.
template <int THREADS>
__device__ __forceinline__ void add_weights(const SparseArgs& a, const SeqPages& sp, const int* pages, int kvh,
                                            const float* scores, int k_begin, int k_end, const float* s_top,
                                            const float* s_inv, float lifted) {
  // Four rows of every thread on their way together, no branch between them: rows behind the end read the last row's
  // scores and add nothing.  (One or two warps per scheduler: what counts here is the number of instructions per row.)
  constexpr int U = 4;
  float top[SP_G], inv[SP_G];
#pragma unroll
  for (int g = 0; g < SP_G; ++g) {
    top[g] = s_top[g];
    inv[g] = g < a.G ? s_inv[g] * lifted : 0.f;
  }
  for (int k0 = k_begin + int(threadIdx.x); k0 < k_end; k0 += U * THREADS) {
    float4 lo[U], hi[U];
    int page[U], off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(k0 + u * THREADS, k_end - 1), e = a.t.page_of(k);
      lo[u] = *reinterpret_cast<const float4*>(scores + size_t(k) * SP_G);
      hi[u] = *reinterpret_cast<const float4*>(scores + size_t(k) * SP_G + 4);
      page[u] = a.t.indices[sp.first + (pages ? pages[e] : e)];  // no page: recorded by the step that read the row
      off[u] = k - e * a.t.P;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float s[8] = {lo[u].x, lo[u].y, lo[u].z, lo[u].w, hi[u].x, hi[u].y, hi[u].z, hi[u].w};
      float w = 0.f;
#pragma unroll
      for (int g = 0; g < SP_G; ++g) w += inv[g] == 0.f ? 0.f : ex2(s[g] - top[g]) * inv[g];
      if (k0 + u * THREADS < k_end && unsigned(page[u]) < unsigned(a.t.num_pages))
        atomicAdd(a.key_mass + (size_t(page[u]) * a.t.P + off[u]) * a.HKV + kvh, w);
    }
  }
}
// the current token's own weight, stored where its row is
__device__ __forceinline__ void add_new_weight(const SparseArgs& a, int b, int kvh, const float* s_new, const float* s_top,
                                               const float* s_inv, float lifted) {
  float w = 0.f;
  for (int g = 0; g < a.G; ++g) w += ex2(s_new[g] - s_top[g]) * s_inv[g];
  const int page = a.new_at[2 * b], off = a.new_at[2 * b + 1];
  if (unsigned(page) < unsigned(a.t.num_pages) && unsigned(off) < unsigned(a.t.P))
    a.key_mass[(size_t(page) * a.t.P + off) * a.HKV + kvh] = w * lifted;
  else
    atomicOr(a.t.status, DS_BAD_PAGE);
}

// The flat form's split: all steps of all (sequence, KV head) rows end to end, `per` of them to a CTA.  Whole warp.
__device__ __forceinline__ int flat_steps(const SparseArgs& a, int b) {
  return (seq_pages(a.t, b).ctx + SP_KEYS - 1) / SP_KEYS;
}
__device__ __forceinline__ int flat_per_cta(const SparseArgs& a) {
  int total = 0;
  for (int b = threadIdx.x & 31; b < a.t.B; b += 32) total += flat_steps(a, b);
  total = __reduce_add_sync(0xffffffffu, total) * a.HKV;
  return max(1, (total + a.n_cta - 1) / a.n_cta);
}

template <int D, int KVF, bool FLAT>
__global__ void __launch_bounds__(32 * SparseCfg<D, KVF>::WARPS, SparseCfg<D, KVF>::CTAS) sparse_decode_kernel(const SparseArgs a) {
  using C = SparseCfg<D, KVF>;
  constexpr int WARPS = C::WARPS, THREADS = 32 * WARPS, TERMS = C::TERMS;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_part[SP_G * D];                        // this CTA's merged output, read by the cluster
  __shared__ float s_ml[2 * SP_G];                          // its maxima and sums, read by the cluster
  __shared__ float s_wml[WARPS][2 * SP_G];
  __shared__ float s_fac[16][SP_G], s_fin[2 * SP_G], s_new[SP_G];
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  // the row of the grid that this CTA works on; in the flat form the first of them, and how many steps to do in all
  int b, kvh, from = 0, todo = 0;
  cg::cluster_group cluster = cg::this_cluster();
  const int NC = FLAT ? 1 : int(cluster.num_blocks()), rank = FLAT ? 0 : int(cluster.block_rank());
  if constexpr (FLAT) {
    __shared__ int s_flat[3];
    if (warp == 0) {
      const int per = flat_per_cta(a);
      const int2 it = find_item(a.t.B, int(blockIdx.x) * per, [&](int i) { return flat_steps(a, i) * a.HKV; });
      if (lane == 0) { s_flat[0] = per; s_flat[1] = it.x; s_flat[2] = it.y; }
    }
    __syncthreads();
    todo = s_flat[0];
    b = s_flat[1];
    if (b < 0) return;  // more CTAs than steps
    const int steps = flat_steps(a, b);
    kvh = s_flat[2] / steps;
    from = s_flat[2] % steps;
  } else {
    b = int(blockIdx.x) / NC / a.HKV;
    kvh = int(blockIdx.x) / NC % a.HKV;
  }
  for (;;) {  // the flat form goes around once per row that it touches
  const int row = b * a.HKV + kvh;
  const float scale_log2 = (a.sm_scale ? a.sm_scale[0] : rsqrtf(float(D))) * SP_LOG2E;
  // query fragments (B operand, heads on the n side).  bf16 / int8 cache: bf16 (int8: in the k order the byte-wise
  // fragments come out in).  E4M3: f16, after scaling each head by the power of two that brings its largest element to
  // [2^14, 2^15): exact but for elements 2^-28 times smaller, which lose bits below 2^-39 of the largest.
  uint32_t qf[D / 16][2];
  float col_scale[2] = {scale_log2, scale_log2};  // of the heads 2 c and 2 c + 1
  float v_mul = 1.f;
  {
    const __nv_bfloat16* qp = a.q + (size_t(b) * a.HQ + size_t(kvh) * a.G + r) * D;
    const bool hv = r < a.G;
    if constexpr (!C::BYTE) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][0] = hv ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + 2 * c) : 0u;
        qf[ks][1] = hv ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + 8 + 2 * c) : 0u;
      }
    } else {
      float amax = 0.f;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint2 raw = make_uint2(0u, 0u);
        if (hv) raw = *reinterpret_cast<const uint2*>(qp + ks * 16 + 4 * c);
        qf[ks][0] = raw.x;
        qf[ks][1] = raw.y;
        amax = fmaxf(amax, fmaxf(fmaxf(fabsf(bf16lo(raw.x)), fabsf(bf16hi(raw.x))),
                                 fmaxf(fabsf(bf16lo(raw.y)), fabsf(bf16hi(raw.y)))));
      }
      if constexpr (KVF == 1) {
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int ex = amax > 0.f && amax < INFINITY ? int(__float_as_uint(amax) >> 23) - 127 : 14;
        const int up = min(14 - ex, 126);
        const float mul = __uint_as_float(uint32_t(up + 127) << 23), back = __uint_as_float(uint32_t(127 - up) << 23);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          qf[ks][0] = pack_f16(bf16lo(qf[ks][0]) * mul, bf16hi(qf[ks][0]) * mul);
          qf[ks][1] = pack_f16(bf16lo(qf[ks][1]) * mul, bf16hi(qf[ks][1]) * mul);
        }
        const float k_mul = a.kv_scale ? a.kv_scale[kvh] : 0.125f;
        v_mul = a.kv_scale ? a.kv_scale[a.HKV + kvh] : 0.125f;
        col_scale[0] *= k_mul * __shfl_sync(0xffffffffu, back, 8 * c);
        col_scale[1] *= k_mul * __shfl_sync(0xffffffffu, back, 8 * c + 4);
      }
    }
  }

  const SeqPages sp = seq_pages(a.t, b);
  const int P = a.t.P;

  // the chosen pages: ascending positions in the sequence's page list; the list ends at the first entry that is not.
  // Every warp reads the whole list for itself: no barrier before the first row can be asked for.
  const int* pages = a.pages ? a.pages + size_t(row) * a.S : nullptr;
  int n_sel = sp.n, n_keys = sp.ctx;
  if (pages) {
    int before = -1;
    n_sel = a.S;
    for (int i0 = 0; i0 < a.S; i0 += 32) {
      const int p = i0 + lane < a.S ? pages[i0 + lane] : -1;
      const int left = __shfl_up_sync(0xffffffffu, p, 1);
      const int prev = lane ? left : before;
      const unsigned end = __ballot_sync(0xffffffffu, p < 0 || p >= sp.n || p <= prev);
      const int cut = end ? __ffs(end) - 1 : 32;
      before = __shfl_sync(0xffffffffu, p, cut ? cut - 1 : 0);
      if (!end) continue;
      if (lane == cut && p != -1) atomicOr(a.t.status, DS_BAD_PAGE);  // not the end of the list, but no page
      n_sel = min(a.S, i0 + cut);
      if (!cut && i0) before = pages[i0 - 1];
      break;
    }
    n_keys = n_sel * P;
    if (n_sel > 0 && before == sp.n - 1) n_keys += sp.ctx - sp.n * P;  // the last page may be part full
  }

  // steps of 32 rows: this CTA's contiguous range, dealt to its warps in turn
  const int steps = (n_keys + SP_KEYS - 1) / SP_KEYS, per = (steps + NC - 1) / NC;
  const int s_begin = FLAT ? from : min(steps, rank * per), s_end = min(steps, s_begin + (FLAT ? todo : per));
  const size_t row_stride = size_t(a.HKV) * C::ROWB;  // bytes between consecutive rows of a page plane
  // scores of this (sequence, KV head): behind S * P rows of every row of the grid, or behind the table entries before
  float* scores = a.scores;
  if (scores)
    scores += (pages ? size_t(row) * a.S : size_t(a.HKV) * sp.first + size_t(kvh) * sp.n) * size_t(P) * SP_G;

  // Where the warp's next 32 tiles of 16 rows lie, one lane each: tile u of the warp is half u & 1 of its step u / 2.
  // Looked up 32 at a time, a round ahead, so that no step waits for the page table or divides by P.
  const int first_step = s_begin + warp, my_steps = first_step < s_end ? (s_end - first_step + WARPS - 1) / WARPS : 0;
  auto tile_row = [&](int u) { return (first_step + (u >> 1) * WARPS) * SP_KEYS + (u & 1) * SP_SUB; };
  auto entry_of = [&](int u) -> int {  // position in the page list of the sequence, -1 behind the end
    const int k = tile_row(u);
    return u < 2 * my_steps && k < n_keys ? (pages ? pages[a.t.page_of(k)] : a.t.page_of(k)) : -1;
  };
  int page_cur, row_cur, entry_next;  // page and row in it of tile (round * 32 + lane); entry of the next round's
  auto look_up = [&](int u0, int entry) {
    const int id = entry >= 0 ? page_at(a.t, sp.first + entry) : 0;
    page_cur = id < 0 ? 0 : id;
    const int k = tile_row(u0 + lane);
    row_cur = entry >= 0 ? k - a.t.page_of(k) * P : 0;
  };
  look_up(0, entry_of(lane));
  entry_next = entry_of(32 + lane);

  const uint32_t sbase = smem_u32(smem) + warp * (C::SLOTS * C::SLOT_BYTES);
  // 32 rows of K (kv 0) or V (kv 1) of the warp's step i into slot (2 i + kv) % 3
  auto issue = [&](int i, int kv, int slot) {
    if (i < my_steps) {
      const int left = n_keys - (first_step + i * WARPS) * SP_KEYS;
      const uint32_t st = sbase + slot * C::SLOT_BYTES;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int src = (2 * i + half) & 31;
        const int page = __shfl_sync(0xffffffffu, page_cur, src), ro = __shfl_sync(0xffffffffu, row_cur, src);
        const uint8_t* base = a.cache + ((size_t(page) * 2 + kv) * P + ro) * row_stride + size_t(kvh) * C::ROWB;
#pragma unroll
        for (int j = 0; j < C::LD / 2; ++j) {
          const int ci = lane + 32 * j, key = ci / C::CPR, ch = ci % C::CPR, at_key = half * SP_SUB + key;
          const uint32_t at = st + at_key * C::ROWB + ((ch ^ (key & C::SWZ)) << 4);
          if (at_key < left)
            cp_async_16(at, base + size_t(key) * row_stride + ch * 16);
          else if (kv == 1)  // rows behind the end are never read: zeros keep 0 * V a zero
            asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0u));
        }
      }
    }
    cp_async_commit();
  };
  // int8: the row scales of a step, lane l holding K (low half) and V of row l; 0 behind the end
  auto load_scales = [&](int i) -> uint32_t {
    uint32_t v = 0u;
    if constexpr (KVF == 2) {
      const int src = (2 * i + (lane >> 4)) & 31;
      const int page = __shfl_sync(0xffffffffu, page_cur, src), ro = __shfl_sync(0xffffffffu, row_cur, src);
      if (i < my_steps && (first_step + i * WARPS) * SP_KEYS + lane < n_keys) {
        const unsigned short* sp16 = reinterpret_cast<const unsigned short*>(a.row_scale) +
                                     (size_t(page) * 2 * P + ro + (lane & 15)) * a.HKV + kvh;
        v = uint32_t(sp16[0]) | uint32_t(sp16[size_t(P) * a.HKV]) << 16;
      }
    }
    return v;
  };

  float oacc[D / 16][4];
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) oacc[mt][0] = oacc[mt][1] = oacc[mt][2] = oacc[mt][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  // half steps in flight: while K of step i is in use, V of step i and K of step i + 1 are on their way, then V of both
  issue(0, 0, 0);
  issue(0, 1, 1);
  uint32_t rs_next = load_scales(0);
  int slot = 0;  // of the half step in use
  for (int i = 0; i < my_steps; ++i) {
    const uint32_t rs = rs_next;
    if (((i + 1) & 15) == 0) {  // the next step is the first of another round of 32 tiles
      look_up(2 * (i + 1), entry_next);
      entry_next = entry_of(2 * (i + 1) + 32 + lane);
    }
    issue(i + 1, 0, slot == 0 ? 2 : slot - 1);
    rs_next = load_scales(i + 1);
    cp_async_wait<2>();
    __syncwarp();
    const int step = first_step + i * WARPS, left = n_keys - step * SP_KEYS;
    uint32_t st = sbase + slot * C::SLOT_BYTES;
    float sacc[2][2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int u = 0; u < 4; ++u) sacc[h][0][u] = sacc[h][1][u] = 0.f;
    {
      const int key = (lane & 7) + (((lane >> 3) & 1) << 3);
      const uint32_t rowa = st + key * C::ROWB;
      if constexpr (!C::BYTE) {
#pragma unroll
        for (int k0 = 0; k0 < D / 16; k0 += 2) {
          uint32_t f[2][2][4];
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int ch = 2 * (k0 + k) + (lane >> 4);
              ldmatrix_x4(rowa + h * SP_SUB * C::ROWB + ((ch ^ (key & C::SWZ)) << 4), f[k][h][0], f[k][h][1], f[k][h][2],
                          f[k][h][3]);
            }
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              mma_bf16_16816(sacc[h][k], f[k][h][0], f[k][h][1], f[k][h][2], f[k][h][3], qf[k0 + k][0], qf[k0 + k][1]);
        }
      } else {
        float ks[2][2];  // int8: scales of the rows r and r + 8 of both tiles
        if constexpr (KVF == 2) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int u = 0; u < 2; ++u) ks[h][u] = bf16lo(__shfl_sync(0xffffffffu, rs, h * 16 + u * 8 + r));
        }
#pragma unroll
        for (int kp = 0; kp < D / 32; ++kp) {  // 32 channels: two mma over bytes taken as b16 pairs
          const int ch = 2 * kp + (lane >> 4);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r0, r1, r2, r3;
            ldmatrix_x4(rowa + h * SP_SUB * C::ROWB + ((ch ^ (key & C::SWZ)) << 4), r0, r1, r2, r3);
            if constexpr (KVF == 2) {
              const float s0 = ks[h][0], s1 = ks[h][1];
              r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
              mma_bf16_16816(sacc[h][0], cvt_s8x2_bf16x2<0, 1>(r0, s0, s0), cvt_s8x2_bf16x2<0, 1>(r1, s1, s1),
                             cvt_s8x2_bf16x2<2, 3>(r0, s0, s0), cvt_s8x2_bf16x2<2, 3>(r1, s1, s1), qf[2 * kp][0],
                             qf[2 * kp][1]);
              mma_bf16_16816(sacc[h][1], cvt_s8x2_bf16x2<0, 1>(r2, s0, s0), cvt_s8x2_bf16x2<0, 1>(r3, s1, s1),
                             cvt_s8x2_bf16x2<2, 3>(r2, s0, s0), cvt_s8x2_bf16x2<2, 3>(r3, s1, s1), qf[2 * kp + 1][0],
                             qf[2 * kp + 1][1]);
            } else {
              mma_f16_16816(sacc[h][0], cvt_kv<0, 1>(r0), cvt_kv<0, 1>(r1), cvt_kv<2, 3>(r0), cvt_kv<2, 3>(r1),
                            qf[2 * kp][0], qf[2 * kp][1]);
              mma_f16_16816(sacc[h][1], cvt_kv<0, 1>(r2), cvt_kv<0, 1>(r3), cvt_kv<2, 3>(r2), cvt_kv<2, 3>(r3),
                            qf[2 * kp + 1][0], qf[2 * kp + 1][1]);
            }
          }
        }
      }
    }
    __syncwarp();  // K's slot is free
    issue(i + 1, 1, slot);
    slot = slot == 2 ? 0 : slot + 1;
    st = sbase + slot * C::SLOT_BYTES;
    float sc[2][4];  // rows r, r, r + 8, r + 8 of both tiles; heads 2 c, 2 c + 1
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        sc[h][u] = h * SP_SUB + r + ((u >> 1) << 3) < left ? (sacc[h][0][u] + sacc[h][1][u]) * col_scale[u & 1] : -INFINITY;
      if (scores) {
        float* at = scores + (size_t(step) * SP_KEYS + h * SP_SUB + r) * SP_G + 2 * c;
        if (h * SP_SUB + r < left) *reinterpret_cast<float2*>(at) = make_float2(sc[h][0], sc[h][1]);
        if (h * SP_SUB + r + 8 < left) *reinterpret_cast<float2*>(at + 8 * SP_G) = make_float2(sc[h][2], sc[h][3]);
      }
    }
    float top[2] = {fmaxf(fmaxf(sc[0][0], sc[0][2]), fmaxf(sc[1][0], sc[1][2])),
                    fmaxf(fmaxf(sc[0][1], sc[0][3]), fmaxf(sc[1][1], sc[1][3]))};
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
    }
    // E4M3: weights 2^8 times larger, up to 256, so that f16 resolves 2^-32 of the largest
    constexpr float LIFT = KVF == 1 ? 8.f : 0.f;
    float alpha[2], ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mn = fmaxf(m_run[h], top[h]);
      const float base = mn == -INFINITY ? 0.f : mn;  // no row with a weight yet
      alpha[h] = ex2(m_run[h] - base);
      m_run[h] = mn;
      ref[h] = base - LIFT;
    }
    // The weights meet V whole: p as three bf16 terms (24 bits) beside bf16 and int8 rows, as two f16 terms (22 bits) beside
    // E4M3 ones.  (One f16 term rounded 4.8 % of the bf16 outputs the other way than the exact sum does, two 0.04 %, for
    // 51.8 -> 53.4 us with 32 sequences of up to 4161 rows; two bf16 terms against three: 88.0 and 91.4 us for 64 x 4096 rows.)
    uint32_t pb[TERMS][2][2];
    l_run[0] *= alpha[0];
    l_run[1] *= alpha[1];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {  // rows r, then r + 8
        const float p0 = ex2(sc[h][2 * u] - ref[0]), p1 = ex2(sc[h][2 * u + 1] - ref[1]);
        l_run[0] += p0;
        l_run[1] += p1;
        float left0 = p0, left1 = p1;  // of the weights, behind the terms so far
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          const uint32_t w = KVF == 1 ? pack_f16(left0, left1) : pack_bf16(left0, left1);
          pb[t][h][u] = movmatrix_trans(w);
          if constexpr (KVF == 1) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
            left0 -= f.x;
            left1 -= f.y;
          } else {
            left0 -= bf16lo(w);
            left1 -= bf16hi(w);
          }
        }
      }
    }
    // A step's products are summed from zero and added here, rounded to nearest: the tensor cores cut off what an
    // accumulator cannot hold, always towards zero, which over thousands of rows is a loss of its own (0.2 % of the outputs
    // of 64 x 4096 rows rounded the other way than the exact sum, 0.04 % so; the plain form in fp32 0.09 %).
    auto add_step = [&](float (&o)[4], const float (&x)[4]) {
#pragma unroll
      for (int u = 0; u < 4; ++u) o[u] = fmaf(o[u], alpha[u & 1], x[u]);
    };
    cp_async_wait<2>();
    __syncwarp();
    if constexpr (!C::BYTE) {
      const int key = (lane & 7) + ((lane >> 4) << 3);
      const uint32_t rowa = st + key * C::ROWB;
      // output tiles whose products go on together: dependent ones lie MB apart (4: 97 us for 64 x 4096 rows, 8: 92)
      constexpr int MB = D / 16 < 8 ? D / 16 : 8;
#pragma unroll
      for (int m0 = 0; m0 < D / 16; m0 += MB) {
        float acc[MB][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t f[MB][4];
#pragma unroll
          for (int m = 0; m < MB; ++m) {
            const int ch = 2 * (m0 + m) + ((lane >> 3) & 1);
            ldmatrix_x4_trans(rowa + h * SP_SUB * C::ROWB + ((ch ^ (key & C::SWZ)) << 4), f[m][0], f[m][1], f[m][2], f[m][3]);
          }
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int m = 0; m < MB; ++m)
              mma_bf16_16816(acc[m], f[m][0], f[m][1], f[m][2], f[m][3], pb[t][h][0], pb[t][h][1]);
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) add_step(oacc[m0 + m], acc[m]);
      }
    } else {
      // transposed b16 loads keep byte pairs (d, d + 1) together: bytes (0, 2) / (1, 3) are the row pairs of channels
      // 2 r / 2 r + 1, so mma row r holds channel 16 mt + 2 r and mma row r + 8 channel 16 mt + 2 r + 1
      float vs[2][4];  // int8: scales of the rows 2 c, 2 c + 1, 2 c + 8, 2 c + 9 of both tiles
      if constexpr (KVF == 2) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int u = 0; u < 4; ++u)
            vs[h][u] = bf16hi(__shfl_sync(0xffffffffu, rs, h * 16 + 2 * c + (u & 1) + ((u >> 1) << 3)));
      }
      const int key = lane & 15;
      const uint32_t rowa = st + key * C::ROWB;
      // 32-channel pieces whose products go on together (1: 55.2 us for 32 sequences of up to 4161 E4M3 rows, 4: 54.3)
      constexpr int MB = D / 32 < 4 ? D / 32 : 4;
#pragma unroll
      for (int m0 = 0; m0 < D / 32; m0 += MB) {
        float acc[2 * MB][4] = {};
#pragma unroll
        for (int i = 0; i < 2 * MB; ++i) {
          const int h = i / MB, m = i % MB, ch = 2 * (m0 + m) + (lane >> 4);
          uint32_t r0, r1, r2, r3;  // (rows 0-7, chunk ch) (rows 8-15, ch) (rows 0-7, ch + 1) (rows 8-15, ch + 1), ch even
          ldmatrix_x4_trans(rowa + h * SP_SUB * C::ROWB + ((ch ^ (key & C::SWZ)) << 4), r0, r1, r2, r3);
          uint32_t x[8];
          if constexpr (KVF == 2) {
            const float va = vs[h][0], vb = vs[h][1], vc = vs[h][2], vd = vs[h][3];
            r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
            x[0] = cvt_s8x2_bf16x2<0, 2>(r0, va, vb); x[1] = cvt_s8x2_bf16x2<1, 3>(r0, va, vb);
            x[2] = cvt_s8x2_bf16x2<0, 2>(r1, vc, vd); x[3] = cvt_s8x2_bf16x2<1, 3>(r1, vc, vd);
            x[4] = cvt_s8x2_bf16x2<0, 2>(r2, va, vb); x[5] = cvt_s8x2_bf16x2<1, 3>(r2, va, vb);
            x[6] = cvt_s8x2_bf16x2<0, 2>(r3, vc, vd); x[7] = cvt_s8x2_bf16x2<1, 3>(r3, vc, vd);
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
              mma_bf16_16816(acc[2 * m], x[0], x[1], x[2], x[3], pb[t][h][0], pb[t][h][1]);
              mma_bf16_16816(acc[2 * m + 1], x[4], x[5], x[6], x[7], pb[t][h][0], pb[t][h][1]);
            }
          } else {
            x[0] = cvt_kv<0, 2>(r0); x[1] = cvt_kv<1, 3>(r0); x[2] = cvt_kv<0, 2>(r1); x[3] = cvt_kv<1, 3>(r1);
            x[4] = cvt_kv<0, 2>(r2); x[5] = cvt_kv<1, 3>(r2); x[6] = cvt_kv<0, 2>(r3); x[7] = cvt_kv<1, 3>(r3);
#pragma unroll
            for (int t = 0; t < TERMS; ++t) {
              mma_f16_16816(acc[2 * m], x[0], x[1], x[2], x[3], pb[t][h][0], pb[t][h][1]);
              mma_f16_16816(acc[2 * m + 1], x[4], x[5], x[6], x[7], pb[t][h][0], pb[t][h][1]);
            }
          }
        }
#pragma unroll
        for (int m = 0; m < 2 * MB; ++m) add_step(oacc[2 * m0 + m], acc[m]);
      }
    }
    __syncwarp();  // V's slot is free
    slot = slot == 2 ? 0 : slot + 1;
  }
  cp_async_wait<0>();
  __syncthreads();  // the ring is free: the warps' partials go there

  float* s_wo = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], o);
    l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], o);
  }
  if (r == 0) {
    s_wml[warp][2 * c] = m_run[0]; s_wml[warp][2 * c + 1] = m_run[1];
    s_wml[warp][SP_G + 2 * c] = l_run[0]; s_wml[warp][SP_G + 2 * c + 1] = l_run[1];
  }
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) {
    const int d0 = C::BYTE ? mt * 16 + 2 * r : mt * 16 + r, d1 = C::BYTE ? d0 + 1 : d0 + 8;
    float* o0 = s_wo + (warp * SP_G + 2 * c) * D;
    o0[d0] = oacc[mt][0] * v_mul; o0[D + d0] = oacc[mt][1] * v_mul;
    o0[d1] = oacc[mt][2] * v_mul; o0[D + d1] = oacc[mt][3] * v_mul;
  }
  // the current token, taken from its own rows: one more partial (l = 1, o = v), merged by the cluster's first CTA
  const bool has_new = !FLAT && a.k_new != nullptr && rank == 0;  // (flat: in the second kernel)
  if (has_new) {
    const __nv_bfloat16* kp = a.k_new + size_t(row) * D;
    for (int g = warp; g < SP_G; g += WARPS) {
      float dot = 0.f;
      if (g < a.G) {
        const __nv_bfloat16* qp = a.q + (size_t(b) * a.HQ + size_t(kvh) * a.G + g) * D;
        for (int d = lane; d < D; d += 32) dot += __bfloat162float(qp[d]) * __bfloat162float(kp[d]);
      }
      dot = warp_sum(dot);
      if (lane == 0) s_new[g] = dot * scale_log2;
    }
  }
  __syncthreads();
  // this CTA's partial: factors of the warps per head, then the weighted sum
  constexpr float LIFTED = KVF == 1 ? 256.f : 1.f;
  if (tid < SP_G) {
    float m = has_new ? s_new[tid] : -INFINITY, l = 0.f;
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_wml[w][tid]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2(s_wml[w][tid] - base);
      s_fac[w][tid] = f;
      l += s_wml[w][SP_G + tid] * f;
    }
    if (has_new) {
      const float f = ex2(s_new[tid] - base) * LIFTED;
      s_fac[15][tid] = f;
      l += f;
    }
    s_ml[tid] = m;
    s_ml[SP_G + tid] = l;
  }
  __syncthreads();
  // a row meets each CTA once and a CTA a row once, in the same order: row + CTA is a slot of their own
  float* part = FLAT ? a.part_o + size_t(row + blockIdx.x) * (SP_G * D) : s_part;
  for (int i = tid; i < SP_G * D; i += THREADS) {
    const int g = i / D;
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) o += s_wo[w * SP_G * D + i] * s_fac[w][g];
    if (has_new) o += __bfloat162float(a.v_new[size_t(row) * D + i % D]) * s_fac[15][g];
    part[i] = o;
  }
  if constexpr (FLAT) {
    if (tid < 2 * SP_G) a.part_ml[size_t(row + blockIdx.x) * (2 * SP_G) + tid] = s_ml[tid];
    todo -= s_end - s_begin;
    from = 0;
    if (++kvh == a.HKV) {
      kvh = 0;
      do { ++b; } while (b < a.t.B && flat_steps(a, b) == 0);
    }
    if (todo <= 0 || b >= a.t.B) return;
    __syncthreads();  // the ring and the partials' arrays are free
    continue;
  } else {
  cluster.sync();
  // every CTA finds the final maxima and sums and writes its share of the output
  __shared__ float s_cm[16][SP_G], s_cl[16][SP_G];
  for (int i = tid; i < NC * SP_G; i += THREADS) {
    const float* other = cluster.map_shared_rank(s_ml, i / SP_G);
    s_cm[i / SP_G][i % SP_G] = other[i % SP_G];
    s_cl[i / SP_G][i % SP_G] = other[SP_G + i % SP_G];
  }
  __syncthreads();
  if (tid < SP_G) {
    float m = -INFINITY, l = 0.f;
    for (int k = 0; k < NC; ++k) m = fmaxf(m, s_cm[k][tid]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int k = 0; k < NC; ++k) {
      const float f = ex2(s_cm[k][tid] - base);
      s_fac[k][tid] = f;
      l += s_cl[k][tid] * f;
    }
    s_fin[tid] = base;
    s_fin[SP_G + tid] = l == 0.f ? 0.f : 1.f / l;  // no row at all, or none with a weight: zeros
  }
  __syncthreads();
  const int share = (SP_G * D / 2 + NC - 1) / NC;  // channel pairs per CTA
  for (int i = rank * share + tid; i < min(SP_G * D / 2, (rank + 1) * share); i += THREADS) {
    const int g = 2 * i / D, d = 2 * i % D;
    if (g >= a.G) continue;
    float o0 = 0.f, o1 = 0.f;
    for (int k = 0; k < NC; ++k) {
      const float2 o = *reinterpret_cast<const float2*>(cluster.map_shared_rank(s_part, k) + 2 * i);
      o0 += o.x * s_fac[k][g];
      o1 += o.y * s_fac[k][g];
    }
    const float inv = s_fin[SP_G + g];
    *reinterpret_cast<uint32_t*>(a.out + (size_t(b) * a.HQ + size_t(kvh) * a.G + g) * D + d) =
        pack_bf16(o0 * inv, o1 * inv);
  }
  if (a.key_mass) {
    add_weights<THREADS>(a, sp, pages, kvh, scores, s_begin * SP_KEYS, min(n_keys, s_end * SP_KEYS), s_fin, s_fin + SP_G, LIFTED);
    if (has_new && tid == 0) add_new_weight(a, b, kvh, s_new, s_fin, s_fin + SP_G, LIFTED);
  }
  cluster.sync();  // no CTA leaves while another still reads its shared memory
  return;
  }
  }
}

// The flat form's second kernel: `chunks` CTAs per (sequence, KV head) merge its partials -- each a share of the output --
// and turn a share of its scores into weights.
template <int D, int KVF>
__global__ void __launch_bounds__(256) sparse_merge_kernel(const SparseArgs a) {
  constexpr float LIFTED = KVF == 1 ? 256.f : 1.f;
  __shared__ int s_flat[2];
  __shared__ float s_m[32][SP_G], s_l[32][SP_G], s_new[SP_G], s_top[SP_G], s_inv[SP_G];
  extern __shared__ float s_fac[];  // [partials of the row][8]
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks, b = row / a.HKV, kvh = row % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  const int steps = flat_steps(a, b), P = a.t.P;
  if (warp == 0) {
    const int per = flat_per_cta(a);
    int before = 0;
    for (int i = lane; i < b; i += 32) before += flat_steps(a, i);
    before = __reduce_add_sync(0xffffffffu, before);
    if (lane == 0) { s_flat[0] = per; s_flat[1] = before * a.HKV + kvh * steps; }
  }
  if (a.k_new) {  // the current token, from its own rows: one more partial (l = 1, o = v)
    const float scale_log2 = (a.sm_scale ? a.sm_scale[0] : rsqrtf(float(D))) * SP_LOG2E;
    float dot = 0.f;
    if (warp < a.G) {
      const __nv_bfloat16 *kp = a.k_new + size_t(row) * D, *qp = a.q + (size_t(b) * a.HQ + size_t(kvh) * a.G + warp) * D;
      for (int d = lane; d < D; d += 32) dot += __bfloat162float(qp[d]) * __bfloat162float(kp[d]);
    }
    dot = warp_sum(dot);
    if (lane == 0) s_new[warp] = dot * scale_log2;
  }
  __syncthreads();
  // (held to the CTAs there are: ranges of a bad table may overlap and add up to more steps than an int holds)
  const int first = min(max(s_flat[1] / s_flat[0], 0), a.n_cta - 1);
  const int n = steps ? min(max((s_flat[1] + steps - 1) / s_flat[0] - first + 1, 0), a.n_cta - first) : 0;
  const float* ml = a.part_ml + size_t(row + first) * (2 * SP_G);
  {
    const int g = tid % SP_G, j0 = tid / SP_G;
    float m = -INFINITY, l = 0.f;
    for (int j = j0; j < n; j += 32) m = fmaxf(m, ml[j * 2 * SP_G + g]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int j = j0; j < n; j += 32) l += ml[j * 2 * SP_G + SP_G + g] * ex2(ml[j * 2 * SP_G + g] - base);
    s_m[j0][g] = m;
    s_l[j0][g] = l;
  }
  __syncthreads();
  if (tid < SP_G) {
    float m = a.k_new ? s_new[tid] : -INFINITY, l = 0.f;
    for (int j = 0; j < 32; ++j) m = fmaxf(m, s_m[j][tid]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int j = 0; j < 32; ++j) l += s_l[j][tid] * ex2(s_m[j][tid] - base);
    if (a.k_new) l += ex2(s_new[tid] - base) * LIFTED;
    s_top[tid] = base;
    s_inv[tid] = l == 0.f ? 0.f : 1.f / l;
  }
  __syncthreads();
  for (int i = tid; i < n * SP_G; i += 256) s_fac[i] = ex2(ml[i / SP_G * 2 * SP_G + i % SP_G] - s_top[i % SP_G]);
  __syncthreads();
  const int share = (SP_G * D / 2 + a.chunks - 1) / a.chunks;  // channel pairs per CTA
  for (int i = chunk * share + tid; i < min(SP_G * D / 2, (chunk + 1) * share); i += 256) {
    const int g = 2 * i / D, d = 2 * i % D;
    if (g >= a.G) continue;
    const float* po = a.part_o + size_t(row + first) * (SP_G * D) + 2 * i;
    float o0 = 0.f, o1 = 0.f;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const float2 o = *reinterpret_cast<const float2*>(po + size_t(j) * (SP_G * D));
      o0 += o.x * s_fac[j * SP_G + g];
      o1 += o.y * s_fac[j * SP_G + g];
    }
    if (a.k_new) {
      const float f = ex2(s_new[g] - s_top[g]) * LIFTED;
      o0 += __bfloat162float(a.v_new[size_t(row) * D + d]) * f;
      o1 += __bfloat162float(a.v_new[size_t(row) * D + d + 1]) * f;
    }
    const float inv = s_inv[g];
    *reinterpret_cast<uint32_t*>(a.out + (size_t(b) * a.HQ + size_t(kvh) * a.G + g) * D + d) = pack_bf16(o0 * inv, o1 * inv);
  }
  if (!a.key_mass) return;
  const float* scores = a.scores + (size_t(a.HKV) * sp.first + size_t(kvh) * sp.n) * size_t(P) * SP_G;
  const int keys = (sp.ctx + a.chunks - 1) / a.chunks;
  add_weights<256>(a, sp, nullptr, kvh, scores, chunk * keys, min(sp.ctx, (chunk + 1) * keys), s_top, s_inv, LIFTED);
  if (a.k_new && chunk == 0 && tid == 0) add_new_weight(a, b, kvh, s_new, s_top, s_inv, LIFTED);
}

// CTAs per (sequence, KV head).  `slots` CTAs are resident at a time.
// Chosen pages: all rows of the grid have about the same length, the most CTAs that still run at once (64 sequences x
// 2 heads x 4096 rows on 148 slots: 1 CTA 90 us, 2: 98, 4: 113).  All pages: lengths differ, so at least one CTA per
// slot, and more to even them out (32 x 4 ragged E4M3 rows with weights on 296 slots: 2 CTAs 59 us, 4: 54, 8: 70).
// Never more than one step per warp; 16 (beyond the portable 8) for a few long rows.
static int sparse_cluster(int64_t rows, int64_t steps, int slots, bool chosen) {
  int c = 1;
  while (c < 8 && (chosen ? rows * c * 2 <= slots : rows * c < slots)) c *= 2;
  if (c == 8 && rows * 16 <= slots && steps >= 16 * 32) c = 16;
  while (c > 1 && c / 2 * 4 >= steps) c /= 2;
  return c;
}

template <int D, int KVF>
static int launch_sparse(const SparseArgs& a, cudaStream_t stream) {
  using C = SparseCfg<D, KVF>;
  const void* f = reinterpret_cast<const void*>(sparse_decode_kernel<D, KVF, false>);
  // the 48 KB that need no opt-in hold the static arrays too: head_dim 64 is above them with exactly 48 KB of ring
  Q35_TRY(ensure_dynamic_smem(f, C::SMEM > 49 * 1024 ? C::SMEM : 49 * 1024));
  const int64_t rows = int64_t(a.t.B) * a.HKV;
  if (a.part_o) {
    const void* flat = reinterpret_cast<const void*>(sparse_decode_kernel<D, KVF, true>);
    Q35_TRY(ensure_dynamic_smem(flat, C::SMEM > 49 * 1024 ? C::SMEM : 49 * 1024));
    launch_pdl(sparse_decode_kernel<D, KVF, true>, dim3(unsigned(a.n_cta)), dim3(32 * C::WARPS), C::SMEM, stream, a);
    Q35_CUDA_LAUNCH_CHECK("attn.sparse_decode rows");
    launch_pdl(sparse_merge_kernel<D, KVF>, dim3(unsigned(rows * a.chunks)), dim3(256), size_t(a.n_cta) * SP_G * 4, stream, a);
    Q35_CUDA_LAUNCH_CHECK("attn.sparse_decode merge");
    return 0;
  }
  const int64_t keys = int64_t(a.t.P) * (a.pages ? a.S : (a.t.n_indices + a.t.B - 1) / a.t.B);
  const int cluster = sparse_cluster(rows, (keys + SP_KEYS - 1) / SP_KEYS, C::CTAS * sm_count(),
                                     a.pages != nullptr);
  cudaError_t e = cudaSuccess;
  if (cluster > 8) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(rows * cluster));
    cfg.blockDim = dim3(32 * C::WARPS);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cluster); attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, sparse_decode_kernel<D, KVF, false>, a);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the caller's next CUDA call
    return fail(Q35_ERR_CUDA, "attn.sparse_decode: %s", cudaGetErrorString(e));
  }
  Q35_CUDA_LAUNCH_CHECK("attn.sparse_decode");
  return 0;
}

int run_attn_sparse_decode(Call& c) {
  const char* role = "attn.sparse_decode";
  KvCache kv;
  Q35_TRY(get_kv_cache(c, role, &kv));
  Tensor q, pages, scale, kn, vn, loc, out, mass, ws;
  Q35_TRY(c.get("q", M(Q35_BF16), &q));
  Q35_TRY(c.get("pages", M(Q35_I32), &pages, false));
  Q35_TRY(c.get("sm_scale", M(Q35_F32), &scale, false));
  Q35_TRY(c.get("k_new", M(Q35_BF16), &kn, false));
  Q35_TRY(c.get("v_new", M(Q35_BF16), &vn, false));
  Q35_TRY(c.get("cache_location", M(Q35_I32), &loc, false));
  Q35_TRY(c.get("key_mass", M(Q35_F32), &mass, false));
  Q35_TRY(c.get("out", M(Q35_BF16), &out));
  Q35_REQUIRE(q.nd == 3, Q35_ERR_SHAPE, "%s: q [B, HQ, D]", role);
  const int64_t B = q.s[0], HQ = q.s[1], D = q.s[2], HKV = kv.HKV, P = kv.P;
  Q35_REQUIRE(kv.D == D && HQ >= 1 && HQ % HKV == 0, Q35_ERR_SHAPE, "%s: head shapes", role);
  Q35_REQUIRE(HQ / HKV <= SP_G, Q35_ERR_UNSUPPORTED, "%s: at most 8 query heads per KV head (got %lld)", role,
              (long long)(HQ / HKV));
  Q35_REQUIRE(D == 64 || D == 128 || D == 256, Q35_ERR_UNSUPPORTED, "%s: head_dim must be 64/128/256", role);
  Q35_REQUIRE(P % SP_SUB == 0, Q35_ERR_UNSUPPORTED, "%s: page size must be a multiple of 16", role);
  Q35_REQUIRE(out.numel() == B * HQ * D, Q35_ERR_SHAPE, "%s: out [B, HQ, D]", role);
  Q35_REQUIRE(!pages.present || (pages.nd == 3 && pages.s[0] == B && pages.s[1] == HKV && pages.s[2] >= 1), Q35_ERR_SHAPE,
              "%s: pages [B, HKV, S]", role);
  Q35_REQUIRE(!scale.present || scale.numel() == 1, Q35_ERR_SHAPE, "%s: sm_scale [1]", role);
  Q35_REQUIRE(kn.present == vn.present, Q35_ERR_MISSING, "%s: k_new and v_new go together", role);
  Q35_REQUIRE(!kn.present || (kn.numel() == B * HKV * D && vn.numel() == B * HKV * D), Q35_ERR_SHAPE,
              "%s: k_new / v_new [B, HKV, D]", role);
  Q35_REQUIRE(!mass.present || mass.numel() == kv.pages * P * HKV, Q35_ERR_SHAPE, "%s: key_mass [pages, P, HKV]", role);
  Q35_REQUIRE(loc.present == (mass.present && kn.present), Q35_ERR_MISSING,
              "%s: cache_location [B, 2] goes with key_mass and k_new: where the current token's own weight is stored", role);
  Q35_REQUIRE(!loc.present || loc.numel() == 2 * B, Q35_ERR_SHAPE, "%s: cache_location [B, 2]", role);
  SparseArgs a{};
  Q35_TRY(get_page_table(c, role, B, P, kv.pages, &a.t));
  const int64_t S = pages.present ? pages.s[2] : 0;
  Q35_REQUIRE(S <= INT_MAX / 2 / P && B * HKV <= INT_MAX / 16, Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  const int64_t rows = pages.present ? B * HKV * S * P : HKV * int64_t(a.t.n_indices) * P;
  // The flat form, for all pages of many rows: every CTA the same number of steps, whatever the lengths, a second kernel
  // that merges.  It pays from 48 steps per CTA and 256 per row on (8 rows of 60000 bf16: 92 us, clusters 146; 74 rows of
  // 32000 E4M3: 203 and 308; but 128 ragged E4M3 rows of up to 131 steps, with weights: 60 and 54); below, and for chosen
  // pages, whose rows are about equally long, one launch of clusters.  Rows too few to fill the GPU's steps stay with the
  // clusters as well, although equal shares serve them better from about 32000 cached rows on (one sequence of two heads,
  // 65536 bf16 rows: 43 us, clusters 78; 131072 E4M3 rows: 47 and 133; 16384: 26 and 26, 23 and 24).
  a.n_cta = sm_count() * (D == 256 ? (kv.fmt ? 2 : 1) : D == 128 ? (kv.fmt ? 3 : 2) : 4);
  const int64_t all_steps = HKV * (int64_t(a.t.n_indices) * P / SP_KEYS);
  Q35_REQUIRE(pages.present || all_steps + B * HKV <= INT_MAX, Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  const bool flat = !pages.present && all_steps >= 48 * int64_t(a.n_cta) && all_steps >= 256 * B * HKV;
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = (off + bytes + 255) / 256 * 256; return o; };
  const int64_t slots = flat ? B * HKV + a.n_cta : 0;
  const int64_t o_scores = take(mass.present ? rows * SP_G * 4 : 0), o_po = take(slots * SP_G * D * 4),
                o_ml = take(slots * 2 * SP_G * 4);
  Q35_TRY(c.workspace(off, &ws));
  if (c.dry || B == 0) return 0;
  Q35_REQUIRE(aligned16(q.p) && aligned16(out.p), Q35_ERR_ALIGN, "%s: q and out must be 16-byte aligned", role);
  a.q = q.as<__nv_bfloat16>(); a.cache = static_cast<const uint8_t*>(kv.p);
  a.kv_scale = kv.kv_scale; a.row_scale = kv.row_scale;
  a.pages = pages.present ? pages.as<int>() : nullptr;
  a.sm_scale = scale.present ? scale.as<float>() : nullptr;
  a.k_new = kn.present ? kn.as<__nv_bfloat16>() : nullptr;
  a.v_new = vn.present ? vn.as<__nv_bfloat16>() : nullptr;
  a.new_at = loc.present ? loc.as<int>() : nullptr;
  a.out = out.as<__nv_bfloat16>();
  a.key_mass = mass.present ? mass.as<float>() : nullptr;
  a.scores = mass.present ? reinterpret_cast<float*>(ws.as<uint8_t>() + o_scores) : nullptr;
  if (flat) {
    a.part_o = reinterpret_cast<float*>(ws.as<uint8_t>() + o_po);
    a.part_ml = reinterpret_cast<float*>(ws.as<uint8_t>() + o_ml);
    const int64_t per_row = int64_t(a.t.n_indices) * P / B;  // the second kernel: a CTA per 2048 rows of the average one
    a.chunks = int(per_row / 2048 + 1);
  }
  a.HQ = int(HQ); a.HKV = int(HKV); a.G = int(HQ / HKV); a.S = int(S);
#define Q35_SPARSE(DD)                                                 \
  (kv.fmt == 0 ? launch_sparse<DD, 0>(a, c.stream) : kv.fmt == 1 ? launch_sparse<DD, 1>(a, c.stream) \
                                                                 : launch_sparse<DD, 2>(a, c.stream))
  if (D == 64) return Q35_SPARSE(64);
  if (D == 128) return Q35_SPARSE(128);
  return Q35_SPARSE(256);
#undef Q35_SPARSE
}

}  // namespace q35
