// attn.sparse_decode: one query token per sequence over chosen pages of its cache (or all of them), optionally adding
// the softmax weight that every cached row receives to key_mass.
//
// With s_gi = q_g . k_i * scale over the rows i of the chosen pages, M_g = max_i s_gi, L_g = sum_i exp(s_gi - M_g):
//   out_g = sum_i exp(s_gi - M_g) v_i / L_g,     key_mass_i += sum_g exp(s_gi - M_g) / L_g   (g over the group's heads).
//
// Bound: HBM, K and V of the chosen rows once.  A cluster of C CTAs serves one (sequence, KV head): its chosen rows,
// laid end to end, are cut into C contiguous ranges, every CTA runs one pass with a running maximum and sum over its
// range, and the C partial results are merged through distributed shared memory -- one launch, no partials in HBM, no
// counters.  Inside a CTA each warp owns groups of 16 rows and its own cp.async ring (16-byte chunks, XOR-swizzled
// rows), with no block barrier in the loop.  Scores are computed transposed (S^T = K Q^T, mma.m16n8k16) so that the up
// to 8 query heads of a KV head are the n = 8 side and O^T takes D / 4 registers a lane.
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
constexpr int SP_KEYS = 16;      // rows per warp and step
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
  int HQ, HKV, G, S;
};

// KVF: 0 bf16, 1 E4M3, 2 int8 rows with scales.  The one-byte formats arrive in half the time, so their dependent chain
// (load fragments, convert, MMA, softmax, MMA) needs two warps per scheduler to hide; bf16 needs one.
template <int D, int KVF>
struct SparseCfg {
  static constexpr bool BYTE = KVF != 0;
  static constexpr int WARPS = BYTE ? 8 : 4;
  static constexpr int STAGES = 3;
  static constexpr int ROWB = D * (BYTE ? 1 : 2);
  static constexpr int CPR = ROWB / 16;                 // 16-byte chunks per row
  static constexpr int SWZ = (CPR < 8 ? CPR : 8) - 1;   // rows narrower than 128 bytes permute fewer chunks
  static constexpr int KV_BYTES = SP_KEYS * ROWB;
  static constexpr int STAGE_BYTES = 2 * KV_BYTES;
  static constexpr int RING = WARPS * STAGES * STAGE_BYTES;
  static constexpr int PART = WARPS * SP_G * D * 4;     // the warps' output partials reuse the ring
  static constexpr int SMEM = RING > PART ? RING : PART;
  static constexpr int LD = SP_KEYS * CPR / 32;         // chunks of K (and of V) per lane and step
};

template <int D, int KVF>
__global__ void __launch_bounds__(32 * SparseCfg<D, KVF>::WARPS, 1) sparse_decode_kernel(const SparseArgs a) {
  using C = SparseCfg<D, KVF>;
  constexpr int WARPS = C::WARPS, THREADS = 32 * WARPS, STAGES = C::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_part[SP_G * D];                        // this CTA's merged output, read by the cluster
  __shared__ float s_ml[2 * SP_G];                          // its maxima and sums, read by the cluster
  __shared__ float s_wml[WARPS][2 * SP_G];
  __shared__ float s_fac[16][SP_G], s_fin[2 * SP_G], s_new[SP_G];
  __shared__ int s_cut;
  pdl_wait();
  pdl_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int NC = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
  const int row = blockIdx.x / NC, b = row / a.HKV, kvh = row % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  const int P = a.t.P;

  // the chosen pages: ascending positions in the sequence's page list; the list ends at the first entry that is not
  const int* pages = a.pages ? a.pages + size_t(row) * a.S : nullptr;
  int n_sel = sp.n, n_keys = sp.ctx;
  if (pages) {
    if (tid == 0) s_cut = a.S;
    __syncthreads();
    for (int i = tid; i < a.S; i += THREADS) {
      const int p = pages[i], before = i ? pages[i - 1] : -1;
      if (p < 0 || p >= sp.n || p <= before) {
        if (p < -1 || (p >= 0 && before >= 0) || p >= sp.n) atomicOr(a.t.status, DS_BAD_PAGE);
        atomicMin(&s_cut, i);
      }
    }
    __syncthreads();
    n_sel = s_cut;
    n_keys = n_sel * P;
    if (n_sel > 0 && pages[n_sel - 1] == sp.n - 1) n_keys += sp.ctx - sp.n * P;  // the last page may be part full
  }
  auto phys = [&](int slot) -> int { return page_at(a.t, sp.first + (pages ? pages[slot] : slot)); };

  // groups of 16 rows: this CTA's contiguous range, dealt to its warps in turn
  const int groups = (n_keys + SP_KEYS - 1) / SP_KEYS, per = (groups + NC - 1) / NC;
  const int g_begin = min(groups, rank * per), g_end = min(groups, g_begin + per);
  const float scale_log2 = (a.sm_scale ? a.sm_scale[0] : rsqrtf(float(D))) * SP_LOG2E;
  const size_t row_stride = size_t(a.HKV) * C::ROWB;  // bytes between consecutive rows of a page plane
  // scores of this (sequence, KV head): behind S * P rows of every row of the grid, or behind the table entries before
  float* scores = a.scores;
  if (scores)
    scores += (pages ? size_t(row) * a.S : size_t(a.HKV) * sp.first + size_t(kvh) * sp.n) * size_t(P) * SP_G;

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

  const uint32_t sbase = smem_u32(smem) + warp * (STAGES * C::STAGE_BYTES);
  const int first_group = g_begin + warp;
  // physical page of a group (16 rows lie in one page: P is a multiple of 16), looked up ahead of its use
  auto group_page = [&](int g) -> int {
    if (g >= g_end) return 0;
    const int p = phys(g * SP_KEYS / P);
    return p < 0 ? 0 : p;
  };
  auto issue = [&](int g, int page) {
    if (g < g_end) {
      const int ro = g * SP_KEYS % P, valid = min(SP_KEYS, n_keys - g * SP_KEYS);
      const uint8_t* kb = a.cache + (size_t(page) * 2 * P + ro) * row_stride + size_t(kvh) * C::ROWB;
      const uint8_t* vb = kb + size_t(P) * row_stride;
      const uint32_t st = sbase + ((g - first_group) / WARPS % STAGES) * C::STAGE_BYTES;
#pragma unroll
      for (int j = 0; j < C::LD; ++j) {
        const int ci = lane + 32 * j, key = ci / C::CPR, ch = ci % C::CPR;
        const uint32_t at = st + key * C::ROWB + ((ch ^ (key & C::SWZ)) << 4);
        if (key < valid) {
          cp_async_16(at, kb + size_t(key) * row_stride + ch * 16);
          cp_async_16(at + C::KV_BYTES, vb + size_t(key) * row_stride + ch * 16);
        } else {  // rows behind the end are never read: zeros keep 0 * V a zero
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at), "r"(0u));
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(at + C::KV_BYTES), "r"(0u));
        }
      }
    }
    cp_async_commit();
  };
  // int8: the row scales this lane's fragments need -- K rows r and r + 8, V rows 2 c, 2 c + 1, 2 c + 8, 2 c + 9 -- two
  // groups ahead in registers; 0 for rows behind the end
  auto load_scales = [&](int g, int page) -> uint3 {
    uint3 v = make_uint3(0u, 0u, 0u);
    if constexpr (KVF == 2) {
      if (g < g_end) {
        const int ro = g * SP_KEYS % P, valid = n_keys - g * SP_KEYS;
        const unsigned short* ks = reinterpret_cast<const unsigned short*>(a.row_scale) +
                                   (size_t(page) * 2 * P + ro) * a.HKV + kvh;
        const unsigned short* vs = ks + size_t(P) * a.HKV;
        auto at = [&](const unsigned short* s, int i) -> uint32_t { return i < valid ? s[size_t(i) * a.HKV] : 0u; };
        v.x = at(ks, r) | at(ks, r + 8) << 16;
        v.y = at(vs, 2 * c) | at(vs, 2 * c + 1) << 16;
        v.z = at(vs, 2 * c + 8) | at(vs, 2 * c + 9) << 16;
      }
    }
    return v;
  };

  float oacc[D / 16][4];
#pragma unroll
  for (int mt = 0; mt < D / 16; ++mt) oacc[mt][0] = oacc[mt][1] = oacc[mt][2] = oacc[mt][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};

  uint3 rs_cur, rs_n1, rs_n2;
  {
    const int p0 = group_page(first_group), p1 = group_page(first_group + WARPS);
    issue(first_group, p0);
    issue(first_group + WARPS, p1);
    rs_cur = load_scales(first_group, p0);
    rs_n1 = load_scales(first_group + WARPS, p1);
  }
  static_assert(STAGES == 3, "two groups in flight ahead of the one in use");
  int page_next = group_page(first_group + 2 * WARPS);

  for (int g = first_group; g < g_end; g += WARPS) {
    issue(g + 2 * WARPS, page_next);
    rs_n2 = load_scales(g + 2 * WARPS, page_next);
    page_next = group_page(g + 3 * WARPS);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const int valid = min(SP_KEYS, n_keys - g * SP_KEYS);
    const uint32_t st = sbase + ((g - first_group) / WARPS % STAGES) * C::STAGE_BYTES;
    float sacc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    {
      const int key = (lane & 7) + (((lane >> 3) & 1) << 3);
      const uint32_t rowa = st + key * C::ROWB;
      if constexpr (!C::BYTE) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const int ch = 2 * ks + (lane >> 4);
          uint32_t a0, a1, a2, a3;
          ldmatrix_x4(rowa + ((ch ^ (key & C::SWZ)) << 4), a0, a1, a2, a3);
          mma_bf16_16816(sacc[ks & 1], a0, a1, a2, a3, qf[ks][0], qf[ks][1]);
        }
      } else {
#pragma unroll
        for (int kp = 0; kp < D / 32; ++kp) {  // 32 channels: two mma over bytes taken as b16 pairs
          const int ch = 2 * kp + (lane >> 4);
          uint32_t r0, r1, r2, r3;
          ldmatrix_x4(rowa + ((ch ^ (key & C::SWZ)) << 4), r0, r1, r2, r3);
          if constexpr (KVF == 2) {
            const float s0 = bf16lo(rs_cur.x), s1 = bf16hi(rs_cur.x);
            r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
            mma_bf16_16816(sacc[0], cvt_s8x2_bf16x2<0, 1>(r0, s0, s0), cvt_s8x2_bf16x2<0, 1>(r1, s1, s1),
                           cvt_s8x2_bf16x2<2, 3>(r0, s0, s0), cvt_s8x2_bf16x2<2, 3>(r1, s1, s1), qf[2 * kp][0],
                           qf[2 * kp][1]);
            mma_bf16_16816(sacc[1], cvt_s8x2_bf16x2<0, 1>(r2, s0, s0), cvt_s8x2_bf16x2<0, 1>(r3, s1, s1),
                           cvt_s8x2_bf16x2<2, 3>(r2, s0, s0), cvt_s8x2_bf16x2<2, 3>(r3, s1, s1), qf[2 * kp + 1][0],
                           qf[2 * kp + 1][1]);
          } else {
            mma_f16_16816(sacc[0], cvt_kv<0, 1>(r0), cvt_kv<0, 1>(r1), cvt_kv<2, 3>(r0), cvt_kv<2, 3>(r1),
                          qf[2 * kp][0], qf[2 * kp][1]);
            mma_f16_16816(sacc[1], cvt_kv<0, 1>(r2), cvt_kv<0, 1>(r3), cvt_kv<2, 3>(r2), cvt_kv<2, 3>(r3),
                          qf[2 * kp + 1][0], qf[2 * kp + 1][1]);
          }
        }
      }
    }
    float sc[4];  // rows r, r, r + 8, r + 8; heads 2 c, 2 c + 1
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sc[i] = r + ((i >> 1) << 3) < valid ? (sacc[0][i] + sacc[1][i]) * col_scale[i & 1] : -INFINITY;
    if (scores) {
      float* at = scores + (size_t(g) * SP_KEYS + r) * SP_G + 2 * c;
      if (r < valid) *reinterpret_cast<float2*>(at) = make_float2(sc[0], sc[1]);
      if (r + 8 < valid) *reinterpret_cast<float2*>(at + 8 * SP_G) = make_float2(sc[2], sc[3]);
    }
    float mt2[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      mt2[0] = fmaxf(mt2[0], __shfl_xor_sync(0xffffffffu, mt2[0], o));
      mt2[1] = fmaxf(mt2[1], __shfl_xor_sync(0xffffffffu, mt2[1], o));
    }
    // E4M3: weights 2^8 times larger, up to 256, so that the f16 pair that carries them resolves 2^-32 of the maximum
    constexpr float LIFT = KVF == 1 ? 8.f : 0.f;
    float alpha[2], ref[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float mn = fmaxf(m_run[h], mt2[h]);
      const float base = mn == -INFINITY ? 0.f : mn;  // no row with a weight yet
      alpha[h] = exp2f(m_run[h] - base);
      m_run[h] = mn;
      ref[h] = base - LIFT;
    }
    const float p0 = exp2f(sc[0] - ref[0]), p1 = exp2f(sc[1] - ref[1]);
    const float p2 = exp2f(sc[2] - ref[0]), p3 = exp2f(sc[3] - ref[1]);
    l_run[0] = l_run[0] * alpha[0] + p0 + p2;
    l_run[1] = l_run[1] * alpha[1] + p1 + p3;
    if (alpha[0] != 1.f || alpha[1] != 1.f) {
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        oacc[mt][0] *= alpha[0]; oacc[mt][1] *= alpha[1];
        oacc[mt][2] *= alpha[0]; oacc[mt][3] *= alpha[1];
      }
    }
    // P enters the P V product as two 16-bit terms (p = hi + lo): one alone would cost as much as the output's rounding
    if constexpr (!C::BYTE) {
      const float h0 = round_bf16(p0), h1 = round_bf16(p1), h2 = round_bf16(p2), h3 = round_bf16(p3);
      const uint32_t pb0 = movmatrix_trans(pack_bf16(h0, h1)), pb1 = movmatrix_trans(pack_bf16(h2, h3));
      const uint32_t pl0 = movmatrix_trans(pack_bf16(p0 - h0, p1 - h1));
      const uint32_t pl1 = movmatrix_trans(pack_bf16(p2 - h2, p3 - h3));
      const int key = (lane & 7) + ((lane >> 4) << 3);
      const uint32_t rowa = st + C::KV_BYTES + key * C::ROWB;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        const int ch = 2 * mt + ((lane >> 3) & 1);
        uint32_t a0, a1, a2, a3;
        ldmatrix_x4_trans(rowa + ((ch ^ (key & C::SWZ)) << 4), a0, a1, a2, a3);
        mma_bf16_16816(oacc[mt], a0, a1, a2, a3, pb0, pb1);
        mma_bf16_16816(oacc[mt], a0, a1, a2, a3, pl0, pl1);
      }
    } else {
      // transposed b16 loads keep byte pairs (d, d + 1) together: bytes (0, 2) / (1, 3) are the row pairs of channels
      // 2 r / 2 r + 1, so mma row r holds channel 16 mt + 2 r and mma row r + 8 channel 16 mt + 2 r + 1
      uint32_t pb0, pb1, pl0, pl1;
      if constexpr (KVF == 2) {
        const float h0 = round_bf16(p0), h1 = round_bf16(p1), h2 = round_bf16(p2), h3 = round_bf16(p3);
        pb0 = movmatrix_trans(pack_bf16(h0, h1));
        pb1 = movmatrix_trans(pack_bf16(h2, h3));
        pl0 = movmatrix_trans(pack_bf16(p0 - h0, p1 - h1));
        pl1 = movmatrix_trans(pack_bf16(p2 - h2, p3 - h3));
      } else {
        auto hi = [](float p) { return __half2float(__float2half_rn(p)); };
        const float h0 = hi(p0), h1 = hi(p1), h2 = hi(p2), h3 = hi(p3);
        pb0 = movmatrix_trans(pack_f16(h0, h1));
        pb1 = movmatrix_trans(pack_f16(h2, h3));
        pl0 = movmatrix_trans(pack_f16(p0 - h0, p1 - h1));
        pl1 = movmatrix_trans(pack_f16(p2 - h2, p3 - h3));
      }
      const int key = lane & 15;
      const uint32_t rowa = st + C::KV_BYTES + key * C::ROWB;
#pragma unroll
      for (int mp = 0; mp < D / 32; ++mp) {
        const int ch = 2 * mp + (lane >> 4);
        uint32_t r0, r1, r2, r3;  // (rows 0-7, chunk 2 mp) (rows 8-15, 2 mp) (rows 0-7, 2 mp + 1) (rows 8-15, 2 mp + 1)
        ldmatrix_x4_trans(rowa + ((ch ^ (key & C::SWZ)) << 4), r0, r1, r2, r3);
        if constexpr (KVF == 2) {
          const float va = bf16lo(rs_cur.y), vb = bf16hi(rs_cur.y), vc = bf16lo(rs_cur.z), vd = bf16hi(rs_cur.z);
          r0 ^= 0x80808080u; r1 ^= 0x80808080u; r2 ^= 0x80808080u; r3 ^= 0x80808080u;
          const uint32_t a0 = cvt_s8x2_bf16x2<0, 2>(r0, va, vb), a1 = cvt_s8x2_bf16x2<1, 3>(r0, va, vb);
          const uint32_t a2 = cvt_s8x2_bf16x2<0, 2>(r1, vc, vd), a3 = cvt_s8x2_bf16x2<1, 3>(r1, vc, vd);
          mma_bf16_16816(oacc[2 * mp], a0, a1, a2, a3, pb0, pb1);
          mma_bf16_16816(oacc[2 * mp], a0, a1, a2, a3, pl0, pl1);
          const uint32_t b0 = cvt_s8x2_bf16x2<0, 2>(r2, va, vb), b1 = cvt_s8x2_bf16x2<1, 3>(r2, va, vb);
          const uint32_t b2 = cvt_s8x2_bf16x2<0, 2>(r3, vc, vd), b3 = cvt_s8x2_bf16x2<1, 3>(r3, vc, vd);
          mma_bf16_16816(oacc[2 * mp + 1], b0, b1, b2, b3, pb0, pb1);
          mma_bf16_16816(oacc[2 * mp + 1], b0, b1, b2, b3, pl0, pl1);
        } else {
          const uint32_t a0 = cvt_kv<0, 2>(r0), a1 = cvt_kv<1, 3>(r0), a2 = cvt_kv<0, 2>(r1), a3 = cvt_kv<1, 3>(r1);
          mma_f16_16816(oacc[2 * mp], a0, a1, a2, a3, pb0, pb1);
          mma_f16_16816(oacc[2 * mp], a0, a1, a2, a3, pl0, pl1);
          const uint32_t b0 = cvt_kv<0, 2>(r2), b1 = cvt_kv<1, 3>(r2), b2 = cvt_kv<0, 2>(r3), b3 = cvt_kv<1, 3>(r3);
          mma_f16_16816(oacc[2 * mp + 1], b0, b1, b2, b3, pb0, pb1);
          mma_f16_16816(oacc[2 * mp + 1], b0, b1, b2, b3, pl0, pl1);
        }
      }
    }
    __syncwarp();
    rs_cur = rs_n1;
    rs_n1 = rs_n2;
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
  const bool has_new = a.k_new != nullptr && rank == 0;
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
      const float f = exp2f(s_wml[w][tid] - base);
      s_fac[w][tid] = f;
      l += s_wml[w][SP_G + tid] * f;
    }
    if (has_new) {
      const float f = exp2f(s_new[tid] - base) * LIFTED;
      s_fac[15][tid] = f;
      l += f;
    }
    s_ml[tid] = m;
    s_ml[SP_G + tid] = l;
  }
  __syncthreads();
  for (int i = tid; i < SP_G * D; i += THREADS) {
    const int g = i / D;
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) o += s_wo[w * SP_G * D + i] * s_fac[w][g];
    if (has_new) o += __bfloat162float(a.v_new[size_t(row) * D + i % D]) * s_fac[15][g];
    s_part[i] = o;
  }
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
      const float f = exp2f(s_cm[k][tid] - base);
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
    // the lifted weights' sums are 2^LIFT times larger: so is what a score stands for
    for (int k = g_begin * SP_KEYS + tid; k < min(n_keys, g_end * SP_KEYS); k += THREADS) {
      const float4 s0 = *reinterpret_cast<const float4*>(scores + size_t(k) * SP_G);
      const float4 s1 = *reinterpret_cast<const float4*>(scores + size_t(k) * SP_G + 4);
      const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
      float w = 0.f;
#pragma unroll
      for (int g = 0; g < SP_G; ++g)
        if (g < a.G) w += exp2f(s[g] - s_fin[g]) * s_fin[SP_G + g];
      const int page = phys(k / P);
      if (page >= 0) atomicAdd(a.key_mass + (size_t(page) * P + k % P) * a.HKV + kvh, w * LIFTED);
    }
    if (has_new && tid == 0) {
      float w = 0.f;
      for (int g = 0; g < a.G; ++g) w += exp2f(s_new[g] - s_fin[g]) * s_fin[SP_G + g];
      const int page = a.new_at[2 * b], off = a.new_at[2 * b + 1];
      if (unsigned(page) < unsigned(a.t.num_pages) && unsigned(off) < unsigned(P))
        a.key_mass[(size_t(page) * P + off) * a.HKV + kvh] = w * LIFTED;
      else
        atomicOr(a.t.status, DS_BAD_PAGE);
    }
  }
  cluster.sync();  // no CTA leaves while another still reads its shared memory
}

template <int D, int KVF>
static int launch_sparse(const SparseArgs& a, int cluster, cudaStream_t stream) {
  using C = SparseCfg<D, KVF>;
  const void* f = reinterpret_cast<const void*>(sparse_decode_kernel<D, KVF>);
  // the 48 KB that need no opt-in hold the static arrays too: head_dim 64 is above them with exactly 48 KB of ring
  Q35_TRY(ensure_dynamic_smem(f, C::SMEM > 49 * 1024 ? C::SMEM : 49 * 1024));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.t.B) * a.HKV * cluster);
  cfg.blockDim = dim3(32 * C::WARPS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster); attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sparse_decode_kernel<D, KVF>, a);
  Q35_REQUIRE(e == cudaSuccess, Q35_ERR_CUDA, "attn.sparse_decode: %s", cudaGetErrorString(e));
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
  Q35_REQUIRE(P % SP_KEYS == 0, Q35_ERR_UNSUPPORTED, "%s: page size must be a multiple of 16", role);
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
  Q35_REQUIRE(S <= INT_MAX / P - 1 && B * HKV <= INT_MAX / 16, Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  const int64_t rows = pages.present ? B * HKV * S * P : HKV * int64_t(a.t.n_indices) * P;
  Q35_TRY(c.workspace(mass.present ? rows * SP_G * 4 : 0, &ws));
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
  a.scores = mass.present ? ws.as<float>() : nullptr;
  a.HQ = int(HQ); a.HKV = int(HKV); a.G = int(HQ / HKV); a.S = int(S);
  const int cluster = 8;
#define Q35_SPARSE(DD)                                                          \
  (kv.fmt == 0 ? launch_sparse<DD, 0>(a, cluster, c.stream)                     \
               : kv.fmt == 1 ? launch_sparse<DD, 1>(a, cluster, c.stream) : launch_sparse<DD, 2>(a, cluster, c.stream))
  if (D == 64) return Q35_SPARSE(64);
  if (D == 128) return Q35_SPARSE(128);
  return Q35_SPARSE(256);
#undef Q35_SPARSE
}

}  // namespace q35
