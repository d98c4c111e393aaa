// attn.key_mass: how much softmax weight a window of queries gives to every cached row.
//
// For the T queries of a sequence (its last T tokens, query t seeing the rows 0 .. ctx - T + t) and the G query heads of
// a KV head, with s_ti = q_t . k_i * scale and lse_t = log sum_i exp(s_ti):
//   key_mass_i (+)= sum_t sum_g exp(s_tgi - lse_tg).
// Two passes over the scores: the first finds lse of every query row, the second adds up columns.  The scores of a pass
// are not kept: T G values a row are more bytes than the row itself as soon as T G > D / 2.
//
// The query rows of a KV head are the G T pairs (token, head), 128 of them to a block, whatever G is.
// Pass 1 (mass_lse): CTA = 128 query rows x a range of keys; the rows' fragments stay in registers, 64-key tiles stream
// through shared memory; running maximum and sum per row, merged over the key ranges by mass_merge.
// Pass 2 (mass_sum): CTA = one 64-key tile, in shared memory once; the blocks of query rows that see it go past.  Every
// sum has one owner and a fixed order: no atomics.
#include "abi.h"
#include "attn_pages.cuh"
#include "kv_formats.cuh"

namespace q35 {

constexpr int KM_ROWS = 128;   // query rows per block, 16 per warp
constexpr int KM_KEYS = 64;    // keys per tile
constexpr float KM_LOG2E = 1.4426950408889634f;

struct MassArgs {
  PageTable t;
  const __nv_bfloat16* q;      // [T_total, HQ, D]
  const uint8_t* cache;
  const float* kv_scale;
  const __nv_bfloat16* row_scale;
  const int* qo_indptr;        // [B + 1]
  const float* sm_scale;       // optional [1]
  float* key_mass;             // [pages, P, HKV]
  float2* part;                // workspace [splits][HQ T_total]: maximum, sum
  float* lse;                  // workspace [HQ T_total]: log2 of the sum of 2^score
  int T_total, HQ, HKV, G, splits, accumulate, q_blocks, key_tiles;
};

// the window of sequence b: tokens q0 .. q0 + T - 1 of q, the first of them at position `first`; T = 0 if there is none
struct Window { int q0, T, first; };
__device__ __forceinline__ Window window_of(const MassArgs& a, int b, const SeqPages& sp) {
  const int q0 = a.qo_indptr[b], q1 = a.qo_indptr[b + 1];
  if (q0 < 0 || q1 < q0 || q1 > a.T_total || q1 - q0 > sp.ctx) {  // the cache must hold the window's own rows
    atomicOr(a.t.status, DS_BAD_TOKEN);
    return {0, 0, 0};
  }
  return {q0, q1 - q0, sp.ctx - (q1 - q0)};
}

// A tile of 64 rows of K as bf16 in shared memory, from registers loaded one tile ahead.  Chunk ch (8 channels) of row
// key lies at position ch ^ swz(key): eight lanes that read two rows' four neighbouring chunks hit all 32 banks.
__device__ __forceinline__ int km_swz(int key) { return (key & 1) << 2 | (key >> 1 & 3); }

template <int D, int KVF>
struct KTile {
  static constexpr int CPR = D * (KVF ? 1 : 2) / 16;       // 16-byte chunks of a stored row
  static constexpr int LD = KM_KEYS * CPR / 256;
  static constexpr int BYTES = KM_KEYS * D * 2;
  uint4 v[LD];
  float sc[LD];

  __device__ __forceinline__ void load(const MassArgs& a, const SeqPages& sp, int kvh, int k0) {
    bool bad = false;
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int i = threadIdx.x + 256 * j, key = i / CPR, ch = i % CPR, pos = k0 + key;
      v[j] = make_uint4(0u, 0u, 0u, 0u);  // rows behind the end: zeros (their scores are masked)
      sc[j] = 0.f;
      if (pos < sp.ctx) {
        const int page = page_or_first(a.t, sp.first + pos / a.t.P, bad);
        const size_t row = (size_t(page) * 2 * a.t.P + pos % a.t.P) * a.HKV + kvh;
        v[j] = *reinterpret_cast<const uint4*>(a.cache + (row * CPR + ch) * 16);
        if constexpr (KVF == 2) sc[j] = __bfloat162float(a.row_scale[row]);
      }
    }
    if (bad) atomicOr(a.t.status, DS_BAD_PAGE);
  }
  __device__ __forceinline__ void store(uint8_t* tile) const {
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int i = threadIdx.x + 256 * j, key = i / CPR, ch = i % CPR;
      uint4* row = reinterpret_cast<uint4*>(tile + key * D * 2);
      if constexpr (KVF == 0) {
        row[ch ^ km_swz(key)] = v[j];
      } else {
        const uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
        uint32_t o[8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if constexpr (KVF == 2) {
            o[2 * u] = cvt_s8x2_bf16x2<0, 1>(w[u] ^ 0x80808080u, sc[j], sc[j]);
            o[2 * u + 1] = cvt_s8x2_bf16x2<2, 3>(w[u] ^ 0x80808080u, sc[j], sc[j]);
          } else {  // E4M3 -> f16 -> bf16, exact
            const uint32_t f0 = cvt_kv<0, 1>(w[u]), f1 = cvt_kv<2, 3>(w[u]);
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&f0));
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&f1));
            o[2 * u] = pack_bf16(x.x, x.y);
            o[2 * u + 1] = pack_bf16(y.x, y.y);
          }
        }
        row[(2 * ch) ^ km_swz(key)] = make_uint4(o[0], o[1], o[2], o[3]);
        row[(2 * ch + 1) ^ km_swz(key)] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
};

// A warp's 16 query rows as MMA fragments.  Lane c of a row's four takes channels 8 c .. 8 c + 7 of every 32 (one 16-byte
// load); the key fragments are read the same way, so both sides agree on the order of k.
template <int D>
struct QRows {
  uint32_t f[D / 32][8];
  __device__ __forceinline__ void load(const MassArgs& a, const Window& w, int kvh, int row0, int rows) {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int m = row0 + r + 8 * half;
      const bool ok = m < rows;
      const int tok = ok ? m / a.G : 0, g = ok ? m % a.G : 0;
      const __nv_bfloat16* p = a.q + (size_t(w.q0 + tok) * a.HQ + size_t(kvh) * a.G + g) * D + 8 * c;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint4 v = ok ? *reinterpret_cast<const uint4*>(p + 32 * j) : make_uint4(0u, 0u, 0u, 0u);
        f[j][half] = v.x; f[j][2 + half] = v.y; f[j][4 + half] = v.z; f[j][6 + half] = v.w;
      }
    }
  }
  // s[nt][0, 1]: row r, keys 8 nt + 2 c, + 1; s[nt][2, 3]: row r + 8
  __device__ __forceinline__ void scores(const uint8_t* tile, float (&s)[8][4]) const {
    const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
#pragma unroll
      for (int nt = 0; nt < 8; ++nt) {
        const int key = nt * 8 + r;
        const uint4 k = *reinterpret_cast<const uint4*>(tile + key * D * 2 + (((4 * j + c) ^ km_swz(key)) << 4));
        mma_bf16_16816(s[nt], f[j][0], f[j][1], f[j][2], f[j][3], k.x, k.y);
        mma_bf16_16816(s[nt], f[j][4], f[j][5], f[j][6], f[j][7], k.z, k.w);
      }
    }
  }
};

__device__ __forceinline__ float mass_scale(const MassArgs& a, int kvh, int D, bool e4m3) {
  const float k_mul = !e4m3 ? 1.f : a.kv_scale ? a.kv_scale[kvh] : 0.125f;
  return (a.sm_scale ? a.sm_scale[0] : rsqrtf(float(D))) * KM_LOG2E * k_mul;
}

template <int D, int KVF>
__global__ void __launch_bounds__(256, 1) mass_lse_kernel(const MassArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int blk = blockIdx.x % a.q_blocks, bh = blockIdx.x / a.q_blocks, b = bh / a.HKV, kvh = bh % a.HKV;
  const int split = blockIdx.y;
  const SeqPages sp = seq_pages(a.t, b);
  const Window w = window_of(a, b, sp);
  const int rows = w.T * a.G;
  const float scale = mass_scale(a, kvh, D, KVF == 1);
  for (int row0 = blk * KM_ROWS; row0 < rows; row0 += a.q_blocks * KM_ROWS) {
    // keys that the block's last row sees, cut into a.splits ranges of whole tiles
    const int last_row = min(row0 + KM_ROWS, rows) - 1, n_keys = w.first + last_row / a.G + 1;
    const int tiles = (n_keys + KM_KEYS - 1) / KM_KEYS, per = (tiles + a.splits - 1) / a.splits;
    const int t0 = min(tiles, split * per), t1 = min(tiles, t0 + per);
    QRows<D> q;
    q.load(a, w, kvh, row0 + warp * 16, rows);
    const int m0 = row0 + warp * 16 + r, m1 = m0 + 8;
    const int see0 = w.first + m0 / a.G, see1 = w.first + m1 / a.G;  // last key of each row
    float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    KTile<D, KVF> next;
    if (t0 < t1) next.load(a, sp, kvh, t0 * KM_KEYS);
    for (int t = t0; t < t1; ++t) {
      __syncthreads();
      next.store(smem);
      __syncthreads();
      if (t + 1 < t1) next.load(a, sp, kvh, (t + 1) * KM_KEYS);
      float s[8][4];
      q.scores(smem, s);
      float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = t * KM_KEYS + nt * 8 + 2 * c + (i & 1);
          s[nt][i] = key <= (i >> 1 ? see1 : see0) ? s[nt][i] * scale : -INFINITY;
          top[i >> 1] = fmaxf(top[i >> 1], s[nt][i]);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        const float mn = fmaxf(mx[h], top[h]), base = mn == -INFINITY ? 0.f : mn;
        float sum = 0.f;
#pragma unroll
        for (int nt = 0; nt < 8; ++nt) sum += exp2f(s[nt][2 * h] - base) + exp2f(s[nt][2 * h + 1] - base);
        l[h] = l[h] * exp2f(mx[h] - base) + sum;
        mx[h] = mn;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int m = h ? m1 : m0;
      if (c == 0 && m < rows) {
        const size_t at = size_t(w.q0 + m / a.G) * a.HQ + size_t(kvh) * a.G + m % a.G;
        a.part[size_t(split) * a.T_total * a.HQ + at] = make_float2(mx[h], l[h]);
      }
    }
  }
}

// lse of every query row from its key ranges; a row with no weight at all (every score -inf) gives +inf: no weight
__global__ void __launch_bounds__(256) mass_merge_kernel(const MassArgs a) {
  pdl_wait();
  pdl_launch();
  const size_t n = size_t(a.T_total) * a.HQ;
  for (size_t i = size_t(blockIdx.x) * 256 + threadIdx.x; i < n; i += size_t(gridDim.x) * 256) {
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part[s * n + i].x);
    const float base = m == -INFINITY ? 0.f : m;
    for (int s = 0; s < a.splits; ++s) {
      const float2 p = a.part[s * n + i];
      l += p.y * exp2f(p.x - base);
    }
    a.lse[i] = l == 0.f ? INFINITY : base + log2f(l);
  }
}

template <int D, int KVF>
__global__ void __launch_bounds__(256, 1) mass_sum_kernel(const MassArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_sum[8][KM_KEYS];
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int bh = blockIdx.x / a.key_tiles, b = bh / a.HKV, kvh = bh % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  const Window w = window_of(a, b, sp);
  const int rows = w.T * a.G;
  if (rows == 0 && a.accumulate) return;
  const float scale = mass_scale(a, kvh, D, KVF == 1);
  for (int tile = blockIdx.x % a.key_tiles; tile * KM_KEYS < sp.ctx; tile += a.key_tiles) {
    const int k0 = tile * KM_KEYS;
    __syncthreads();
    {
      KTile<D, KVF> k;
      k.load(a, sp, kvh, k0);
      k.store(smem);
    }
    __syncthreads();
    float col[8][2];
#pragma unroll
    for (int nt = 0; nt < 8; ++nt) col[nt][0] = col[nt][1] = 0.f;
    // the first query row that sees key k0 belongs to token k0 - w.first
    const int from = max(0, k0 - w.first) * a.G / KM_ROWS * KM_ROWS;
    for (int row0 = from; row0 < rows; row0 += KM_ROWS) {
      QRows<D> q;
      q.load(a, w, kvh, row0 + warp * 16, rows);
      const int m0 = row0 + warp * 16 + r, m1 = m0 + 8;
      auto lse = [&](int m) {
        return m < rows ? a.lse[size_t(w.q0 + m / a.G) * a.HQ + size_t(kvh) * a.G + m % a.G] : INFINITY;
      };
      const float l0 = lse(m0), l1 = lse(m1);
      const int see0 = m0 < rows ? w.first + m0 / a.G : -1, see1 = m1 < rows ? w.first + m1 / a.G : -1;
      float s[8][4];
      q.scores(smem, s);
#pragma unroll
      for (int nt = 0; nt < 8; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = k0 + nt * 8 + 2 * c + i;
          if (key <= see0) col[nt][i] += exp2f(s[nt][i] * scale - l0);
          if (key <= see1) col[nt][i] += exp2f(s[nt][2 + i] * scale - l1);
        }
    }
#pragma unroll
    for (int nt = 0; nt < 8; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) col[nt][i] += __shfl_xor_sync(0xffffffffu, col[nt][i], o);
        if (r == 0) s_sum[warp][nt * 8 + 2 * c + i] = col[nt][i];
      }
    __syncthreads();
    if (threadIdx.x < KM_KEYS && k0 + int(threadIdx.x) < sp.ctx) {
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += s_sum[u][threadIdx.x];
      const int pos = k0 + threadIdx.x, page = page_at(a.t, sp.first + pos / a.t.P);
      if (page >= 0) {
        float* dst = a.key_mass + (size_t(page) * a.t.P + pos % a.t.P) * a.HKV + kvh;
        *dst = a.accumulate ? *dst + sum : sum;
      }
    }
  }
}

template <int D, int KVF>
static int launch_mass(const MassArgs& a, cudaStream_t stream) {
  const int smem = KTile<D, KVF>::BYTES;
  const unsigned heads = unsigned(a.t.B) * a.HKV;
  if (a.T_total > 0) {
    launch_pdl(mass_lse_kernel<D, KVF>, dim3(heads * a.q_blocks, unsigned(a.splits)), dim3(256), smem, stream, a);
    Q35_CUDA_LAUNCH_CHECK("attn.key_mass rows");
    const int64_t n = int64_t(a.T_total) * a.HQ, blocks = (n + 255) / 256;
    launch_pdl(mass_merge_kernel, dim3(unsigned(blocks < 1024 ? blocks : 1024)), dim3(256), 0, stream, a);
    Q35_CUDA_LAUNCH_CHECK("attn.key_mass merge");
  }
  launch_pdl(mass_sum_kernel<D, KVF>, dim3(heads * a.key_tiles), dim3(256), smem, stream, a);
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
  Q35_REQUIRE(B >= 0 && mass.numel() == kv.pages * P * HKV, Q35_ERR_SHAPE, "%s: qo_indptr [B + 1], key_mass [pages, P, HKV]",
              role);
  Q35_REQUIRE(!scale.present || scale.numel() == 1, Q35_ERR_SHAPE, "%s: sm_scale [1]", role);
  Q35_REQUIRE(T * HQ <= INT_MAX / 2 && B * HKV <= INT_MAX / 1024, Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  MassArgs a{};
  Q35_TRY(get_page_table(c, role, B, P, kv.pages, &a.t));
  // pass 1 fills the GPU from (sequence, KV head) x blocks of query rows x ranges of keys
  const int64_t heads = B * HKV, rows = B ? (T * (HQ / HKV) + B - 1) / B : 0;
  const int64_t keys = B ? (int64_t(a.t.n_indices) * P + B - 1) / B : 0;
  int64_t qb = (rows + KM_ROWS - 1) / KM_ROWS;
  if (qb < 1) qb = 1;
  const int64_t tiles = (keys + KM_KEYS - 1) / KM_KEYS;
  int64_t splits = heads ? 2 * sm_count() / (heads * qb) : 1;
  if (splits > tiles / 2) splits = tiles / 2;
  if (splits < 1) splits = 1;
  if (splits > 64) splits = 64;
  a.q_blocks = int(qb); a.splits = int(splits); a.key_tiles = int(tiles < 1 ? 1 : tiles);
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = (off + bytes + 255) / 256 * 256; return o; };
  const int64_t o_part = take(splits * T * HQ * 8), o_lse = take(T * HQ * 4);
  Q35_TRY(c.workspace(off, &ws));
  if (c.dry || B == 0) return 0;
  Q35_REQUIRE(aligned16(q.p), Q35_ERR_ALIGN, "%s: q must be 16-byte aligned", role);
  Q35_REQUIRE(heads * a.key_tiles <= INT_MAX && heads * qb <= INT_MAX, Q35_ERR_UNSUPPORTED, "%s: sizes beyond 32 bits", role);
  a.q = q.as<__nv_bfloat16>(); a.cache = static_cast<const uint8_t*>(kv.p);
  a.kv_scale = kv.kv_scale; a.row_scale = kv.row_scale;
  a.qo_indptr = qo.as<int>();
  a.sm_scale = scale.present ? scale.as<float>() : nullptr;
  a.key_mass = mass.as<float>();
  uint8_t* w = ws.as<uint8_t>();
  a.part = reinterpret_cast<float2*>(w + o_part);
  a.lse = reinterpret_cast<float*>(w + o_lse);
  a.T_total = int(T); a.HQ = int(HQ); a.HKV = int(HKV); a.G = int(HQ / HKV);
  a.accumulate = acc.present;
#define Q35_MASS(DD) \
  (kv.fmt == 0 ? launch_mass<DD, 0>(a, c.stream) : kv.fmt == 1 ? launch_mass<DD, 1>(a, c.stream) : launch_mass<DD, 2>(a, c.stream))
  if (D == 64) return Q35_MASS(64);
  if (D == 128) return Q35_MASS(128);
  return Q35_MASS(256);
#undef Q35_MASS
}

}  // namespace q35
