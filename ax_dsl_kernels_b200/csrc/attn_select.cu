// Choosing the pages a query attends to: attn.page_bounds (what the keys of a page can be) and attn.select_pages (the
// pages whose keys can score highest).
//
// For a page with keys k_1 .. k_m let lo_d = min_i k_id and hi_d = max_i k_id.  Then q . k_i <= sum_d max(q_d lo_d,
// q_d hi_d) for every key of the page, and the right side costs 1 / (P / 2) of the products with all P keys.  A KV head
// is shared by G query heads, so a page's score is the maximum of the G bounds.
#include "abi.h"
#include "attn_pages.cuh"
#include "kv_formats.cuh"

namespace q35 {

// ---------------------------------------------------------------------------------------------------------------
// attn.page_bounds.  Bound: HBM (the K rows are read once, the bounds are 2 / P of them).  The K rows of a page are one
// contiguous block [P, HKV * D], so a CTA takes a page: thread = one 16-byte column chunk, the rows dealt to 256 / chunks
// row groups whose results meet in shared memory.  minimum and maximum are exact in the stored format: E4M3 codes as
// f16, int8 rows as the bf16 values bf16(int8 * scale).  A NaN in a valid row makes that channel's bounds NaN.
struct BoundsArgs {
  PageTable t;
  const uint8_t* cache;
  const __nv_bfloat16* row_scale;
  const int* first_page;   // optional [B]: pages before it are left as they are
  __nv_bfloat16* out;      // [pages, 2, HKV, D]
  int HKV, D;
  int per_seq;             // 0: CTA = table entry; > 0: that many CTAs per sequence walk its pages from first_page
};

template <int KVF> struct Pair { using T = __nv_bfloat162; };
template <> struct Pair<1> { using T = __half2; };

template <int KVF>
__device__ __forceinline__ typename Pair<KVF>::T bits_pair(uint32_t u) {
  return *reinterpret_cast<typename Pair<KVF>::T*>(&u);
}

template <int KVF>
__device__ __forceinline__ void page_bounds_one(const BoundsArgs& a, int page, int valid, uint4* s_red) {
  using T = typename Pair<KVF>::T;
  constexpr int NP = KVF == 0 ? 4 : 8;  // channel pairs per 16-byte chunk
  const int tid = threadIdx.x;
  const int row_bytes = a.HKV * a.D * (KVF == 0 ? 2 : 1), chunks = row_bytes / 16;
  const uint8_t* rows = a.cache + size_t(page) * 2 * a.t.P * row_bytes;
  const uint32_t inf2 = KVF == 1 ? 0x7C007C00u : 0x7F807F80u;  // +inf, +inf
  for (int c0 = 0; c0 < chunks; c0 += 256) {
    const int nc = min(256, chunks - c0), groups = 256 / nc;
    const int ch = tid % nc, grp = tid / nc;
    T lo[NP], hi[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      lo[i] = bits_pair<KVF>(inf2);
      hi[i] = bits_pair<KVF>(inf2 | 0x80008000u);
    }
    if (grp < groups) {
      const uint8_t* col = rows + (c0 + ch) * 16;
      const int head = (c0 + ch) * 16 / a.D;  // one-byte formats: 16 channels of one head
      constexpr int U = 8;                     // rows in flight per thread
      for (int r0 = grp; r0 < valid; r0 += groups * U) {
        uint4 v[U];
        float sc[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * groups;
          if (r < valid) {
            v[u] = ldg_nc_16(col + size_t(r) * row_bytes);
            if constexpr (KVF == 2)
              sc[u] = __bfloat162float(a.row_scale[(size_t(page) * 2 * a.t.P + r) * a.HKV + head]);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (r0 + u * groups >= valid) break;
          const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if constexpr (KVF == 0) {
              const T x = bits_pair<KVF>(w[j]);
              lo[j] = __hmin2_nan(lo[j], x);
              hi[j] = __hmax2_nan(hi[j], x);
            } else {
              uint32_t p0, p1;
              if constexpr (KVF == 1) {
                p0 = cvt_kv<0, 1>(w[j]);
                p1 = cvt_kv<2, 3>(w[j]);
              } else {
                p0 = cvt_s8x2_bf16x2<0, 1>(w[j] ^ 0x80808080u, sc[u], sc[u]);
                p1 = cvt_s8x2_bf16x2<2, 3>(w[j] ^ 0x80808080u, sc[u], sc[u]);
              }
              lo[2 * j] = __hmin2_nan(lo[2 * j], bits_pair<KVF>(p0));
              hi[2 * j] = __hmax2_nan(hi[2 * j], bits_pair<KVF>(p0));
              lo[2 * j + 1] = __hmin2_nan(lo[2 * j + 1], bits_pair<KVF>(p1));
              hi[2 * j + 1] = __hmax2_nan(hi[2 * j + 1], bits_pair<KVF>(p1));
            }
          }
        }
      }
    }
    uint4* mine = s_red + tid * (NP / 2);
#pragma unroll
    for (int i = 0; i < NP / 4; ++i) {
      mine[i] = reinterpret_cast<const uint4*>(lo)[i];
      mine[NP / 4 + i] = reinterpret_cast<const uint4*>(hi)[i];
    }
    __syncthreads();
    // column chunk ch, half h (0 = minimum, 1 = maximum): one thread folds the groups and writes the channels
    for (int idx = tid; idx < nc * 2; idx += 256) {
      const int c = idx >> 1, h = idx & 1;
      T acc[NP];
#pragma unroll
      for (int i = 0; i < NP / 4; ++i) reinterpret_cast<uint4*>(acc)[i] = s_red[c * (NP / 2) + h * (NP / 4) + i];
      for (int g = 1; g < groups; ++g) {
        T o[NP];
#pragma unroll
        for (int i = 0; i < NP / 4; ++i)
          reinterpret_cast<uint4*>(o)[i] = s_red[(g * nc + c) * (NP / 2) + h * (NP / 4) + i];
#pragma unroll
        for (int i = 0; i < NP; ++i) acc[i] = h ? __hmax2_nan(acc[i], o[i]) : __hmin2_nan(acc[i], o[i]);
      }
      uint32_t w[NP];
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (KVF == 1) {
          const float2 f = __half22float2(acc[i]);
          w[i] = pack_bf16(f.x, f.y);
        } else {
          w[i] = *reinterpret_cast<const uint32_t*>(&acc[i]);
        }
      }
      __nv_bfloat16* dst = a.out + (size_t(page) * 2 + h) * a.HKV * a.D + size_t(c0 + c) * (2 * NP);
#pragma unroll
      for (int i = 0; i < NP / 4; ++i)
        reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
    __syncthreads();
  }
}

template <int KVF>
__global__ void __launch_bounds__(256) page_bounds_kernel(const BoundsArgs a) {
  pdl_wait();
  pdl_launch();
  __shared__ uint4 s_red[256 * (KVF == 0 ? 2 : 4)];
  if (a.per_seq == 0) {
    const int e = blockIdx.x;  // the sequence of entry e: the last b with indptr[b] <= e
    int lo = 0, hi = a.t.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.t.indptr[mid] <= e) lo = mid; else hi = mid;
    }
    const SeqPages sp = seq_pages(a.t, lo);
    const int i = e - sp.first;
    if (i < 0 || i >= sp.n) return;
    const int page = page_at(a.t, e);
    if (page >= 0) page_bounds_one<KVF>(a, page, min(a.t.P, sp.ctx - i * a.t.P), s_red);
    return;
  }
  const int b = blockIdx.x / a.per_seq;
  const SeqPages sp = seq_pages(a.t, b);
  for (int i = max(0, a.first_page[b]) + int(blockIdx.x) % a.per_seq; i < sp.n; i += a.per_seq) {
    const int page = page_at(a.t, sp.first + i);
    if (page >= 0) page_bounds_one<KVF>(a, page, min(a.t.P, sp.ctx - i * a.t.P), s_red);
  }
}

int run_attn_page_bounds(Call& c) {
  const char* role = "attn.page_bounds";
  KvCache kv;
  Q35_TRY(get_kv_cache(c, role, &kv));
  Tensor first, out, indptr;
  Q35_TRY(c.get("indptr", M(Q35_I32), &indptr));
  Q35_TRY(c.get("first_page", M(Q35_I32), &first, false));
  Q35_TRY(c.get("page_bounds", M(Q35_BF16), &out));
  const int64_t B = indptr.numel() - 1;
  Q35_REQUIRE(B >= 0 && B <= INT_MAX / 4, Q35_ERR_SHAPE, "%s: indptr [B + 1]", role);
  BoundsArgs a{};
  Q35_TRY(get_page_table(c, role, B, kv.P, kv.pages, &a.t));
  Q35_REQUIRE(kv.D % 16 == 0, Q35_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 16", role);
  Q35_REQUIRE(kv.fmt != 1 || !kv.kv_scale, Q35_ERR_UNSUPPORTED,
              "%s: the bounds of an E4M3 cache are those of its stored codes; kv_scale does not enter", role);
  Q35_REQUIRE(out.nd == 4 && out.s[0] == kv.pages && out.s[1] == 2 && out.s[2] == kv.HKV && out.s[3] == kv.D,
              Q35_ERR_SHAPE, "%s: page_bounds [pages, 2, HKV, D]", role);
  Q35_REQUIRE(!first.present || first.numel() >= B, Q35_ERR_SHAPE, "%s: first_page [B]", role);
  c.ws_need = 0;
  if (c.dry || B == 0 || a.t.n_indices == 0) return 0;
  Q35_REQUIRE(aligned16(out.p), Q35_ERR_ALIGN, "%s: page_bounds must be 16-byte aligned", role);
  a.cache = static_cast<const uint8_t*>(kv.p); a.row_scale = kv.row_scale;
  a.first_page = first.present ? first.as<int>() : nullptr;
  a.out = out.as<__nv_bfloat16>(); a.HKV = int(kv.HKV); a.D = int(kv.D);
  // A decode step passes first_page and has a page or two per sequence to do: a CTA per table entry would be thousands
  // of CTAs that only look.  There, a few CTAs per sequence (enough to fill the GPU twice) walk from first_page on.
  if (first.present) {
    const int64_t avg = (a.t.n_indices + B - 1) / B, fill = (4 * sm_count() + B - 1) / B;
    a.per_seq = int(avg < fill ? avg : fill);
  }
  const unsigned grid = unsigned(first.present ? B * a.per_seq : a.t.n_indices);
  if (kv.fmt == 0) launch_pdl(page_bounds_kernel<0>, dim3(grid), dim3(256), 0, c.stream, a);
  else if (kv.fmt == 1) launch_pdl(page_bounds_kernel<1>, dim3(grid), dim3(256), 0, c.stream, a);
  else launch_pdl(page_bounds_kernel<2>, dim3(grid), dim3(256), 0, c.stream, a);
  Q35_CUDA_LAUNCH_CHECK("attn.page_bounds");
  return 0;
}

// ---------------------------------------------------------------------------------------------------------------
// attn.select_pages: the S best pages of every (sequence, KV head), ties to the lower page, the first and the last ones
// always, in ascending order.
//
// The order of the scores decides, and two summation orders of the same bf16 products can disagree about two close
// pages.  So the scores are found twice: sum_d max(q_d lo_d, q_d hi_d) = max(q, 0) . hi + min(q, 0) . lo is a product
// of bf16 rows that the tensor cores do for all heads at once in fp32, with an error of at most n 2^-23 sum |terms| for
// any order of n = 2 D terms; and the few pages within that error of the border (usually one to ten) are scored again
// in fp64, where the sum of 512 products of 16 significant bits is as good as exact.
// Bound: HBM for the bounds (each read once); at one sequence the launch and the chain of the selection.
struct SelectArgs {
  const __nv_bfloat16* q;       // [B, HQ, D]
  const __nv_bfloat16* bounds;  // [pages, 2, HKV, D]
  PageTable t;                  // P unused
  const int* keep;              // optional [2]: first, last
  int* out;                     // [B, HKV, S]
  int HQ, HKV, G, D, S, gx;
  // workspace, [HKV * n_indices] each: entries of (b, kvh) start at HKV * indptr[b] + kvh * n
  float2* score;                // score and its error bound
  double* zscore;               // fp64 scores of the zone
  int* zone;                    // pages of the zone
  uint8_t* flag;                // 0 out, 1 in, 2 zone
};

// pages of sequence b that hold a row, without knowing P
__device__ __forceinline__ int2 select_range(const SelectArgs& a, int b) {
  const int lo = a.t.indptr[b], hi = a.t.indptr[b + 1];
  if (lo < 0 || hi < lo || hi > a.t.n_indices) {
    atomicOr(a.t.status, DS_BAD_PAGE);
    return make_int2(0, 0);
  }
  return make_int2(lo, hi - lo - (hi > lo && a.t.last_page_len[b] <= 0 ? 1 : 0));
}
__device__ __forceinline__ int select_page(const SelectArgs& a, int e) {
  const int id = page_at(a.t, e);
  return id < 0 ? 0 : id;
}
__device__ __forceinline__ uint32_t pos_pair(uint32_t x) {
  __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t neg_pair(uint32_t x) {
  __nv_bfloat162 v = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float max_nan(float x, float y) { return x != x ? x : y != y ? y : fmaxf(x, y); }

// One warp scores 16 pages: A = the pages' hi and lo rows, B = max(q, 0) and min(q, 0) of 8 heads.  Both operands take
// their k index from 16-byte loads (lane c of a row's four holds channels 8 c .. 8 c + 7 of every 32), so the fragments
// come straight from global memory and a row is read in full sectors.
template <int D>
__global__ void __launch_bounds__(128) select_score_kernel(const SelectArgs a) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int row = blockIdx.x / a.gx, b = row / a.HKV, h = row % a.HKV;
  const int2 rg = select_range(a, b);
  const int n = rg.y;
  const size_t base = size_t(a.HKV) * rg.x + size_t(h) * n;
  for (int p0 = ((blockIdx.x % a.gx) * 4 + warp) * 16; p0 < n; p0 += a.gx * 64) {
    const int i0 = min(p0 + r, n - 1), i1 = min(p0 + r + 8, n - 1);
    const size_t plane = size_t(a.HKV) * D;
    const __nv_bfloat16* lo0 = a.bounds + size_t(select_page(a, rg.x + i0)) * 2 * plane + size_t(h) * D + 8 * c;
    const __nv_bfloat16* lo1 = a.bounds + size_t(select_page(a, rg.x + i1)) * 2 * plane + size_t(h) * D + 8 * c;
    float best0 = -INFINITY, best1 = -INFINITY, q1max = 0.f, kmax0 = 0.f, kmax1 = 0.f;
    for (int g0 = 0; g0 < a.G; g0 += 8) {
      const bool hv = g0 + r < a.G;
      const __nv_bfloat16* qp = a.q + (size_t(b) * a.HQ + size_t(h) * a.G + (hv ? g0 + r : 0)) * D + 8 * c;
      float ap[4] = {0.f, 0.f, 0.f, 0.f}, an[4] = {0.f, 0.f, 0.f, 0.f};
      float q1 = 0.f;
      uint32_t km0 = 0u, km1 = 0u;
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        const uint4 l0 = ldg_nc_16(lo0 + j * 32), l1 = ldg_nc_16(lo1 + j * 32);
        const uint4 h0 = ldg_nc_16(lo0 + plane + j * 32), h1 = ldg_nc_16(lo1 + plane + j * 32);
        uint4 qv = make_uint4(0u, 0u, 0u, 0u);
        if (hv) qv = *reinterpret_cast<const uint4*>(qp + j * 32);
        mma_bf16_16816(ap, h0.x, h1.x, h0.y, h1.y, pos_pair(qv.x), pos_pair(qv.y));
        mma_bf16_16816(an, l0.x, l1.x, l0.y, l1.y, neg_pair(qv.x), neg_pair(qv.y));
        mma_bf16_16816(ap, h0.z, h1.z, h0.w, h1.w, pos_pair(qv.z), pos_pair(qv.w));
        mma_bf16_16816(an, l0.z, l1.z, l0.w, l1.w, neg_pair(qv.z), neg_pair(qv.w));
        const uint32_t qw[4] = {qv.x, qv.y, qv.z, qv.w};
        const uint32_t w0[8] = {l0.x, l0.y, l0.z, l0.w, h0.x, h0.y, h0.z, h0.w};
        const uint32_t w1[8] = {l1.x, l1.y, l1.z, l1.w, h1.x, h1.y, h1.z, h1.w};
#pragma unroll
        for (int u = 0; u < 4; ++u) q1 += fabsf(bf16lo(qw[u])) + fabsf(bf16hi(qw[u]));
#pragma unroll
        for (int u = 0; u < 8; ++u) {  // largest magnitude of the rows' bounds: bf16 magnitudes order as integers
          km0 = __vmaxu2(km0, w0[u] & 0x7fff7fffu);
          km1 = __vmaxu2(km1, w1[u] & 0x7fff7fffu);
        }
      }
      q1 += __shfl_xor_sync(0xffffffffu, q1, 1);
      q1 += __shfl_xor_sync(0xffffffffu, q1, 2);
      q1max = fmaxf(q1max, q1);  // of head r of this block of heads; over the heads below
      kmax0 = fmaxf(kmax0, fmaxf(bf16lo(km0), bf16hi(km0)));
      kmax1 = fmaxf(kmax1, fmaxf(bf16lo(km1), bf16hi(km1)));
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (g0 + 2 * c + u < a.G) {
          best0 = max_nan(best0, ap[u] + an[u]);
          best1 = max_nan(best1, ap[2 + u] + an[2 + u]);
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      best0 = max_nan(best0, __shfl_xor_sync(0xffffffffu, best0, o));
      best1 = max_nan(best1, __shfl_xor_sync(0xffffffffu, best1, o));
      kmax0 = fmaxf(kmax0, __shfl_xor_sync(0xffffffffu, kmax0, o));
      kmax1 = fmaxf(kmax1, __shfl_xor_sync(0xffffffffu, kmax1, o));
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) q1max = fmaxf(q1max, __shfl_xor_sync(0xffffffffu, q1max, o));
    if (c == 0) {  // 2 D terms of at most |q|_1 kmax in all: an error of 2 D 2^-23 of that at most
      const float rel = 2.f * D / 8388608.f;
      if (p0 + r < n) a.score[base + p0 + r] = make_float2(best0, q1max * kmax0 * rel);
      if (p0 + r + 8 < n) a.score[base + p0 + r + 8] = make_float2(best1, q1max * kmax1 * rel);
    }
  }
}

__device__ __forceinline__ unsigned long long order_key64(double x) {
  if (x != x) x = -INFINITY;
  const unsigned long long u = __double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// The r-th largest (r >= 1) of key(0 .. n - 1), digit by digit from the top: a histogram of the digits of the keys that
// agree with the prefix so far, then the digit in which the rank falls.  above = how many keys are larger.
template <typename K, typename F>
__device__ K block_kth_largest(F key, int n, int r, int* hist, int* above) {
  __shared__ int s_digit, s_rank;
  K prefix = 0;
  int rank = r;
  for (int shift = int(sizeof(K)) * 8 - 8; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const K k = key(i);
      if (shift == int(sizeof(K)) * 8 - 8 || ((k ^ prefix) >> (shift + 8)) == 0) atomicAdd(&hist[int(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {  // lane l sums the digits 255 - 8 l .. 248 - 8 l, then the warp scans from the top
      const int l = threadIdx.x;
      int sum = 0;
      for (int u = 0; u < 8; ++u) sum += hist[255 - 8 * l - u];
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (l >= o) inc += v;
      }
      int before = inc - sum;
      if (before < rank && rank <= inc) {
        for (int u = 0; u < 8; ++u) {
          const int cnt = hist[255 - 8 * l - u];
          if (rank <= before + cnt) {
            s_digit = 255 - 8 * l - u;
            s_rank = rank - before;
            break;
          }
          before += cnt;
        }
      }
    }
    __syncthreads();
    prefix |= K(s_digit) << shift;
    rank = s_rank;
    __syncthreads();
  }
  *above = r - rank;
  return prefix;
}

constexpr int SEL_THREADS = 1024;

// one CTA per (sequence, KV head): the choice
template <int D>
__global__ void __launch_bounds__(SEL_THREADS) select_choose_kernel(const SelectArgs a) {
  pdl_wait();
  pdl_launch();
  __shared__ int s_hist[256];
  __shared__ int s_scan[32];
  __shared__ float s_max[32];
  __shared__ int s_zone;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x, b = row / a.HKV, h = row % a.HKV;
  const int2 rg = select_range(a, b);
  const int n = rg.y, S = a.S;
  int* out = a.out + size_t(row) * S;
  if (n <= S) {
    for (int i = tid; i < S; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const size_t base = size_t(a.HKV) * rg.x + size_t(h) * n;
  const float2* score = a.score + base;
  uint8_t* flag = a.flag + base;
  int last = a.keep ? min(max(a.keep[1], 0), S) : 0;
  const int first = a.keep ? min(max(a.keep[0], 0), S - last) : 0;
  const int m = n - first - last, rank = S - first - last;  // rank of the m free pages; rank < m because S < n
  // largest error bound of a free page (inf and NaN: every page is scored again)
  float e = 0.f;
  for (int i = tid; i < m; i += SEL_THREADS) e = max_nan(e, score[first + i].y);
#pragma unroll
  for (int o = 16; o; o >>= 1) e = max_nan(e, __shfl_xor_sync(0xffffffffu, e, o));
  if (lane == 0) s_max[warp] = e;
  if (tid == 0) s_zone = 0;
  __syncthreads();
  e = s_max[0];
  for (int w = 1; w < 32; ++w) e = max_nan(e, s_max[w]);
  const bool all = !(e < INFINITY);
  int in = 0;  // pages certainly chosen
  if (rank > 0) {
    int above;
    const uint32_t kth = block_kth_largest<uint32_t>([&](int i) { return order_key(score[first + i].x); }, m, rank, s_hist,
                                                     &above);
    // the rank-th score as a float again; a true score differs from its fp32 one by e at most, so does the border
    const float tau = __uint_as_float(kth & 0x80000000u ? kth & 0x7fffffffu : ~kth);
    const float top = tau + 2.f * e, low = tau - 2.f * e;
    for (int i = tid; i < m; i += SEL_THREADS) {
      const float s = score[first + i].x;
      int f;
      if (all || !(s > top || s < low)) {
        f = 2;
        a.zone[base + atomicAdd(&s_zone, 1)] = first + i;
      } else {
        f = s > top;
        in += f;
      }
      flag[first + i] = uint8_t(f);
    }
    for (int o = 16; o; o >>= 1) in += __shfl_xor_sync(0xffffffffu, in, o);
    if (lane == 0) s_scan[warp] = in;
    __syncthreads();
    in = 0;
    for (int w = 0; w < 32; ++w) in += s_scan[w];
    const int z = s_zone, need = rank - in;  // need <= z: the zone holds the border
    const size_t plane = size_t(a.HKV) * D;
    for (int j = warp; j < z; j += 32) {
      const int i = a.zone[base + j];
      const __nv_bfloat16* lo = a.bounds + size_t(select_page(a, rg.x + i)) * 2 * plane + size_t(h) * D;
      double best = -INFINITY;
      bool nan = false;
      for (int g = 0; g < a.G; ++g) {
        const __nv_bfloat16* qp = a.q + (size_t(b) * a.HQ + size_t(h) * a.G + g) * D;
        double sum = 0.;
        for (int d = lane; d < D; d += 32) {
          const float q = __bfloat162float(qp[d]);
          const float qpos = q != q ? q : fmaxf(q, 0.f), qneg = q != q ? q : fminf(q, 0.f);
          sum += double(qpos) * double(__bfloat162float(lo[plane + d])) + double(qneg) * double(__bfloat162float(lo[d]));
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        nan |= sum != sum;
        best = fmax(best, sum);
      }
      if (lane == 0) a.zscore[base + i] = nan ? -INFINITY : best;
    }
    __syncthreads();
    const int* zone = a.zone + base;
    const double* zs = a.zscore + base;
    if (z <= 2048) {  // each page of the zone counts the pages that go before it
      for (int j = tid; j < z; j += SEL_THREADS) {
        const int i = zone[j];
        const double s = zs[i];
        int before = 0;
        for (int k = 0; k < z; ++k) {
          const int i2 = zone[k];
          const double s2 = zs[i2];
          before += s2 > s || (s2 == s && i2 < i);
        }
        flag[i] = before < need;
      }
    } else {  // pages that hardly differ: the border by digits, equal ones by index below
      int above64;
      const unsigned long long k64 = block_kth_largest<unsigned long long>(
          [&](int j) { return order_key64(zs[zone[j]]); }, z, need, s_hist, &above64);
      for (int j = tid; j < z; j += SEL_THREADS) {
        const int i = zone[j];
        const unsigned long long k = order_key64(zs[i]);
        flag[i] = k > k64 ? 1 : k < k64 ? 0 : 2;
      }
      __syncthreads();
      // of the pages equal to the border (flag 2) the first need - above64 in order
      int left = need - above64;
      for (int i0 = 0; i0 < m; i0 += SEL_THREADS) {
        const int i = first + i0 + tid;
        const bool eq = i0 + tid < m && flag[i] == 2;
        const unsigned ball = __ballot_sync(0xffffffffu, eq);
        if (lane == 0) s_scan[warp] = __popc(ball);
        __syncthreads();
        int before = __popc(ball & ((1u << lane) - 1)), total = 0;
        for (int w = 0; w < 32; ++w) {
          if (w < warp) before += s_scan[w];
          total += s_scan[w];
        }
        if (eq) flag[i] = before < left;
        left = max(0, left - total);
        __syncthreads();
      }
    }
    __syncthreads();
  }
  // ascending output: the first pages, the chosen ones, the last ones
  int at = 0;
  for (int i0 = 0; i0 < n; i0 += SEL_THREADS) {
    const int i = i0 + tid;
    const bool take = i < n && (i < first || i >= n - last || (rank > 0 && flag[i] == 1));
    const unsigned ball = __ballot_sync(0xffffffffu, take);
    if (lane == 0) s_scan[warp] = __popc(ball);
    __syncthreads();
    int pos = at + __popc(ball & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) pos += s_scan[w];
      total += s_scan[w];
    }
    if (take && pos < S) out[pos] = i;
    at += total;
    __syncthreads();
  }
}

int run_attn_select_pages(Call& c) {
  const char* role = "attn.select_pages";
  Tensor q, bounds, keep, out, ws;
  Q35_TRY(c.get("q", M(Q35_BF16), &q));
  Q35_TRY(c.get("page_bounds", M(Q35_BF16), &bounds));
  Q35_TRY(c.get("keep", M(Q35_I32), &keep, false));
  Q35_TRY(c.get("pages", M(Q35_I32), &out));
  Q35_REQUIRE(q.nd == 3 && bounds.nd == 4 && bounds.s[1] == 2 && out.nd == 3, Q35_ERR_SHAPE,
              "%s: q [B, HQ, D], page_bounds [pages, 2, HKV, D], pages [B, HKV, S]", role);
  const int64_t B = q.s[0], HQ = q.s[1], D = q.s[2], HKV = bounds.s[2], S = out.s[2];
  Q35_REQUIRE(bounds.s[3] == D && HKV >= 1 && HQ >= 1 && HQ % HKV == 0, Q35_ERR_SHAPE, "%s: head shapes", role);
  Q35_REQUIRE(D == 64 || D == 128 || D == 256, Q35_ERR_UNSUPPORTED, "%s: head_dim must be 64/128/256", role);
  Q35_REQUIRE(out.s[0] == B && out.s[1] == HKV && S >= 1 && S <= INT_MAX, Q35_ERR_SHAPE, "%s: pages [B, HKV, S]", role);
  Q35_REQUIRE(!keep.present || keep.numel() == 2, Q35_ERR_SHAPE, "%s: keep [2]", role);
  Q35_REQUIRE(bounds.s[0] >= 1 && bounds.s[0] <= INT_MAX && B * HKV <= INT_MAX / 4, Q35_ERR_SHAPE, "%s: sizes", role);
  SelectArgs a{};
  Q35_TRY(get_page_table(c, role, B, 1, bounds.s[0], &a.t));
  const int64_t E = HKV * int64_t(a.t.n_indices);
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = (off + bytes + 255) / 256 * 256; return o; };
  const int64_t o_sc = take(E * 8), o_zs = take(E * 8), o_zone = take(E * 4), o_flag = take(E);
  Q35_TRY(c.workspace(off, &ws));
  if (c.dry || B == 0) return 0;
  Q35_REQUIRE(aligned16(q.p) && aligned16(bounds.p), Q35_ERR_ALIGN, "%s: q and page_bounds must be 16-byte aligned", role);
  a.q = q.as<__nv_bfloat16>(); a.bounds = bounds.as<__nv_bfloat16>();
  a.keep = keep.present ? keep.as<int>() : nullptr;
  a.out = out.as<int>();
  a.HQ = int(HQ); a.HKV = int(HKV); a.G = int(HQ / HKV); a.D = int(D); a.S = int(S);
  uint8_t* w = ws.as<uint8_t>();
  a.score = reinterpret_cast<float2*>(w + o_sc); a.zscore = reinterpret_cast<double*>(w + o_zs);
  a.zone = reinterpret_cast<int*>(w + o_zone); a.flag = w + o_flag;
  // CTAs of 64 pages for twice the average sequence; longer ones go around
  a.gx = int((2 * ((a.t.n_indices + B - 1) / B) + 63) / 64);
  if (a.gx < 1) a.gx = 1;
  const int64_t most = INT_MAX / (B * HKV);
  if (a.gx > most) a.gx = int(most);
  const dim3 grid(unsigned(B * HKV * a.gx));
  if (D == 64) launch_pdl(select_score_kernel<64>, grid, dim3(128), 0, c.stream, a);
  else if (D == 128) launch_pdl(select_score_kernel<128>, grid, dim3(128), 0, c.stream, a);
  else launch_pdl(select_score_kernel<256>, grid, dim3(128), 0, c.stream, a);
  Q35_CUDA_LAUNCH_CHECK("attn.select_pages scores");
  const dim3 rows(unsigned(B * HKV));
  if (D == 64) launch_pdl(select_choose_kernel<64>, rows, dim3(SEL_THREADS), 0, c.stream, a);
  else if (D == 128) launch_pdl(select_choose_kernel<128>, rows, dim3(SEL_THREADS), 0, c.stream, a);
  else launch_pdl(select_choose_kernel<256>, rows, dim3(SEL_THREADS), 0, c.stream, a);
  Q35_CUDA_LAUNCH_CHECK("attn.select_pages choice");
  return 0;
}

}  // namespace q35
