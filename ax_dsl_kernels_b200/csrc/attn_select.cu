// Choosing the pages a query attends to: attn.page_bounds (what the keys of a page can be) and attn.select_pages (the
// pages whose keys can score highest).
//
// For a page with keys k_1 .. k_m let lo_d = min_i k_id and hi_d = max_i k_id.  Then q . k_i <= sum_d max(q_d lo_d,
// q_d hi_d) for every key of the page, and the right side costs 1 / (P / 2) of the products with all P keys.  A KV head
// is shared by G query heads, so a page's score is the maximum of the G bounds.
#include <cooperative_groups.h>
#include "abi.h"
#include "attn_pages.cuh"
#include "block_select.cuh"
#include "kv_formats.cuh"

namespace q35 {

namespace cg = cooperative_groups;

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
  const int from = min(max(0, a.first_page[b]), sp.n);  // whatever the tensor holds: sums of it stay below 2^31
  for (int i = from + int(blockIdx.x) % a.per_seq; i < sp.n; i += a.per_seq) {
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
// any order of n = 2 D terms, and a third product, |q| . max(|lo|, |hi|), bounds that sum; the few pages within that
// error of the border (most often one to three) are scored again in fp64: a sum of 256 products of 16 significant bits is
// exact there while they lie within 2^28 of one another, else rounded at 2^-53 of its largest partial sum.  (An infinite
// bound turns 0 * inf of the split form into a NaN and the error into infinity: then every page is scored again, by the
// definition.)
//
// Bound: HBM for the bounds (each read once); at one sequence the chain of the selection.  One launch: a cluster of up
// to 8 CTAs scores the pages of one (sequence, KV head) and leaves the scores in the shared memory of its first CTA,
// which chooses (two kernels with the scores in HBM between them, graph replays with the bounds in L2: 21.6 us instead of
// 10.0 for 256 pages, 31.8 instead of 18.0 for 32 rows of 2048).
struct SelectArgs {
  const __nv_bfloat16* q;       // [B, HQ, D]
  const __nv_bfloat16* bounds;  // [pages, 2, HKV, D]
  PageTable t;                  // P unused
  const int* keep;              // optional [2]: first, last
  int* out;                     // [B, HKV, S]
  int HQ, HKV, G, S;
  int cap;                      // pages whose scores and flags fit the shared memory
  // workspace, [HKV * n_indices] each, entries of (b, kvh) from HKV * indptr[b] + kvh * n on: where more is needed than
  // fits the shared memory
  float* score;
  uint8_t* flag;                // 0 out, 1 in, 2 undecided
  double* zscore;               // fp64 scores of the undecided pages
  int* zone;                    // their positions
};

constexpr int SEL_THREADS = 512, SEL_WARPS = 16;
constexpr int SEL_CAP = 16384;     // pages of a sequence that stay in shared memory
constexpr int SEL_KEYS = 4;        // pages per thread and round of the output
static_assert(SEL_KEYS * SEL_WARPS == 64, "the output's scan takes two counts a lane");
constexpr int SEL_ZONE = 512;      // undecided pages that stay in shared memory

// pages of sequence b that hold a row, without knowing P
__device__ __forceinline__ int2 select_range(const SelectArgs& a, int b) {
  const int lo = a.t.indptr[b], hi = a.t.indptr[b + 1];
  const bool range = lo >= 0 && hi >= lo && hi <= a.t.n_indices;
  const int last = range && hi > lo ? a.t.last_page_len[b] : 0;
  if (!range || last < 0) {
    atomicOr(a.t.status, DS_BAD_PAGE);
    return make_int2(0, 0);
  }
  return make_int2(lo, hi - lo - (hi > lo && last == 0 ? 1 : 0));
}
__device__ __forceinline__ uint32_t pos_pair(uint32_t x) {
  __nv_bfloat162 v = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t neg_pair(uint32_t x) {
  __nv_bfloat162 v = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&x), __floats2bfloat162_rn(0.f, 0.f));
  return *reinterpret_cast<uint32_t*>(&v);
}
// larger magnitudes of two pairs (a NaN gives way to a number)
__device__ __forceinline__ uint32_t abs_max_pair(uint32_t x, uint32_t y) {
  x &= 0x7fff7fffu;
  y &= 0x7fff7fffu;
  __nv_bfloat162 v = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&x), *reinterpret_cast<__nv_bfloat162*>(&y));
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ float max_nan(float x, float y) { return x != x ? x : y != y ? y : fmaxf(x, y); }
__device__ __forceinline__ unsigned long long order_key64(double x) {
  if (x != x) x = -INFINITY;
  const unsigned long long u = __double_as_longlong(x + 0.0);
  return u >> 63 ? ~u : u | (1ull << 63);
}

// One warp scores the 16 pages from p0 on: A = the pages' hi and lo rows, B = max(q, 0) and min(q, 0) of 8 heads.  Both
// operands take their k index from 16-byte loads (lane c of a row's four holds channels 8 c .. 8 c + 7 of every 32), so
// the fragments come straight from global memory and a row is read in full sectors.  Returns the largest error bound.
template <int D>
__device__ __forceinline__ float score_pages(const SelectArgs& a, int b, int h, int first, int n, int p0, float* score) {
  const int lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
  const size_t plane = size_t(a.HKV) * D;
  bool bad = false;
  const int g0 = page_or_first(a.t, first + min(p0 + r, n - 1), bad);
  const int g1 = page_or_first(a.t, first + min(p0 + r + 8, n - 1), bad);
  const uint4* lo0 = reinterpret_cast<const uint4*>(a.bounds + size_t(g0) * 2 * plane + size_t(h) * D + 8 * c);
  const uint4* lo1 = reinterpret_cast<const uint4*>(a.bounds + size_t(g1) * 2 * plane + size_t(h) * D + 8 * c);
  const size_t up = plane / 8;  // from a minimum to its maximum, in 16-byte pieces
  float best0 = -INFINITY, best1 = -INFINITY, err = 0.f;
  for (int q0 = 0; q0 < a.G; q0 += 8) {
    const bool hv = q0 + r < a.G;
    const uint4* qp = reinterpret_cast<const uint4*>(a.q + (size_t(b) * a.HQ + size_t(h) * a.G + (hv ? q0 + r : 0)) * D + 8 * c);
    float ap[4] = {0.f, 0.f, 0.f, 0.f}, an[4] = {0.f, 0.f, 0.f, 0.f}, as[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int NB = D / 32 < 4 ? D / 32 : 4;  // 32-channel pieces whose loads go out together
#pragma unroll
    for (int j0 = 0; j0 < D / 32; j0 += NB) {
      uint4 l0[NB], l1[NB], h0[NB], h1[NB], qv[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        l0[j] = __ldg(lo0 + (j0 + j) * 4);
        l1[j] = __ldg(lo1 + (j0 + j) * 4);
        h0[j] = __ldg(lo0 + up + (j0 + j) * 4);
        h1[j] = __ldg(lo1 + up + (j0 + j) * 4);
        qv[j] = hv ? __ldg(qp + (j0 + j) * 4) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        mma_bf16_16816(ap, h0[j].x, h1[j].x, h0[j].y, h1[j].y, pos_pair(qv[j].x), pos_pair(qv[j].y));
        mma_bf16_16816(an, l0[j].x, l1[j].x, l0[j].y, l1[j].y, neg_pair(qv[j].x), neg_pair(qv[j].y));
        mma_bf16_16816(as, abs_max_pair(h0[j].x, l0[j].x), abs_max_pair(h1[j].x, l1[j].x), abs_max_pair(h0[j].y, l0[j].y),
                       abs_max_pair(h1[j].y, l1[j].y), qv[j].x & 0x7fff7fffu, qv[j].y & 0x7fff7fffu);
        mma_bf16_16816(ap, h0[j].z, h1[j].z, h0[j].w, h1[j].w, pos_pair(qv[j].z), pos_pair(qv[j].w));
        mma_bf16_16816(an, l0[j].z, l1[j].z, l0[j].w, l1[j].w, neg_pair(qv[j].z), neg_pair(qv[j].w));
        mma_bf16_16816(as, abs_max_pair(h0[j].z, l0[j].z), abs_max_pair(h1[j].z, l1[j].z), abs_max_pair(h0[j].w, l0[j].w),
                       abs_max_pair(h1[j].w, l1[j].w), qv[j].z & 0x7fff7fffu, qv[j].w & 0x7fff7fffu);
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (q0 + 2 * c + u < a.G) {
        best0 = max_nan(best0, ap[u] + an[u]);
        best1 = max_nan(best1, ap[2 + u] + an[2 + u]);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) err = fmaxf(err, as[u]);  // a NaN here comes with a score that is NaN, and ranks last
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    best0 = max_nan(best0, __shfl_xor_sync(0xffffffffu, best0, o));
    best1 = max_nan(best1, __shfl_xor_sync(0xffffffffu, best1, o));
  }
  if (c == 0) {
    if (p0 + r < n) score[p0 + r] = best0;
    if (p0 + r + 8 < n) score[p0 + r + 8] = best1;
  }
  if (bad) atomicOr(a.t.status, DS_BAD_PAGE);
  // 2 D terms, the three sums' own roundings, the final addition: (2 D + 8) 2^-23, and 1 + 2^-9 for `as` being rounded
  return err * ((2 * D + 8) * (1.f + 1.f / 512) / 8388608.f);
}

// The r-th largest (r >= 1) of the 64-bit keys key(0 .. n - 1), digit by digit from the top: a histogram of the digits of
// the keys that agree with the prefix so far, then the digit in which the rank falls.  above = how many keys are larger.
template <typename F>
__device__ unsigned long long block_kth64(F key, int n, int r, int* hist, int* above) {
  __shared__ int s_digit, s_rank;
  using K = unsigned long long;
  K prefix = 0;
  int rank = r;
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const K k = key(i);
      if (shift == 56 || ((k ^ prefix) >> (shift + 8)) == 0) atomicAdd(&hist[int(k >> shift) & 255], 1);
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

template <int D>
__global__ void __launch_bounds__(SEL_THREADS, 1) select_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_err[8 * SEL_WARPS];  // one entry per warp of the cluster
  __shared__ KthScratch<SEL_THREADS> s_kth;
  __shared__ int s_hist[256];
  __shared__ int s_red[2][SEL_WARPS], s_count[SEL_KEYS][SEL_WARPS], s_total;
  __shared__ int s_zone[SEL_ZONE];
  __shared__ double s_zscore[SEL_ZONE];
  __shared__ int s_nz;
  pdl_wait();
  pdl_launch();
  cg::cluster_group cluster = cg::this_cluster();
  auto started = cluster.barrier_arrive();  // its shared memory is written from outside once the first CTA runs
  const int NC = int(cluster.num_blocks()), crank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / NC, b = row / a.HKV, h = row % a.HKV;
  const int2 rg = select_range(a, b);
  const int n = rg.y, S = a.S;
  const size_t base = size_t(a.HKV) * rg.x + size_t(h) * n;
  float* s_score = reinterpret_cast<float*>(smem);
  const bool fits = n <= a.cap;
  cluster.barrier_wait(std::move(started));
  if (n > S) {
    float* score = fits ? cluster.map_shared_rank(s_score, 0) : a.score + base;
    float err = 0.f;
    for (int p0 = (warp * NC + crank) * 16; p0 < n; p0 += NC * SEL_WARPS * 16)
      err = fmaxf(err, score_pages<D>(a, b, h, rg.x, n, p0, score));
#pragma unroll
    for (int o = 16; o; o >>= 1) err = fmaxf(err, __shfl_xor_sync(0xffffffffu, err, o));
    if (lane == 0) cluster.map_shared_rank(s_err, 0)[crank * SEL_WARPS + warp] = err;
  }
  if (!fits) __threadfence();
  cluster.sync();
  if (crank) return;  // only the first CTA's memory is read from here on
  int* out = a.out + size_t(row) * S;
  if (n <= S) {
    for (int i = tid; i < S; i += SEL_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const float* score = fits ? s_score : a.score + base;
  uint8_t* flag = fits ? smem + size_t(a.cap) * 4 : a.flag + base;
  const int last = a.keep ? min(max(a.keep[1], 0), S) : 0;
  const int first = a.keep ? min(max(a.keep[0], 0), S - last) : 0;
  const int m = n - first - last, rank = S - first - last;  // rank of the m free pages; rank < m because S < n
  if (rank > 0) {
    float e = 0.f;
    for (int w = 0; w < NC * SEL_WARPS; ++w) e = fmaxf(e, s_err[w]);
    const bool all = !(e < INFINITY);  // sums that overflow fp32: every page is scored again
    uint32_t kth;
    if (m <= 4 * SEL_THREADS) {
      uint32_t k[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) k[j] = tid + j * SEL_THREADS < m ? order_key(score[first + tid + j * SEL_THREADS]) : 0u;
      kth = block_kth<SEL_THREADS, true>(
          [&](auto f) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (tid + j * SEL_THREADS < m) f(k[j]);
          },
          rank, s_kth);
    } else {
      kth = block_kth<SEL_THREADS, true>(
          [&](auto f) {
            for (int i = tid; i < m; i += SEL_THREADS) f(order_key(score[first + i]));
          },
          rank, s_kth);
    }
    // the rank-th score as a float again; a true score differs from its fp32 one by e at most, so does the border
    const float tau = key_value(kth);
    const float top = tau + 2.f * e, low = tau - 2.f * e;
    int in = 0, near = 0;
    for (int i = tid; i < m; i += SEL_THREADS) {
      const float s = score[first + i];
      const int f = all || !(s > top || s < low) ? 2 : s > top;
      in += f == 1;
      near += f == 2;
      flag[first + i] = uint8_t(f);
    }
    in = __reduce_add_sync(0xffffffffu, in);
    near = __reduce_add_sync(0xffffffffu, near);
    if (lane == 0) { s_red[0][warp] = in; s_red[1][warp] = near; }
    __syncthreads();
    in = 0;
    int z = 0;  // undecided pages
#pragma unroll
    for (int w = 0; w < SEL_WARPS; ++w) { in += s_red[0][w]; z += s_red[1][w]; }
    const int need = rank - in;  // 1 <= need <= z: the zone holds the border
    const size_t plane = size_t(a.HKV) * D;
    if (z == need) {  // nothing undecided
      for (int i = tid; i < m; i += SEL_THREADS) flag[first + i] = flag[first + i] != 0;
    } else {
      int* zone = z <= SEL_ZONE ? s_zone : a.zone + base;
      double* zs = z <= SEL_ZONE ? s_zscore : a.zscore + base;
      if (tid == 0) s_nz = 0;
      __syncthreads();
      for (int i = tid; i < m; i += SEL_THREADS)
        if (flag[first + i] == 2) zone[atomicAdd(&s_nz, 1)] = first + i;
      __syncthreads();
      for (int j = warp; j < z; j += SEL_WARPS) {
        const int i = zone[j];
        bool bad = false;
        const __nv_bfloat16* lo = a.bounds + size_t(page_or_first(a.t, rg.x + i, bad)) * 2 * plane + size_t(h) * D;
        // every lane its D / 32 channels of the page, eight heads' partial sums at a time; folding halves of the warp
        // leaves lane l the sum of head (l >> 2) & 7
        // A channel's term is q * hi for q > 0 and q * lo for q < 0; for q = 0 it is 0, or NaN beside an infinite bound.
        constexpr int CH = D / 32;
        double l[CH], u[CH], z0[CH];
#pragma unroll
        for (int i = 0; i < CH; i += 2) {
          const uint32_t l2 = *reinterpret_cast<const uint32_t*>(lo + lane * CH + i);
          const uint32_t u2 = *reinterpret_cast<const uint32_t*>(lo + plane + lane * CH + i);
          l[i] = bf16lo(l2); l[i + 1] = bf16hi(l2); u[i] = bf16lo(u2); u[i + 1] = bf16hi(u2);
          z0[i] = bf16lo(l2) * 0.f + bf16lo(u2) * 0.f;
          z0[i + 1] = bf16hi(l2) * 0.f + bf16hi(u2) * 0.f;
        }
        double best = -INFINITY;
        for (int q0 = 0; q0 < a.G; q0 += 8) {
          double sum[8];
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            const __nv_bfloat16* qp = a.q + (size_t(b) * a.HQ + size_t(h) * a.G + min(q0 + g, a.G - 1)) * D + lane * CH;
            sum[g] = 0.;
#pragma unroll
            for (int i = 0; i < CH; i += 2) {
              const uint32_t q2 = *reinterpret_cast<const uint32_t*>(qp + i);
              const float qa = bf16lo(q2), qb = bf16hi(q2);
              sum[g] += double(qa) * (qa > 0.f ? u[i] : qa < 0.f ? l[i] : z0[i]);
              sum[g] += double(qb) * (qb > 0.f ? u[i + 1] : qb < 0.f ? l[i + 1] : z0[i + 1]);
            }
          }
#pragma unroll
          for (int half = 4; half; half >>= 1)
#pragma unroll
            for (int g = 0; g < half; ++g) {
              const bool up = lane & (half * 4);
              const double other = __shfl_xor_sync(0xffffffffu, up ? sum[g] : sum[g + half], half * 4);
              sum[g] = (up ? sum[g + half] : sum[g]) + other;
            }
          sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 2);
          sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 1);
          best = best != best || sum[0] != sum[0] ? NAN : fmax(best, sum[0]);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          const double other = __shfl_xor_sync(0xffffffffu, best, o);
          best = best != best || other != other ? NAN : fmax(best, other);
        }
        if (lane == 0) zs[j] = best != best ? -INFINITY : best;
      }
      __syncthreads();
      if (z <= SEL_ZONE) {  // each page of the zone counts the pages that go before it
        for (int j = tid; j < z; j += SEL_THREADS) {
          const int i = zone[j];
          const double s = zs[j];
          int before = 0;
          for (int k = 0; k < z; ++k) before += zs[k] > s || (zs[k] == s && zone[k] < i);
          flag[i] = before < need;
        }
      } else {  // pages that hardly differ: the border by digits, equal ones by position
        int above;
        const unsigned long long k64 =
            block_kth64([&](int j) { return order_key64(zs[j]); }, z, need, s_hist, &above);
        for (int j = tid; j < z; j += SEL_THREADS) {
          const unsigned long long k = order_key64(zs[j]);
          flag[zone[j]] = k > k64 ? 1 : k < k64 ? 0 : 2;
        }
        __syncthreads();
        int left = need - above;  // of the pages equal to the border (flag 2) the first `left` in order
        for (int i0 = 0; i0 < m; i0 += SEL_THREADS) {
          const int i = first + i0 + tid;
          const bool eq = i0 + tid < m && flag[i] == 2;
          const unsigned ball = __ballot_sync(0xffffffffu, eq);
          if (lane == 0) s_red[0][warp] = __popc(ball);
          __syncthreads();
          int before = __popc(ball & ((1u << lane) - 1)), total = 0;
          for (int w = 0; w < SEL_WARPS; ++w) {
            if (w < warp) before += s_red[0][w];
            total += s_red[0][w];
          }
          if (eq) flag[i] = before < left;
          left = max(0, left - total);
          __syncthreads();
        }
      }
    }
  }
  __syncthreads();
  // ascending output, SEL_KEYS pages per thread at a time: counts per (round, warp), one scan over them, then the places
  int at = 0;
  for (int c0 = 0; c0 < n; c0 += SEL_KEYS * SEL_THREADS) {
    unsigned ball[SEL_KEYS];
#pragma unroll
    for (int j = 0; j < SEL_KEYS; ++j) {
      const int i = c0 + j * SEL_THREADS + tid;
      ball[j] = __ballot_sync(0xffffffffu, i < n && (i < first || i >= n - last || (rank > 0 && flag[i] == 1)));
      if (lane == 0) s_count[j][warp] = __popc(ball[j]);
    }
    __syncthreads();
    if (warp == 0) {  // 64 counts, two to a lane
      int* cnt = &s_count[0][0] + 2 * lane;
      const int x = cnt[0], y = cnt[1];
      int inc = x + y;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      cnt[0] = inc - x - y;
      cnt[1] = inc - y;
      if (lane == 31) s_total = inc;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SEL_KEYS; ++j) {
      const int pos = at + s_count[j][warp] + __popc(ball[j] & ((1u << lane) - 1));
      if ((ball[j] >> lane & 1) && pos < S) out[pos] = c0 + j * SEL_THREADS + tid;
    }
    at += s_total;
    __syncthreads();
  }
}

template <int D>
static int launch_select(const SelectArgs& a, int cluster, cudaStream_t stream) {
  const int smem = a.cap * 5;
  Q35_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(select_kernel<D>), SEL_CAP * 5));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.t.B) * a.HKV * cluster);
  cfg.blockDim = dim3(SEL_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster); attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, select_kernel<D>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the caller's next CUDA call
    return fail(Q35_ERR_CUDA, "attn.select_pages: %s", cudaGetErrorString(e));
  }
  Q35_CUDA_LAUNCH_CHECK("attn.select_pages");
  return 0;
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
  Q35_REQUIRE(bounds.s[0] >= 1 && bounds.s[0] <= INT_MAX && B * HKV <= INT_MAX / 16, Q35_ERR_SHAPE, "%s: sizes", role);
  SelectArgs a{};
  Q35_TRY(get_page_table(c, role, B, 1, bounds.s[0], &a.t));
  a.cap = a.t.n_indices < SEL_CAP ? (a.t.n_indices + 15) / 16 * 16 : SEL_CAP;
  const int64_t E = HKV * int64_t(a.t.n_indices), big = a.t.n_indices > SEL_CAP ? E : 0;
  int64_t off = 0;
  auto take = [&](int64_t bytes) { const int64_t o = off; off = (off + bytes + 255) / 256 * 256; return o; };
  const int64_t o_zs = take(E * 8), o_zone = take(E * 4), o_sc = take(big * 4), o_flag = take(big);
  Q35_TRY(c.workspace(off, &ws));
  if (c.dry || B == 0) return 0;
  Q35_REQUIRE(aligned16(q.p) && aligned16(bounds.p), Q35_ERR_ALIGN, "%s: q and page_bounds must be 16-byte aligned", role);
  a.q = q.as<__nv_bfloat16>(); a.bounds = bounds.as<__nv_bfloat16>();
  a.keep = keep.present ? keep.as<int>() : nullptr;
  a.out = out.as<int>();
  a.HQ = int(HQ); a.HKV = int(HKV); a.G = int(HQ / HKV); a.S = int(S);
  uint8_t* w = ws.as<uint8_t>();
  a.zscore = reinterpret_cast<double*>(w + o_zs);
  a.zone = reinterpret_cast<int*>(w + o_zone);
  a.score = reinterpret_cast<float*>(w + o_sc); a.flag = w + o_flag;
  // four 16-page tiles per CTA for the average sequence (an SM reads a quarter of a megabyte in 3 us), as far as all
  // clusters run at once, one CTA to an SM (clusters of 8 that have to share SMs do not all find a place: 32 rows of 2048
  // pages, bounds from HBM, 25.4 us with 4, 28.9 with 8)
  const int64_t tiles = ((a.t.n_indices + B - 1) / B + 15) / 16;
  int cluster = 1;
  while (cluster < 8 && cluster * 4 < tiles && B * HKV * cluster * 2 <= sm_count()) cluster *= 2;
  if (D == 64) return launch_select<64>(a, cluster, c.stream);
  if (D == 128) return launch_select<128>(a, cluster, c.stream);
  return launch_select<256>(a, cluster, c.stream);
}

}  // namespace q35
