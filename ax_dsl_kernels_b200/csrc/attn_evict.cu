// attn.evict: every (sequence, KV head) keeps the min(K, ctx) cached rows with the highest key_mass -- the first and the
// last ones always, ties to the lower position -- and moves them, in order, to the sequence's first rows, in place.
//
// evict_choose, one CTA per (sequence, KV head): the border by digits from the top, then one pass that writes the kept
// positions in ascending order.  evict_move: row j of the result is row kept[j] >= j of the cache.
// Bound: HBM, every row that changes place read and written once.
//
// In place and in parallel: the moves of different channels do not touch each other, so a CTA owns a column slice of 64
// bytes (of K or V of one head) and takes the kept rows in order, a chunk at a time -- all loads, a barrier, all stores.
// A chunk stores to rows below its end j1, later chunks load from rows kept[j] >= j >= j1: no store meets a later load.
#include "abi.h"
#include "attn_pages.cuh"

namespace q35 {

struct EvictArgs {
  PageTable t;
  uint8_t* cache;
  __nv_bfloat16* row_scale;    // int8 cache
  float* key_mass;             // [pages, P, HKV]
  const int* keep;             // optional [2]: first, last
  int* kept;                   // [B, HKV, K]
  int HKV, K, row_bytes;       // row_bytes of one head
};

constexpr int EV_THREADS = 1024;

__global__ void __launch_bounds__(EV_THREADS) evict_choose_kernel(const EvictArgs a) {
  pdl_wait();
  pdl_launch();
  __shared__ int s_hist[256];
  __shared__ int s_scan[2][32];
  __shared__ int s_digit, s_rank;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.HKV, h = blockIdx.x % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  const int n = sp.ctx, K = a.K;
  int* out = a.kept + size_t(blockIdx.x) * K;
  if (n <= K) {
    for (int i = tid; i < K; i += EV_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int last = a.keep ? min(max(a.keep[1], 0), K) : 0;
  const int first = a.keep ? min(max(a.keep[0], 0), K - last) : 0;
  const int m = n - first - last, rank = K - first - last;
  bool bad = false;
  auto key = [&](int i) -> uint32_t {  // of position first + i
    const int pos = first + i, page = page_or_first(a.t, sp.first + pos / a.t.P, bad);
    return order_key(a.key_mass[(size_t(page) * a.t.P + pos % a.t.P) * a.HKV + h]);
  };
  uint32_t border = 0;
  int equal = 0;  // how many of the rows that equal the border are kept
  if (rank > 0) {
    int left = rank;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += EV_THREADS) s_hist[i] = 0;
      __syncthreads();
      for (int i = tid; i < m; i += EV_THREADS) {
        const uint32_t k = key(i);
        if (shift == 24 || ((k ^ border) >> (shift + 8)) == 0) atomicAdd(&s_hist[k >> shift & 255], 1);
      }
      __syncthreads();
      if (tid == 0) {
        int d = 255, rest = left;
        while (d > 0 && rest > s_hist[d]) rest -= s_hist[d--];
        s_digit = d;
        s_rank = rest;
      }
      __syncthreads();
      border |= uint32_t(s_digit) << shift;
      left = s_rank;
      __syncthreads();
    }
    equal = left;
  }
  int at = 0, seen = 0;
  for (int i0 = 0; i0 < n; i0 += EV_THREADS) {
    const int i = i0 + tid;
    const bool forced = i < n && (i < first || i >= n - last);
    const uint32_t k = i < n && !forced && rank > 0 ? key(i - first) : 0u;
    const bool eq = i < n && !forced && rank > 0 && k == border;
    const unsigned be = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) s_scan[0][warp] = __popc(be);
    __syncthreads();
    int before = seen + __popc(be & ((1u << lane) - 1)), total_eq = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += s_scan[0][w];
      total_eq += s_scan[0][w];
    }
    const bool take = forced || (i < n && rank > 0 && (k > border || (eq && before < equal)));
    const unsigned bt = __ballot_sync(0xffffffffu, take);
    if (lane == 0) s_scan[1][warp] = __popc(bt);
    __syncthreads();
    int pos = at + __popc(bt & ((1u << lane) - 1)), total = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) pos += s_scan[1][w];
      total += s_scan[1][w];
    }
    if (take && pos < K) out[pos] = i;
    at += total;
    seen += total_eq;
    __syncthreads();
  }
  if (bad) atomicOr(a.t.status, DS_BAD_PAGE);
}

constexpr int EM_THREADS = 512;
constexpr int EM_SLICE = 64;                      // bytes of a row a CTA moves
constexpr int EM_ROWS = EM_THREADS / (EM_SLICE / 16);  // rows per round of loads
constexpr int EM_U = 8;                           // rounds in flight

// blockIdx.y: slices of K, slices of V, then one CTA for what a row has beside its elements (mass, int8 scales)
__global__ void __launch_bounds__(EM_THREADS) evict_move_kernel(const EvictArgs a) {
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x;
  const int b = blockIdx.x / a.HKV, h = blockIdx.x % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  if (sp.ctx <= a.K) return;  // everything stays where it is
  const int n = a.K, P = a.t.P, slices = a.row_bytes / EM_SLICE;
  const int* kept = a.kept + size_t(blockIdx.x) * a.K;
  // row (position) -> index of its K row among all rows of the cache, -1 if the table names no page
  auto row_of = [&](int pos) -> int64_t {
    const int page = page_at(a.t, sp.first + pos / P);
    return page < 0 ? -1 : (int64_t(page) * 2 * P + pos % P) * a.HKV + h;
  };
  if (int(blockIdx.y) < 2 * slices) {
    const int v = int(blockIdx.y) >= slices, slice = int(blockIdx.y) - v * slices;
    uint8_t* base = a.cache + size_t(v) * P * a.HKV * a.row_bytes + slice * EM_SLICE + (tid & 3) * 16;
    for (int j0 = 0; j0 < n; j0 += EM_ROWS * EM_U) {
      uint4 x[EM_U];
      int64_t to[EM_U];
#pragma unroll
      for (int u = 0; u < EM_U; ++u) {
        const int j = j0 + u * EM_ROWS + (tid >> 2);
        to[u] = -1;
        if (j < n) {
          const int src = kept[j];
          if (src != j && src > j && src < sp.ctx) {
            const int64_t from = row_of(src);
            if (from >= 0) {
              to[u] = row_of(j);
              x[u] = *reinterpret_cast<const uint4*>(base + from * a.row_bytes);
            }
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < EM_U; ++u)
        if (to[u] >= 0) *reinterpret_cast<uint4*>(base + to[u] * a.row_bytes) = x[u];
    }
    return;
  }
  for (int j0 = 0; j0 < n; j0 += EM_THREADS * 4) {
    float mass[4];
    __nv_bfloat16 ks[4], vs[4];
    int64_t to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + u * EM_THREADS + tid;
      to[u] = -1;
      if (j < n) {
        const int src = kept[j];
        if (src > j && src < sp.ctx) {
          const int64_t from = row_of(src);
          if (from >= 0) {
            to[u] = row_of(j);
            const int64_t page = from / (int64_t(2) * P * a.HKV), in = from % (int64_t(2) * P * a.HKV);
            mass[u] = a.key_mass[page * P * a.HKV + in];
            if (a.row_scale) {
              ks[u] = a.row_scale[from];
              vs[u] = a.row_scale[from + int64_t(P) * a.HKV];
            }
          }
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (to[u] < 0) continue;
      const int64_t page = to[u] / (int64_t(2) * P * a.HKV), in = to[u] % (int64_t(2) * P * a.HKV);
      a.key_mass[page * P * a.HKV + in] = mass[u];
      if (a.row_scale) {
        a.row_scale[to[u]] = ks[u];
        a.row_scale[to[u] + int64_t(P) * a.HKV] = vs[u];
      }
    }
  }
}

int run_attn_evict(Call& c) {
  const char* role = "attn.evict";
  KvCache kv;
  Q35_TRY(get_kv_cache(c, role, &kv));
  Tensor mass, keep, kept;
  Q35_TRY(c.get("key_mass", M(Q35_F32), &mass));
  Q35_TRY(c.get("keep", M(Q35_I32), &keep, false));
  Q35_TRY(c.get("kept", M(Q35_I32), &kept));
  Q35_REQUIRE(!kv.kv_scale, Q35_ERR_UNSUPPORTED, "%s: kv_scale does not enter", role);
  Q35_REQUIRE(kept.nd == 3 && kept.s[1] == kv.HKV && kept.s[2] >= 1 && kept.s[2] <= INT_MAX / 2, Q35_ERR_SHAPE,
              "%s: kept [B, HKV, K]", role);
  Q35_REQUIRE(mass.numel() == kv.pages * kv.P * kv.HKV, Q35_ERR_SHAPE, "%s: key_mass [pages, P, HKV]", role);
  Q35_REQUIRE(!keep.present || keep.numel() == 2, Q35_ERR_SHAPE, "%s: keep [2]", role);
  EvictArgs a{};
  const int64_t B = kept.s[0];
  Q35_TRY(get_page_table(c, role, B, kv.P, kv.pages, &a.t));
  a.row_bytes = int(kv.D) * kv.elt();
  Q35_REQUIRE(a.row_bytes % EM_SLICE == 0, Q35_ERR_UNSUPPORTED, "%s: a row of a head must be a multiple of 64 bytes", role);
  Q35_REQUIRE(B * kv.HKV <= INT_MAX, Q35_ERR_SHAPE, "%s: sizes beyond 32 bits", role);
  c.ws_need = 0;
  if (c.dry || B == 0) return 0;
  a.cache = static_cast<uint8_t*>(const_cast<void*>(kv.p));
  a.row_scale = const_cast<__nv_bfloat16*>(kv.row_scale);
  a.key_mass = mass.as<float>(); a.keep = keep.present ? keep.as<int>() : nullptr; a.kept = kept.as<int>();
  a.HKV = int(kv.HKV); a.K = int(kept.s[2]);
  launch_pdl(evict_choose_kernel, dim3(unsigned(B * kv.HKV)), dim3(EV_THREADS), 0, c.stream, a);
  Q35_CUDA_LAUNCH_CHECK("attn.evict choice");
  launch_pdl(evict_move_kernel, dim3(unsigned(B * kv.HKV), unsigned(2 * (a.row_bytes / EM_SLICE) + 1)), dim3(EM_THREADS), 0,
             c.stream, a);
  Q35_CUDA_LAUNCH_CHECK("attn.evict moves");
  return 0;
}

}  // namespace q35
