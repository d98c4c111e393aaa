// The page table and the paged cache as the long-context roles see them (attn.page_bounds, attn.select_pages,
// attn.sparse_decode, attn.key_mass, attn.evict): host-side binding and device-side lookups.  Nothing found in the
// device tables is trusted: ranges, page ids and lengths are checked before an address is formed from them.
#pragma once
#include <climits>
#include "abi.h"
#include "common.cuh"

namespace q35 {

struct PageTable {
  const int* indptr;         // [B + 1]
  const int* indices;        // [n_indices]
  const int* last_page_len;  // [B]
  int B, P, num_pages, n_indices;
  int* status;
  uint32_t p_mul; int p_shift;   // position / P as a high product and a shift
  __device__ __forceinline__ int page_of(int pos) const {
    return int((__umulhi(p_mul, uint32_t(pos)) + uint32_t(pos)) >> p_shift);
  }
};

// 2^x by the special-function unit, 2 ulp; results below 2^-126 are 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The pages of sequence b: indices[first .. first + n), n counting only pages that hold a row, ctx rows in all.
// A range outside the table or a last page longer than P is recorded and the sequence counts as empty.
struct SeqPages { int first, n, ctx; };
__device__ __forceinline__ SeqPages seq_pages(const PageTable& t, int b) {
  const int lo = t.indptr[b], hi = t.indptr[b + 1];
  if (lo < 0 || hi < lo || hi > t.n_indices) {
    atomicOr(t.status, DS_BAD_PAGE);
    return {0, 0, 0};
  }
  if (hi == lo) return {lo, 0, 0};
  const int n = hi - lo, last = t.last_page_len[b];
  if (last < 0 || last > t.P) {
    atomicOr(t.status, DS_BAD_PAGE);
    return {0, 0, 0};
  }
  return {lo, last ? n : n - 1, (n - 1) * t.P + last};
}

// physical page of table entry e (inside the table), -1 (recorded) when the id is not a page of the cache
__device__ __forceinline__ int page_at(const PageTable& t, int e) {
  const int id = t.indices[e];
  if (unsigned(id) < unsigned(t.num_pages)) return id;
  atomicOr(t.status, DS_BAD_PAGE);
  return -1;
}

// The same without the record: page 0 for an id that is none, which `bad` remembers.  A record on the spot would wait for
// the id before the next instruction; callers that have several lookups on their way report once, behind them.
__device__ __forceinline__ int page_or_first(const PageTable& t, int e, bool& bad) {
  const int id = t.indices[e];
  const bool no = unsigned(id) >= unsigned(t.num_pages);
  bad |= no;
  return no ? 0 : id;
}

// a float as an unsigned integer of the same order; NaN ranks with -inf, and -0 with 0
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Which sequence, and which of its items, an index stands for when sequence b has count(b) items (whole warp); -1: none
template <typename Count>
__device__ __forceinline__ int2 find_item(int B, int index, Count count) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int c = b0 + lane < B ? count(b0 + lane) : 0;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + inc > index);
    if (hit) {
      const int l = __ffs(hit) - 1, at = index - before - __shfl_sync(0xffffffffu, inc - c, l);
      // ranges of a bad table may overlap, and the counts of a warp's sequences then wrap around: no item
      return unsigned(at) < unsigned(__shfl_sync(0xffffffffu, c, l)) ? make_int2(b0 + l, at) : make_int2(-1, 0);
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
  return make_int2(-1, 0);
}

struct KvCache {
  const void* p = nullptr;                    // [pages, 2, P, HKV, D]
  int fmt = 0;                                // 0 bf16, 1 E4M3, 2 int8 with row scales
  const float* kv_scale = nullptr;            // E4M3: [2, HKV], or null = the constant form (stored = 8 x value)
  const __nv_bfloat16* row_scale = nullptr;   // int8: [pages, 2, P, HKV]
  int64_t pages = 0, P = 0, HKV = 0, D = 0;
  int elt() const { return fmt == 0 ? 2 : 1; }
};

inline int get_kv_cache(Call& c, const char* role, KvCache* kv) {
  Tensor cache, ks, rs;
  Q35_TRY(c.get("paged_kv_cache", M(Q35_BF16) | M_FP8, &cache));
  Q35_TRY(c.get("kv_scale", M(Q35_F32), &ks, false));
  Q35_TRY(c.get("paged_kv_scale", M(Q35_BF16), &rs, false));
  Q35_REQUIRE(cache.nd == 5 && cache.s[1] == 2, Q35_ERR_SHAPE, "%s: paged_kv_cache [pages, 2, P, HKV, D]", role);
  kv->pages = cache.s[0]; kv->P = cache.s[2]; kv->HKV = cache.s[3]; kv->D = cache.s[4];
  Q35_REQUIRE(kv->pages >= 1 && kv->pages <= INT_MAX && kv->P >= 1 && kv->P <= INT_MAX && kv->HKV >= 1, Q35_ERR_SHAPE,
              "%s: an empty cache", role);
  Q35_REQUIRE(kv->HKV <= 4096 && kv->D >= 1 && kv->D <= 4096, Q35_ERR_SHAPE, "%s: HKV and D up to 4096", role);
  kv->fmt = cache.dtype == Q35_BF16 ? 0 : cache.dtype == Q35_E4M3 ? 1 : 2;
  Q35_REQUIRE(rs.present == (kv->fmt == 2), Q35_ERR_DTYPE,
              "%s: an int8 cache (bound as bytes) comes with paged_kv_scale, the other formats without", role);
  Q35_REQUIRE(!ks.present || kv->fmt == 1, Q35_ERR_DTYPE, "%s: kv_scale goes with an E4M3 cache", role);
  Q35_REQUIRE(!ks.present || ks.numel() == 2 * kv->HKV, Q35_ERR_SHAPE, "%s: kv_scale [2, HKV]", role);
  Q35_REQUIRE(!rs.present || rs.numel() == kv->pages * 2 * kv->P * kv->HKV, Q35_ERR_SHAPE,
              "%s: paged_kv_scale [pages, 2, P, HKV]", role);
  Q35_REQUIRE(c.dry || aligned16(cache.p), Q35_ERR_ALIGN, "%s: paged_kv_cache must be 16-byte aligned", role);
  kv->p = cache.p;
  kv->kv_scale = ks.present ? ks.as<float>() : nullptr;
  kv->row_scale = rs.present ? rs.as<__nv_bfloat16>() : nullptr;
  return 0;
}

// B sequences; P and num_pages of the cache the table points into
inline int get_page_table(Call& c, const char* role, int64_t B, int64_t P, int64_t num_pages, PageTable* t) {
  Tensor indptr, indices, last;
  Q35_TRY(c.get("indptr", M(Q35_I32), &indptr));
  Q35_TRY(c.get("indices", M(Q35_I32), &indices));
  Q35_TRY(c.get("last_page_len", M(Q35_I32), &last));
  Q35_REQUIRE(indptr.numel() == B + 1 && last.numel() >= B, Q35_ERR_SHAPE, "%s: indptr [B + 1], last_page_len [B]", role);
  Q35_REQUIRE(indices.numel() <= INT_MAX / 2 / P, Q35_ERR_UNSUPPORTED,  // kernels step behind the end before they look
              "%s: %lld table entries of %lld rows: at most 2^30 positions", role, (long long)indices.numel(),
              (long long)P);
  t->indptr = indptr.as<int>(); t->indices = indices.as<int>(); t->last_page_len = last.as<int>();
  t->B = int(B); t->P = int(P); t->num_pages = int(num_pages); t->n_indices = int(indices.numel());
  // n / P for n < 2^30: with 2^(l - 1) < P <= 2^l and m = floor(2^32 (2^l - P) / P) + 1, (umulhi(m, n) + n) >> l is exact
  int l = 0;
  while ((int64_t(1) << l) < P) ++l;
  t->p_mul = uint32_t((uint64_t(1) << 32) * ((uint64_t(1) << l) - uint64_t(P)) / uint64_t(P) + 1);
  t->p_shift = l;
  if (!c.dry) {
    t->status = device_status_ptr();
    Q35_REQUIRE(t->status != nullptr, Q35_ERR_CUDA, "%s: no device status word", role);
  }
  return 0;
}

}  // namespace q35
