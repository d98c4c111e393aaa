// The r-th largest of many floats by one thread block (attn.select_pages, attn.evict), as order_key's integers.
#pragma once
#include "attn_pages.cuh"

namespace q35 {

// order_key's inverse
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr int KTH_BINS = 1024, KTH_LIST = 64;

template <int THREADS>
struct KthScratch {
  int hist[KTH_BINS];
  uint4 count[2][THREADS / 32];
  uint32_t red[2][THREADS / 32];
  int warp_sum[THREADS / 32];
  uint32_t list[KTH_LIST];
  int bin, rank, in_bin, listed;
};

// each(f) calls f(key) for every key of the calling thread, at most 2047 of them; 1 <= r <= number of keys in the block.
// Returns the r-th largest key to every thread.
//
// First one histogram of 1024 bins between the smallest and the largest key, evenly spaced by value (BY_VALUE: scores,
// which spread like a normal distribution) or by key (weights, which spread over octaves); the keys of the bin that
// holds the r-th, seldom more than a few, are ranked directly.  Where they are many -- equal keys, far outliers, infinite
// ends -- the interval is narrowed by seven pivots at a time instead, whose keys are counted: four rounds of pivots
// evenly spaced by value, then by key, an eighth of the interval a round, so that 11 more end it whatever the keys.
template <int THREADS, bool BY_VALUE, typename Each>
__device__ uint32_t block_kth(Each each, int r, KthScratch<THREADS>& s) {
  constexpr int WARPS = THREADS / 32, PER = KTH_BINS / THREADS, VALUE_ROUNDS = 4;
  static_assert(KTH_BINS % THREADS == 0, "whole bins per thread");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t lo = 0xffffffffu, hi = 0u;
  each([&](uint32_t k) { lo = min(lo, k); hi = max(hi, k); });
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  __syncthreads();  // an earlier call's reads
  if (lane == 0) { s.red[0][warp] = lo; s.red[1][warp] = hi; }
#pragma unroll
  for (int i = 0; i < PER; ++i) s.hist[tid + i * THREADS] = 0;
  if (tid == 0) s.listed = 0;
  __syncthreads();
  lo = __reduce_min_sync(0xffffffffu, s.red[0][lane % WARPS]);
  hi = __reduce_max_sync(0xffffffffu, s.red[1][lane % WARPS]);
  if (lo == hi) return lo;
  const float vlo = key_value(lo), scale = BY_VALUE ? (KTH_BINS - 1) / (key_value(hi) - vlo) : (KTH_BINS - 1) / float(hi - lo);
  if (scale > 0.f && scale < INFINITY) {
    // rounding keeps the order, so a bin holds an interval of keys
    auto bin_of = [&](uint32_t k) { return min(KTH_BINS - 1, int((BY_VALUE ? key_value(k) - vlo : float(k - lo)) * scale)); };
    each([&](uint32_t k) { atomicAdd(&s.hist[bin_of(k)], 1); });
    __syncthreads();
    int cnt[PER], sum = 0;  // thread t owns the bins PER t .. PER t + PER - 1 counted from the top
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cnt[i] = s.hist[KTH_BINS - 1 - (tid * PER + i)];
      sum += cnt[i];
    }
    int inc = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) s.warp_sum[warp] = inc;
    __syncthreads();
    int before = inc - sum + int(__reduce_add_sync(0xffffffffu, lane < warp ? unsigned(s.warp_sum[lane % WARPS]) : 0u));
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (before < r && r <= before + cnt[i]) {
        s.bin = KTH_BINS - 1 - (tid * PER + i);
        s.rank = r - before;
        s.in_bin = cnt[i];
      }
      before += cnt[i];
    }
    __syncthreads();
    const int bin = s.bin, n = s.in_bin, rank = s.rank;
    if (n <= KTH_LIST) {
      each([&](uint32_t k) {
        if (bin_of(k) == bin) s.list[atomicAdd(&s.listed, 1)] = k;
      });
      __syncthreads();
      uint32_t found = 0u;  // every warp for itself: the key with fewer than rank keys above it and rank at or above it
      for (int i = lane; i < n; i += 32) {
        const uint32_t k = s.list[i];
        int above = 0, equal = 0;
        for (int j = 0; j < n; ++j) {
          above += s.list[j] > k;
          equal += s.list[j] == k;
        }
        if (above < rank && rank <= above + equal) found = k;
      }
      return __reduce_max_sync(0xffffffffu, found);
    }
  }
  for (int round = 0; lo < hi; ++round) {  // at least r keys are >= lo, fewer than r are > hi
    uint32_t p[8];  // ascending, in (lo, hi]; p[7] repeats p[6]
    const float flo = key_value(lo), step = (key_value(hi) - flo) * 0.125f;
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      const uint32_t by_key = lo + max(uint32_t((uint64_t(hi - lo) * (j + 1)) >> 3), 1u);
      // not a number (an infinite end), or rounded to an end: the clamp keeps every pivot inside
      const uint32_t by_value = order_key(fmaf(step, float(j + 1), flo));
      p[j] = round < VALUE_ROUNDS ? min(max(by_value, lo + 1), hi) : by_key;
    }
    p[7] = p[6];
    uint32_t c[4] = {0u, 0u, 0u, 0u};  // counts of p[i] and p[i + 4] in the halves of c[i]
    each([&](uint32_t k) {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] += (k >= p[i] ? 1u : 0u) + (k >= p[i + 4] ? 0x10000u : 0u);
    });
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = __reduce_add_sync(0xffffffffu, c[i]);
    if (lane == 0) s.count[round & 1][warp] = make_uint4(c[0], c[1], c[2], c[3]);
    __syncthreads();
    const uint4 w = s.count[round & 1][lane % WARPS];
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    uint32_t nlo = lo, nhi = hi;
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      const uint32_t mine = lane < WARPS ? (j < 4 ? x[j] & 0xffffu : x[j - 4] >> 16) : 0u;
      if (int(__reduce_add_sync(0xffffffffu, mine)) >= r) nlo = p[j];
      else nhi = min(nhi, p[j] - 1);
    }
    lo = nlo;
    hi = nhi;
  }
  return lo;
}

}  // namespace q35
