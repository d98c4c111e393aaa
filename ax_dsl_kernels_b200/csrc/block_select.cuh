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
  uint32_t red[2][THREADS / 32];
  int warp_sum[THREADS / 32];
  int count[2][THREADS / 32][8];
  uint32_t list[KTH_LIST];
  int bin, rank, in_bin, listed;
};

// each(f) calls f(key) for every key of the calling thread; 1 <= r <= number of keys in the block.  Returns the r-th
// largest key to every thread.
//
// A histogram of 1024 bins between the smallest and the largest key, evenly spaced by value (BY_VALUE: scores, which
// spread like a normal distribution) or by key (weights, which spread over octaves), finds the bin that holds the r-th;
// up to 64 keys of it are ranked directly, more get a histogram of their own.  Keys that three histograms do not
// separate (far outliers, infinite ends) are left to pivots: seven at a time cut the interval, the keys at or above each
// of them are counted, an eighth of the interval stays, so that 11 rounds end it whatever the keys.
template <int THREADS, bool BY_VALUE, typename Each>
__device__ uint32_t block_kth(Each each, int r, KthScratch<THREADS>& s) {
  constexpr int WARPS = THREADS / 32, PER = KTH_BINS / THREADS;
  static_assert(KTH_BINS % THREADS == 0 && WARPS <= 32, "whole bins per thread");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t lo = 0u, hi = 0xffffffffu;
  int rank = r;  // among the keys in [lo, hi]
  auto tighten = [&](auto in) {  // lo, hi = smallest and largest key with in(key)
    uint32_t least = 0xffffffffu, most = 0u;
    each([&](uint32_t k) {
      if (in(k)) { least = min(least, k); most = max(most, k); }
    });
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();  // what was read from the scratch before
    if (lane == 0) { s.red[0][warp] = least; s.red[1][warp] = most; }
#pragma unroll
    for (int i = 0; i < PER; ++i) s.hist[tid + i * THREADS] = 0;
    if (tid == 0) s.listed = 0;
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, s.red[0][lane % WARPS]);
    hi = __reduce_max_sync(0xffffffffu, s.red[1][lane % WARPS]);
  };
  tighten([](uint32_t) { return true; });
  for (int level = 0; level < 3; ++level) {
    if (lo == hi) return lo;
    const float vlo = key_value(lo), scale = (KTH_BINS - 1) / (BY_VALUE ? key_value(hi) - vlo : float(hi - lo));
    if (!(scale > 0.f && scale < INFINITY)) break;
    const uint32_t from = lo, to = hi;
    // rounding keeps the order, so a bin holds an interval of keys
    auto bin_of = [&](uint32_t k) {
      return min(KTH_BINS - 1, int((BY_VALUE ? key_value(k) - vlo : float(k - from)) * scale));
    };
    each([&](uint32_t k) {
      if (k >= from && k <= to) atomicAdd(&s.hist[bin_of(k)], 1);
    });
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
      if (before < rank && rank <= before + cnt[i]) {
        s.bin = KTH_BINS - 1 - (tid * PER + i);
        s.rank = rank - before;
        s.in_bin = cnt[i];
      }
      before += cnt[i];
    }
    __syncthreads();
    const int bin = s.bin, n = s.in_bin;
    rank = s.rank;
    if (n <= KTH_LIST) {
      each([&](uint32_t k) {
        if (k >= from && k <= to && bin_of(k) == bin) s.list[atomicAdd(&s.listed, 1)] = k;
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
    tighten([&](uint32_t k) { return k >= from && k <= to && bin_of(k) == bin; });
  }
  for (int round = 0; lo < hi; ++round) {  // at least r keys are >= lo, fewer than r are > hi
    uint32_t p[7];  // ascending, in (lo, hi]
    int c[7];
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      p[j] = lo + max(uint32_t((uint64_t(hi - lo) * (j + 1)) >> 3), 1u);
      c[j] = 0;
    }
    each([&](uint32_t k) {
#pragma unroll
      for (int j = 0; j < 7; ++j) c[j] += k >= p[j];
    });
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      c[j] = __reduce_add_sync(0xffffffffu, c[j]);
      if (lane == 0) s.count[round & 1][warp][j] = c[j];
    }
    __syncthreads();
    uint32_t nlo = lo, nhi = hi;
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      const int mine = lane < WARPS ? s.count[round & 1][lane % WARPS][j] : 0;
      if (__reduce_add_sync(0xffffffffu, mine) >= r) nlo = p[j];
      else nhi = min(nhi, p[j] - 1);
    }
    lo = nlo;
    hi = nhi;
  }
  return lo;
}

}  // namespace q35
