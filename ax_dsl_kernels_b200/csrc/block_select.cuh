// The r-th largest of many floats by one thread block (attn.select_pages) or a cluster of them (attn.evict), as
// order_key's integers.
#pragma once
#include <cooperative_groups.h>
#include "attn_pages.cuh"

namespace q35 {

// order_key's inverse
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

constexpr int KTH_BITS = 10, KTH_BINS = 1 << KTH_BITS, KTH_LIST = 64;

template <int THREADS>
struct KthScratch {
  int hist[KTH_BINS];
  uint32_t red[2][THREADS / 32];
  int warp_sum[THREADS / 32];
  int count[2][THREADS / 32][8];
  uint32_t list[KTH_LIST], all[KTH_LIST], found;
  uint32_t ends[2];        // of this block's keys, read by its cluster
  int total[2][7];         // likewise
  int above[KTH_LIST], same[KTH_LIST];
  int bin, rank, in_bin, listed;
};

// each(f) calls f(key) for every key of the calling thread; 1 <= r <= number of keys in the block, or (CLUSTER) in the
// blocks of the cluster together, which all call this.  Returns the r-th largest key to every thread.  Blocks of a cluster
// read each other's scratch: none may leave before the cluster has met once more.
//
// A histogram of 1024 bins between the smallest and the largest key, evenly spaced by value (BY_VALUE: scores, which
// spread like a normal distribution) or by key (weights, which spread over octaves), finds the bin that holds the r-th;
// up to 64 keys of it are ranked directly, more get a histogram of their own.  Keys that three histograms do not
// separate (far outliers, infinite ends) are left to pivots: seven at a time cut the interval, the keys at or above each
// of them are counted, an eighth of the interval stays, so that 11 rounds end it whatever the keys.
template <int THREADS, bool BY_VALUE, bool CLUSTER = false, typename Each>
__device__ uint32_t block_kth(Each each, int r, KthScratch<THREADS>& s) {
  namespace cg = cooperative_groups;
  constexpr int WARPS = THREADS / 32, PER = KTH_BINS / THREADS;
  static_assert(KTH_BINS % THREADS == 0 && WARPS <= 32, "whole bins per thread");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t lo = 0u, hi = 0xffffffffu;
  int rank = r;  // among the keys in [lo, hi]
  cg::cluster_group cluster = cg::this_cluster();
  const int NC = CLUSTER ? int(cluster.num_blocks()) : 1;
  auto sync = [&] {
    if constexpr (CLUSTER) cluster.sync();
    else __syncthreads();
  };
  auto of = [&](int block, auto* p) { return CLUSTER ? cluster.map_shared_rank(p, block) : p; };
  auto tighten = [&](auto in) {  // lo, hi = smallest and largest key with in(key)
    uint32_t least = 0xffffffffu, most = 0u;
    each([&](uint32_t k) {
      if (in(k)) { least = min(least, k); most = max(most, k); }
    });
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    sync();  // what was read from the scratch before
    if (lane == 0) { s.red[0][warp] = least; s.red[1][warp] = most; }
#pragma unroll
    for (int i = 0; i < PER; ++i) s.hist[tid + i * THREADS] = 0;
    if (tid == 0) s.listed = 0;
    if (tid < KTH_LIST) s.above[tid] = s.same[tid] = 0;
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, s.red[0][lane % WARPS]);
    hi = __reduce_max_sync(0xffffffffu, s.red[1][lane % WARPS]);
    if constexpr (CLUSTER) {
      if (tid == 0) { s.ends[0] = lo; s.ends[1] = hi; }
      sync();
      lo = __reduce_min_sync(0xffffffffu, of(lane % NC, s.ends)[0]);
      hi = __reduce_max_sync(0xffffffffu, of(lane % NC, s.ends)[1]);
    }
  };
  tighten([](uint32_t) { return true; });
  for (int level = 0; level < 3; ++level) {
    if (lo == hi) return lo;
    const uint32_t from = lo, to = hi;
    const float vlo = key_value(lo), scale = (KTH_BINS - 1) / (key_value(hi) - vlo);
    const int shift = max(0, 32 - KTH_BITS - __clz(hi - lo));  // hi - lo < KTH_BINS << shift
    if (BY_VALUE && !(scale > 0.f && scale < INFINITY)) break;
    auto bin_of = [&](uint32_t k) {  // rounding keeps the order, so a bin holds an interval of keys either way
      return BY_VALUE ? min(KTH_BINS - 1, int((key_value(k) - vlo) * scale)) : int((k - from) >> shift);
    };
    each([&](uint32_t k) {
      if (k >= from && k <= to) atomicAdd(&s.hist[bin_of(k)], 1);
    });
    sync();
    int cnt[PER], sum = 0;  // thread t owns the bins PER t .. PER t + PER - 1 counted from the top
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      cnt[i] = 0;
#pragma unroll 4
      for (int k = 0; k < NC; ++k) cnt[i] += of(k, s.hist)[KTH_BINS - 1 - (tid * PER + i)];
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
      sync();
      if constexpr (CLUSTER) {  // the blocks' lists behind one another
        const int from_block = tid / KTH_LIST, at = tid % KTH_LIST;
        if (from_block < NC) {
          int before_it = 0;
          for (int k = 0; k < from_block; ++k) before_it += *of(k, &s.listed);
          if (at < *of(from_block, &s.listed)) s.all[before_it + at] = of(from_block, s.list)[at];
        }
        __syncthreads();
      }
      const uint32_t* list = CLUSTER ? s.all : s.list;
      // every key of the list against every other, a part of them per thread: the one with fewer than rank keys above it
      // and rank at or above it
      const int i = tid % KTH_LIST;
      if (i < n) {
        const uint32_t k = list[i];
        int above = 0, same = 0;
        for (int j = tid / KTH_LIST; j < n; j += THREADS / KTH_LIST) {
          above += list[j] > k;
          same += list[j] == k;
        }
        if (above) atomicAdd(&s.above[i], above);
        if (same) atomicAdd(&s.same[i], same);
      }
      __syncthreads();
      if (tid < n && s.above[tid] < rank && rank <= s.above[tid] + s.same[tid]) s.found = list[tid];
      __syncthreads();
      return s.found;
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
    for (int j = 0; j < 7; ++j) c[j] = __reduce_add_sync(0xffffffffu, lane < WARPS ? s.count[round & 1][lane % WARPS][j] : 0);
    if constexpr (CLUSTER) {
      if (tid == 0) {
#pragma unroll
        for (int j = 0; j < 7; ++j) s.total[round & 1][j] = c[j];
      }
      sync();
#pragma unroll
      for (int j = 0; j < 7; ++j) c[j] = __reduce_add_sync(0xffffffffu, lane < NC ? of(lane % NC, s.total[round & 1])[j] : 0);
    }
#pragma unroll
    for (int j = 0; j < 7; ++j) {
      if (c[j] >= r) nlo = p[j];
      else nhi = min(nhi, p[j] - 1);
    }
    lo = nlo;
    hi = nhi;
  }
  return lo;
}

}  // namespace q35
