// attn.evict: every (sequence, KV head) keeps the min(K, ctx) cached rows with the highest key_mass -- the first and the
// last ones always, ties to the lower position -- and moves them, in order, to the sequence's first rows, in place.
//
// evict_choose, one CTA per (sequence, KV head): the weights once into shared memory as ordered integers, the border by
// block_kth, then one pass that writes the kept positions in ascending order.
// evict_move: row j of the result is row kept[j] >= j of the cache.  Bound: HBM, every row that changes place read and
// written once.
//
// In place and in parallel: a cluster takes the kept rows in rounds of consecutive j.  A round stores to rows below its
// end j1, later rounds load from rows kept[j] >= j >= j1, so loads may run ahead of stores as they like; a round's stores
// only have to wait until the whole cluster has loaded that round.  A thread owns one row of the round: it asks for its
// K and V rows with two bulk copies, and a round later, after the cluster's barrier, sends them off with two more.  No
// data passes through registers, and two rounds' bytes are on their way per CTA.
// (One CTA per 64-byte column slice, with the rows through registers: 121 us instead of MOVE at 32 x 4000 bf16 rows.)
#include <cooperative_groups.h>
#include "abi.h"
#include "attn_pages.cuh"
#include "block_select.cuh"
#include "tc_ptx.cuh"

namespace q35 {

namespace cg = cooperative_groups;

struct EvictArgs {
  PageTable t;
  uint8_t* cache;
  __nv_bfloat16* row_scale;    // int8 cache
  float* key_mass;             // [pages, P, HKV]
  const int* keep;             // optional [2]: first, last
  int* kept;                   // [B, HKV, K]
  uint32_t* keys;              // workspace [HKV * n_indices * P], for rows that do not fit the shared memory
  int HKV, K, row_bytes;       // row_bytes of one head
  int cap;                     // rows whose keys fit the shared memory
  int per_round;               // rows per CTA and round of moves
};

constexpr int EV_THREADS = 1024;
constexpr int EV_CAP = 48 * 1024;   // keys in shared memory: 192 KB
constexpr int EV_U = 8;             // positions per thread on their way together

__global__ void __launch_bounds__(EV_THREADS) evict_choose_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ KthScratch<EV_THREADS> s_kth;
  __shared__ int s_count[EV_U][32], s_total, s_gt[32], s_eq[32];
  pdl_wait();
  pdl_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int b = blockIdx.x / a.HKV, h = blockIdx.x % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  const int n = sp.ctx, K = a.K, P = a.t.P;
  int* out = a.kept + size_t(blockIdx.x) * K;
  if (n <= K) {
    for (int i = tid; i < K; i += EV_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int last = a.keep ? min(max(a.keep[1], 0), K) : 0;
  const int first = a.keep ? min(max(a.keep[0], 0), K - last) : 0;
  const int rank = K - first - last;
  // keys of the free positions first .. n - last - 1, the forced ones' slots unused
  uint32_t* keys = n <= a.cap ? s_keys : a.keys + (size_t(a.HKV) * sp.first + size_t(h) * sp.n) * P;
  const int f0 = first, f1 = n - last;
  uint32_t border = 0u;
  int equal = 0;         // how many of the rows that equal the border are kept
  bool ties = false;     // and whether that is not all of them
  if (rank > 0) {
    bool bad = false;
    for (int i0 = f0 + tid; i0 < f1; i0 += EV_U * EV_THREADS) {
      int page[EV_U], off[EV_U];
#pragma unroll
      for (int u = 0; u < EV_U; ++u) {
        const int i = min(i0 + u * EV_THREADS, f1 - 1), e = a.t.page_of(i);
        page[u] = page_or_first(a.t, sp.first + e, bad);
        off[u] = i - e * P;
      }
      float w[EV_U];
#pragma unroll
      for (int u = 0; u < EV_U; ++u) w[u] = a.key_mass[(size_t(page[u]) * P + off[u]) * a.HKV + h];
#pragma unroll
      for (int u = 0; u < EV_U; ++u)
        if (i0 + u * EV_THREADS < f1) keys[i0 + u * EV_THREADS] = order_key(w[u]);
    }
    if (bad) atomicOr(a.t.status, DS_BAD_PAGE);
    // a thread reads only the keys that it wrote itself until the barriers of block_kth are behind it
    auto each = [&](auto f) {
      for (int i = f0 + tid; i < f1; i += EV_THREADS) f(keys[i]);
    };
    border = block_kth<EV_THREADS, false>(each, rank, s_kth);
    int gt = 0, eq = 0;
    each([&](uint32_t k) {
      gt += k > border;
      eq += k == border;
    });
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) { s_gt[warp] = gt; s_eq[warp] = eq; }
    __syncthreads();
    equal = rank - __reduce_add_sync(0xffffffffu, s_gt[lane]);
    ties = equal != __reduce_add_sync(0xffffffffu, s_eq[lane]);
  }
  // how many flags are set before each of the thread's positions c0 + u * EV_THREADS + tid, and in all (s_total)
  auto scan = [&](const bool (&flag)[EV_U], int (&at)[EV_U]) {
    unsigned ball[EV_U];
#pragma unroll
    for (int u = 0; u < EV_U; ++u) {
      ball[u] = __ballot_sync(0xffffffffu, flag[u]);
      if (lane == 0) s_count[u][warp] = __popc(ball[u]);
    }
    __syncthreads();
    if (warp == 0) {  // EV_U * 32 counts, EV_U consecutive ones to a lane
      int* cnt = &s_count[0][0] + EV_U * lane;
      int sum = 0, c[EV_U];
#pragma unroll
      for (int u = 0; u < EV_U; ++u) { c[u] = sum; sum += cnt[u]; }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
#pragma unroll
      for (int u = 0; u < EV_U; ++u) cnt[u] = inc - sum + c[u];
      if (lane == 31) s_total = inc;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < EV_U; ++u) at[u] = s_count[u][warp] + __popc(ball[u] & ((1u << lane) - 1));
  };
  int done = 0, seen = 0;  // kept rows, and rows equal to the border, before this round of positions
  for (int c0 = 0; c0 < n; c0 += EV_U * EV_THREADS) {
    bool take[EV_U], eq[EV_U];
    int at[EV_U];
#pragma unroll
    for (int u = 0; u < EV_U; ++u) {
      const int i = c0 + u * EV_THREADS + tid;
      const bool free_row = i >= f0 && i < f1 && rank > 0;
      const uint32_t k = free_row ? keys[i] : 0u;
      eq[u] = free_row && k == border;
      take[u] = i < n && (i < f0 || i >= f1 || (free_row && k > border));
    }
    if (ties) {
      scan(eq, at);
#pragma unroll
      for (int u = 0; u < EV_U; ++u) eq[u] = eq[u] && seen + at[u] < equal;
      seen += s_total;
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < EV_U; ++u) take[u] |= eq[u];
    scan(take, at);
#pragma unroll
    for (int u = 0; u < EV_U; ++u)
      if (take[u] && done + at[u] < K) out[done + at[u]] = c0 + u * EV_THREADS + tid;
    done += s_total;
    __syncthreads();
  }
}

constexpr int EM_THREADS = 256;
constexpr int EM_BUF = 96 * 1024;  // bytes of a round per CTA; two rounds

__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(smem_dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_src), "r"(bytes) : "memory");
}

__global__ void __launch_bounds__(EM_THREADS, 1) evict_move_kernel(const EvictArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_bar[2];
  const uint32_t bar = smem_u32(s_bar);
  const int tid = threadIdx.x;
  if (tid == 0) {
    tc::mbar_init(bar, EM_THREADS);
    tc::mbar_init(bar + 8, EM_THREADS);
    tc::fence_barrier_init();
    tc::fence_proxy_async();
  }
  __syncthreads();
  pdl_wait();
  pdl_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int NC = int(cluster.num_blocks()), crank = int(cluster.block_rank());
  const int row = blockIdx.x / NC, b = row / a.HKV, h = row % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  if (sp.ctx <= a.K) return;  // everything stays where it is: the whole cluster leaves
  const int n = a.K, P = a.t.P, R = a.per_round;
  const int* kept = a.kept + size_t(row) * a.K;
  const int rounds = (n + NC * R - 1) / (NC * R);
  const uint32_t mine = smem_u32(smem) + uint32_t(tid) * 2 * a.row_bytes;  // this thread's K and V row in buffer 0
  // row (position) -> index of its K row among all rows of the cache; -1 where the table names no page
  auto row_of = [&](int pos) -> int64_t {
    const int e = a.t.page_of(pos), page = a.t.indices[sp.first + e];
    return unsigned(page) < unsigned(a.t.num_pages) ? (int64_t(page) * 2 * P + (pos - e * P)) * a.HKV + h : -1;
  };
  const int64_t v_rows = int64_t(P) * a.HKV;  // from a K row to its V row
  auto mass_at = [&](int64_t r) {  // [pages, 2, P, HKV] -> [pages, P, HKV]
    const int64_t page = r / (2 * v_rows);
    return a.key_mass + (r - page * v_rows);
  };
  // this thread's row of a round: from where to where, -1 = nothing to do
  int64_t from[2] = {-1, -1}, to[2] = {-1, -1};
  float mass[2] = {0.f, 0.f};
  __nv_bfloat16 ks[2] = {}, vs[2] = {};
  auto look_up = [&](int i, int64_t& src, int64_t& dst) {
    const int j = (i * NC + crank) * R + tid;
    src = dst = -1;
    if (i < rounds && tid < R && j < n) {
      const int pos = kept[j];
      if (pos > j && pos < sp.ctx) {
        src = row_of(pos);
        dst = row_of(j);
        if (src < 0 || dst < 0) {
          atomicOr(a.t.status, DS_BAD_PAGE);
          src = dst = -1;
        }
      }
    }
  };
  auto load = [&](int u) {  // u: buffer
    const uint32_t at = mine + u * EM_BUF, bu = bar + 8 * u;
    if (from[u] >= 0) {
      tc::mbar_expect_tx(bu, 2 * a.row_bytes);
      const uint8_t* src = a.cache + from[u] * a.row_bytes;
      bulk_load(at, src, a.row_bytes, bu);
      bulk_load(at + a.row_bytes, src + v_rows * a.row_bytes, a.row_bytes, bu);
      mass[u] = *mass_at(from[u]);
      if (a.row_scale) {
        ks[u] = a.row_scale[from[u]];
        vs[u] = a.row_scale[from[u] + v_rows];
      }
    } else {
      tc::mbar_arrive(bu);
    }
  };
  auto step = [&](int i, auto cur, auto nxt) {  // cur, nxt: compile-time buffer numbers keep the registers indexed
    constexpr int U = decltype(cur)::value, V = decltype(nxt)::value;
    if (i + 1 < rounds) {
      look_up(i + 1, from[V], to[V]);
      asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the other buffer has been sent off
      load(V);
    }
    const bool ok = tc::mbar_wait(bar + 8 * U, (i >> 1) & 1);
    if (!ok) {  // recorded; nothing of this round is stored, and the copies on their way get as long again to land
      atomicOr(a.t.status, DS_WAIT_TIMEOUT);
      tc::mbar_wait(bar + 8 * U, (i >> 1) & 1);
    }
    cluster.sync();  // the whole cluster has loaded this round
    if (ok && to[U] >= 0) {
      const uint32_t at = mine + U * EM_BUF;
      uint8_t* dst = a.cache + to[U] * a.row_bytes;
      bulk_store(dst, at, a.row_bytes);
      bulk_store(dst + v_rows * a.row_bytes, at + a.row_bytes, a.row_bytes);
      *mass_at(to[U]) = mass[U];
      if (a.row_scale) {
        a.row_scale[to[U]] = ks[U];
        a.row_scale[to[U] + v_rows] = vs[U];
      }
    }
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  };
  look_up(0, from[0], to[0]);
  load(0);
  for (int i = 0; i < rounds; i += 2) {
    step(i, std::integral_constant<int, 0>(), std::integral_constant<int, 1>());
    if (i + 1 < rounds) step(i + 1, std::integral_constant<int, 1>(), std::integral_constant<int, 0>());
  }
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
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
  Q35_REQUIRE(a.row_bytes % 64 == 0, Q35_ERR_UNSUPPORTED, "%s: a row of a head must be a multiple of 64 bytes", role);
  Q35_REQUIRE(B * kv.HKV <= INT_MAX / 16, Q35_ERR_SHAPE, "%s: sizes beyond 32 bits", role);
  const int64_t positions = int64_t(a.t.n_indices) * kv.P;  // no sequence has more
  a.cap = int(positions < EV_CAP ? (positions + 31) / 32 * 32 : EV_CAP);
  Tensor ws;
  Q35_TRY(c.workspace(positions > EV_CAP ? positions * kv.HKV * 4 : 0, &ws));
  if (c.dry || B == 0) return 0;
  a.cache = static_cast<uint8_t*>(const_cast<void*>(kv.p));
  a.row_scale = const_cast<__nv_bfloat16*>(kv.row_scale);
  a.key_mass = mass.as<float>(); a.keep = keep.present ? keep.as<int>() : nullptr; a.kept = kept.as<int>();
  a.HKV = int(kv.HKV); a.K = int(kept.s[2]);
  a.keys = ws.present ? ws.as<uint32_t>() : nullptr;
  const int64_t rows = B * kv.HKV;
  Q35_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(evict_choose_kernel), EV_CAP * 4));
  launch_pdl(evict_choose_kernel, dim3(unsigned(rows)), dim3(EV_THREADS), size_t(a.cap) * 4, c.stream, a);
  Q35_CUDA_LAUNCH_CHECK("attn.evict choice");
  // as many CTAs per (sequence, KV head) as run at once on an SM each, while a round gives every one of them rows
  a.per_round = EM_BUF / (2 * a.row_bytes) < EM_THREADS ? EM_BUF / (2 * a.row_bytes) : EM_THREADS;
  int cluster = 1;
  while (cluster < 16 && rows * cluster * 2 <= sm_count() && int64_t(cluster) * a.per_round < a.K) cluster *= 2;
  const void* f = reinterpret_cast<const void*>(evict_move_kernel);
  Q35_TRY(ensure_dynamic_smem(f, 2 * EM_BUF));
  cudaError_t e = cudaSuccess;
  if (cluster > 8) e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(rows * cluster));
    cfg.blockDim = dim3(EM_THREADS);
    cfg.dynamicSmemBytes = 2 * EM_BUF;
    cfg.stream = c.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cluster); attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, evict_move_kernel, a);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the caller's next CUDA call
    return fail(Q35_ERR_CUDA, "attn.evict: %s", cudaGetErrorString(e));
  }
  Q35_CUDA_LAUNCH_CHECK("attn.evict moves");
  return 0;
}

}  // namespace q35
