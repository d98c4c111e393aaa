// attn.evict: every (sequence, KV head) keeps the min(K, ctx) cached rows with the highest key_mass -- the first and the
// last ones always, ties to the lower position -- and moves them, in order, to the sequence's first rows, in place.
//
// evict_choose, a cluster per (sequence, KV head): the weights once into registers as ordered integers, the border by
// block_kth, then one pass that writes the kept positions in ascending order.
// evict_move: row j of the result is row kept[j] >= j of the cache.  Bound: HBM, every row that changes place read and
// written once.
//
// In place and in parallel: a cluster takes the kept rows in rounds of consecutive j.  A round stores to rows below its
// end j1, later rounds load from rows kept[j] >= j >= j1, so loads may run ahead of stores as they like; a round's stores
// only have to wait until the whole cluster has loaded that round.  A warp owns whole rows of a round: cp.async brings
// them into its part of the shared memory, and it stores them from there while the cluster's barrier for the next round
// closes and the one after that is on its way.  (An SM stores 27 bytes a cycle here; loads and barriers hide behind it.)
// (Choice and moves, 32 x 4000 of up to 16384 bf16 rows, calls among others: one CTA per 64-byte column slice, without clusters, 175 us; this
// 50, with a choice by one CTA per row 60.  115 MB read and written take 35 us at HBM's rate.  One bulk copy per row and
// direction instead of cp.async and stores: as long.)
#include <cooperative_groups.h>
#include "abi.h"
#include "attn_pages.cuh"
#include "block_select.cuh"

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
  int cap;                     // rows whose keys fit a CTA's shared memory
  int per_warp;                // rows per warp and round of moves
  int planes;                  // of a row per CTA: 2 = K and V, 1 = one of them (blockIdx.y)
};

constexpr int EV_THREADS = 1024;
constexpr int EV_REGS = 16;         // most keys per thread in registers: 16384 rows per CTA
constexpr int EV_CAP = 48 * 1024;   // keys in shared memory, 192 KB, where the registers do not hold them
constexpr int EV_U = 8;             // most positions per thread and round

struct ChooseScratch {
  KthScratch<EV_THREADS> kth;
  int count[2][EV_U][32], gt[32], eq[32];
  int sums[2];  // rows above the border and rows equal to it, read by the cluster
};

// The choice for one (sequence, KV head) of n > K rows, by a cluster: every CTA takes a range of positions, whose keys it
// holds -- key(m) is that of position p0 + m * 1024 + t, set by put(m, key) -- and writes the kept ones among them.
// M: static number of keys per thread (0: as many as there are, in a loop).
template <int M, typename Put, typename Key>
__device__ __forceinline__ void evict_choose(const EvictArgs& a, const SeqPages& sp, int h, int p0, int p1, int* out,
                                             ChooseScratch& s, Put put, Key key) {
  constexpr int U = M && M < EV_U ? M : EV_U;
  cg::cluster_group cluster = cg::this_cluster();
  const int NC = int(cluster.num_blocks()), crank = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = sp.ctx, K = a.K, P = a.t.P;
  const int last = a.keep ? min(max(a.keep[1], 0), K) : 0;
  const int first = a.keep ? min(max(a.keep[0], 0), K - last) : 0;
  const int rank = K - first - last, f0 = first, f1 = n - last;  // the free rows, of which `rank` are kept
  const int rounds = M ? M : (p1 - p0 + EV_THREADS - 1) / EV_THREADS;
  auto position = [&](int m) { return p0 + m * EV_THREADS + tid; };
  auto is_free = [&](int m) {
    const int i = position(m);
    return i >= f0 && i < f1 && i < p1;
  };
  uint32_t border = 0u;
  int equal = 0;         // how many of the rows that equal the border are kept
  bool ties = false;     // and whether that is not all of them
  int seen = 0;          // rows equal to the border before this round of positions
  int done = min(p0, f0) + max(0, p0 - f1);  // and kept rows
  if (rank > 0) {
    bool bad = false;
#pragma unroll
    for (int m0 = 0; m0 < rounds; m0 += U) {
      int page[U], off[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(position(m0 + u), n - 1), e = a.t.page_of(i);
        page[u] = page_or_first(a.t, sp.first + e, bad);
        off[u] = i - e * P;
      }
      float w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = a.key_mass[(size_t(page[u]) * P + off[u]) * a.HKV + h];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (M || position(m0 + u) < p1) put(m0 + u, order_key(w[u]));
    }
    if (bad) atomicOr(a.t.status, DS_BAD_PAGE);
    auto each = [&](auto f) {
#pragma unroll
      for (int m = 0; m < rounds; ++m)
        if (is_free(m)) f(key(m));
    };
    border = block_kth<EV_THREADS, false, true>(each, rank, s.kth);
    int gt = 0, eq = 0;
    each([&](uint32_t k) {
      gt += k > border;
      eq += k == border;
    });
    gt = __reduce_add_sync(0xffffffffu, gt);
    eq = __reduce_add_sync(0xffffffffu, eq);
    if (lane == 0) { s.gt[warp] = gt; s.eq[warp] = eq; }
    __syncthreads();
    gt = __reduce_add_sync(0xffffffffu, s.gt[lane]);
    eq = __reduce_add_sync(0xffffffffu, s.eq[lane]);
    if (tid == 0) { s.sums[0] = gt; s.sums[1] = eq; }
    cluster.sync();
    const int* sums = cluster.map_shared_rank(s.sums, lane % NC);
    gt = lane < NC ? sums[0] : 0;
    eq = lane < NC ? sums[1] : 0;
    equal = rank - __reduce_add_sync(0xffffffffu, gt);
    ties = equal != __reduce_add_sync(0xffffffffu, eq);
    seen = __reduce_add_sync(0xffffffffu, lane < crank ? eq : 0);
    done += __reduce_add_sync(0xffffffffu, lane < crank ? gt : 0) + min(seen, equal);
  }
  auto gathered = cluster.barrier_arrive();  // nobody reads another's scratch from here on
  // how many flags are set before each of the thread's positions of a round; returns how many in all.  Calls alternate
  // between two sets of counts: one barrier each.
  int turn = 0;
  auto scan = [&](const bool (&flag)[U], int (&at)[U]) {
    int (&count)[EV_U][32] = s.count[turn ^= 1];
    unsigned ball[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ball[u] = __ballot_sync(0xffffffffu, flag[u]);
      if (lane == 0) count[u][warp] = __popc(ball[u]);
    }
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = count[u][lane];
      at[u] = total + __reduce_add_sync(0xffffffffu, lane < warp ? c : 0) + __popc(ball[u] & ((1u << lane) - 1));
      total += __reduce_add_sync(0xffffffffu, c);
    }
    return total;
  };
#pragma unroll
  for (int m0 = 0; m0 < rounds; m0 += U) {
    if (p0 + m0 * EV_THREADS >= p1) break;
    bool take[U], eq[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int m = m0 + u, i = position(m);
      const bool free_row = is_free(m) && rank > 0;
      const uint32_t k = free_row ? key(m) : 0u;
      eq[u] = free_row && k == border;
      take[u] = i < p1 && (i < f0 || i >= f1 || (free_row && k > border));
    }
    if (ties) {
      const int total = scan(eq, at);
#pragma unroll
      for (int u = 0; u < U; ++u) eq[u] = eq[u] && seen + at[u] < equal;
      seen += total;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) take[u] |= eq[u];
    const int total = scan(take, at);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (take[u] && done + at[u] < K) out[done + at[u]] = position(m0 + u);
    done += total;
  }
  cluster.barrier_wait(std::move(gathered));
}

__global__ void __launch_bounds__(EV_THREADS) evict_choose_kernel(const EvictArgs a) {
  extern __shared__ __align__(16) uint32_t s_keys[];
  __shared__ ChooseScratch s;
  pdl_wait();
  pdl_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int NC = int(cluster.num_blocks()), crank = int(cluster.block_rank());
  const int tid = threadIdx.x, row = blockIdx.x / NC, b = row / a.HKV, h = row % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  int* out = a.kept + size_t(row) * a.K;
  if (sp.ctx <= a.K) {  // the whole cluster
    for (int i = crank * EV_THREADS + tid; i < a.K; i += NC * EV_THREADS) out[i] = i < sp.ctx ? i : -1;
    return;
  }
  const int part = (sp.ctx + NC - 1) / NC, p0 = min(sp.ctx, crank * part), p1 = min(sp.ctx, p0 + part);
  auto in_registers = [&](auto m) {
    uint32_t k[decltype(m)::value];
    evict_choose<decltype(m)::value>(a, sp, h, p0, p1, out, s, [&](int i, uint32_t x) { k[i] = x; },
                                     [&](int i) { return k[i]; });
  };
  if (part <= 2 * EV_THREADS) in_registers(std::integral_constant<int, 2>());
  else if (part <= 4 * EV_THREADS) in_registers(std::integral_constant<int, 4>());
  else if (part <= 8 * EV_THREADS) in_registers(std::integral_constant<int, 8>());
  else if (part <= EV_REGS * EV_THREADS) in_registers(std::integral_constant<int, EV_REGS>());
  else {
    uint32_t* keys = part <= a.cap ? s_keys : a.keys + (size_t(a.HKV) * sp.first + size_t(h) * sp.n) * a.t.P + p0;
    evict_choose<0>(a, sp, h, p0, p1, out, s, [&](int m, uint32_t x) { keys[m * EV_THREADS + tid] = x; },
                    [&](int m) { return keys[m * EV_THREADS + tid]; });
  }
}

constexpr int EM_THREADS = 512, EM_WARPS = EM_THREADS / 32;
constexpr int EM_BUF = 64 * 1024;  // bytes of a round per CTA; three rounds
constexpr int EM_PIECES = 8;       // most 16-byte pieces of a row (K and V) per lane: rows of up to 2048 bytes

template <int PL>
__global__ void __launch_bounds__(EM_THREADS, 1) evict_move_kernel(const EvictArgs a) {
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int NC = int(cluster.num_blocks()), crank = int(cluster.block_rank());
  const int row = blockIdx.x / NC, b = row / a.HKV, h = row % a.HKV;
  const SeqPages sp = seq_pages(a.t, b);
  if (sp.ctx <= a.K) return;  // everything stays where it is: the whole cluster leaves
  const int n = a.K, P = a.t.P, RW = a.per_warp, R = RW * EM_WARPS;
  const int* kept = a.kept + size_t(row) * a.K;
  const int rounds = (n + NC * R - 1) / (NC * R);
  const int64_t v_rows = int64_t(P) * a.HKV;  // from a K row to its V row, in rows
  auto mass_at = [&](int64_t r) {             // [pages, 2, P, HKV] -> [pages, P, HKV]
    const int64_t page = r / (2 * v_rows);
    return a.key_mass + (r - page * v_rows);
  };
  // Lane l < RW of a warp knows the warp's row l of a round: from where to where, -1 = nothing to do.  The lookups run
  // ahead of the copies, one step of their chain (kept position, page ids, rows) per round, so that no round waits for
  // the page table.
  int64_t from[3] = {-1, -1, -1}, to[3] = {-1, -1, -1};
  float mass[3] = {0.f, 0.f, 0.f};
  __nv_bfloat16 ks[3] = {}, vs[3] = {};
  auto index_of = [&](int i) { return (i * NC + crank) * R + warp * RW + lane; };
  auto position = [&](int i) -> int {  // kept position of the row of round i, -1 where there is none
    const int j = index_of(i);
    return i < rounds && lane < RW && j < n ? kept[j] : -1;
  };
  int pos_next, pos_cur, src_page, dst_page;  // position of round i + 3; position and page ids of round i + 2
  auto ask_pages = [&](int i) {               // page ids of round i, whose position is in pos_cur
    const int j = index_of(i);
    src_page = dst_page = -1;
    if (pos_cur > j && pos_cur < sp.ctx) {
      src_page = a.t.indices[sp.first + a.t.page_of(pos_cur)];
      dst_page = a.t.indices[sp.first + a.t.page_of(j)];
    } else {
      pos_cur = -1;
    }
  };
  auto row_at = [&](int page, int pos) { return (int64_t(page) * 2 * P + (pos - a.t.page_of(pos) * P)) * a.HKV + h; };
  auto resolve = [&](int i, int64_t& src, int64_t& dst) {
    src = dst = -1;
    if (pos_cur < 0) return;
    if (unsigned(src_page) < unsigned(a.t.num_pages) && unsigned(dst_page) < unsigned(a.t.num_pages)) {
      src = row_at(src_page, pos_cur);
      dst = row_at(dst_page, index_of(i));
    } else {
      atomicOr(a.t.status, DS_BAD_PAGE);
    }
  };
  // 16-byte pieces, pp to a row (K, then V, or one of them): a lane's PL pieces of every row that it takes part in, `rows` rows to an
  // instruction of the warp where a row has fewer than 32
  const int pr = a.row_bytes / 16, pp = a.planes * pr, rows = pp < 32 ? 32 / pp : 1;
  const int sub = pp < 32 ? lane / pp : 0, piece0 = pp < 32 ? lane % pp : lane;
  const int64_t v_off = v_rows * a.row_bytes, own_off = blockIdx.y ? v_off : 0;
  const bool has_k = blockIdx.y == 0, has_v = a.planes == 2 || blockIdx.y == 1;
  int64_t in_cache[PL];
  bool has[PL];
#pragma unroll
  for (int q = 0; q < PL; ++q) {
    const int p = piece0 + 32 * q;
    has[q] = sub < rows && p < pp;
    in_cache[q] = p < pr ? own_off + p * 16 : v_off + (p - pr) * 16;
  }
  uint8_t* const ring = smem + size_t(warp) * RW * a.planes * a.row_bytes;  // the warp's rows in buffer 0
  auto pieces = [&](int64_t where, auto f) {  // f(address in the cache, offset in the warp's buffer) for every piece
    const unsigned long long mine = where >= 0 ? reinterpret_cast<unsigned long long>(a.cache) + where * a.row_bytes : 0ull;
#pragma unroll 4
    for (int r0 = 0; r0 < RW; r0 += rows) {
      const int l = r0 + sub;
      uint8_t* at = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, mine, l & 31));
      if (l >= RW) at = nullptr;
#pragma unroll
      for (int q = 0; q < PL; ++q)
        if (at && has[q]) f(at + in_cache[q], (l * pp + piece0 + 32 * q) * 16);
    }
  };
  auto load = [&](int i, int u) {  // round i, looked up, into buffer u; then the next lookups
    resolve(i, from[u], to[u]);
    __syncwarp();  // the warp has read what the buffer held
    const uint32_t base = smem_u32(ring) + u * EM_BUF;
    pieces(from[u], [&](uint8_t* src, int off) { cp_async_16(base + off, src); });
    cp_async_commit();
    if (from[u] >= 0) {
      if (has_k) mass[u] = *mass_at(from[u]);
      if (a.row_scale) {
        if (has_k) ks[u] = a.row_scale[from[u]];
        if (has_v) vs[u] = a.row_scale[from[u] + v_rows];
      }
    }
    pos_cur = pos_next;
    ask_pages(i + 1);
    pos_next = position(i + 2);
  };
  auto store = [&](int u) {
    const uint8_t* base = ring + u * EM_BUF;
    pieces(to[u], [&](uint8_t* dst, int off) {
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(base + off);
    });
    if (to[u] >= 0) {
      if (has_k) *mass_at(to[u]) = mass[u];
      if (a.row_scale) {
        if (has_k) a.row_scale[to[u]] = ks[u];
        if (has_v) a.row_scale[to[u] + v_rows] = vs[u];
      }
    }
  };
  // Round i has arrived: tell the cluster, store round i - 1 meanwhile (the cluster has loaded that one), ask for i + 2.
  auto step = [&](int i, auto cur, auto prv) {  // compile-time buffer numbers keep the registers indexed
    cp_async_wait<1>();
    auto token = cluster.barrier_arrive();
    if (i > 0) store(decltype(prv)::value);
    cluster.barrier_wait(std::move(token));
    load(i + 2, decltype(prv)::value);
    if (i + 1 == rounds) store(decltype(cur)::value);
  };
  pos_cur = position(0);
  pos_next = position(1);
  ask_pages(0);
  load(0, 0);
  load(1, 1);
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  using B2 = std::integral_constant<int, 2>;
  for (int i = 0; i < rounds; i += 3) {
    step(i, B0(), B2());
    if (i + 1 < rounds) step(i + 1, B1(), B0());
    if (i + 2 < rounds) step(i + 2, B2(), B1());
  }
}

template <typename F>
static int launch_evict(F f, const EvictArgs& a, dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (cluster > 8) e = cudaFuncSetAttribute(reinterpret_cast<const void*>(f), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(cluster); attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, f, a);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();  // reported here, not by the caller's next CUDA call
    return fail(Q35_ERR_CUDA, "attn.evict: %s", cudaGetErrorString(e));
  }
  Q35_CUDA_LAUNCH_CHECK("attn.evict");
  return 0;
}

template <int PL>
static int launch_evict_move(const EvictArgs& a, int rows, int cluster, cudaStream_t stream) {
  Q35_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(evict_move_kernel<PL>), 3 * EM_BUF));
  return launch_evict(evict_move_kernel<PL>, a, dim3(unsigned(rows * cluster), unsigned(2 / a.planes)), EM_THREADS,
                      3 * EM_BUF, cluster, stream);
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
  Q35_REQUIRE(a.row_bytes <= 256 * EM_PIECES, Q35_ERR_UNSUPPORTED, "%s: a row of a head has %d bytes, at most 2048", role,
              a.row_bytes);
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
  // as many CTAs per (sequence, KV head) as there are SMs for and rows of the average sequence to give each two a thread
  int choosers = 1;
  while (choosers < 8 && rows * choosers * 2 <= sm_count() && positions > B * choosers * 2 * EV_THREADS) choosers *= 2;
  // (no keys in shared memory where every sequence fits the registers)
  Q35_TRY(launch_evict(evict_choose_kernel, a, dim3(unsigned(rows * choosers)), EV_THREADS,
                       positions > int64_t(choosers) * EV_REGS * EV_THREADS ? size_t(a.cap) * 4 : 0, choosers, c.stream));
  // as many CTAs per (sequence, KV head) as run at once on an SM each, while a round gives every one of them rows; K and
  // V, which are moved alike, each by a cluster of its own where the SMs are enough for both
  auto per_warp = [&](int planes) {
    const int n = EM_BUF / (planes * a.row_bytes * EM_WARPS);
    return n < 32 ? n : 32;
  };
  a.planes = 2;
  int cluster = 1;
  while (cluster < 16 && rows * cluster * 2 <= sm_count() && int64_t(cluster) * per_warp(2) * EM_WARPS < a.K) cluster *= 2;
  if (rows * cluster * 2 <= sm_count() && int64_t(cluster) * per_warp(1) * EM_WARPS < a.K) a.planes = 1;
  a.per_warp = per_warp(a.planes);
  const int bytes = a.planes * a.row_bytes;
  Q35_TRY(bytes <= 512    ? launch_evict_move<1>(a, int(rows), cluster, c.stream)
          : bytes <= 1024 ? launch_evict_move<2>(a, int(rows), cluster, c.stream)
                          : launch_evict_move<EM_PIECES>(a, int(rows), cluster, c.stream));
  return 0;
}

}  // namespace q35
