"""The long-context roles where they can go wrong: infinite keys beside every head group, refused windows, tables and counts
at their limits, scratch memory and streams.

Tolerances: those of test_gpu_long_context.py, with the share that a score's error has kept to the weight that is added:
w (2 (D + 4) 2^-23 R + 2^-18 + terms 2^-23) for a weight w that is a sum of `terms` exponentials, and 2^-24 of the result for
every addition to what the row held."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import long_context as olc  # noqa: E402
from test_gpu_long_context import check_out, gpu, gpu_scales, make, poison_behind, q_rows, random_pages  # noqa: E402, F401


def check_added(got, ref, old, reach, D, terms, adds=1):
    """got against ref = old + weights, row by row"""
    got, old = got.double().cpu(), old.double()
    w = (ref - old).abs()
    tol = w * (2 * (D + 4) * 2.0 ** -23 * reach + 2.0 ** -18 + terms * 2.0 ** -23) + adds * 2.0 ** -24 * (old.abs() + w) + 1e-30
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - ref).abs() / tol).max():.3g} of the tolerance"


def windows(T):
    return torch.tensor([0, *torch.tensor(T).cumsum(0).tolist()], dtype=torch.int32)


# ---------------------------------------------------------------------------------------------------- window weights
@pytest.mark.parametrize("G,D", [(3, 64), (5, 128), (6, 256), (7, 64), (48, 128), (43, 64), (8, 128)])
def test_key_mass_beside_keys_masked_by_infinity(G, D):
    """head groups that fill a block of 128 query rows and that do not; tiles that the whole block sees"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, ctxs, T = 64, 2, [700, 400], [60, 45]
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 51)
    q = q_rows(sum(T), HKV * G, D, g)
    q[:, :, 0] = 1.0
    for b in range(2):
        page, row = olc._places(*table, P, b)
        for i in (0, 3, 200, 300, ctxs[b] - 2):
            cache[page[i], 0, row[i]] = 0.0
            cache[page[i], 0, row[i], :, 0] = float("-inf")
    old = torch.zeros((cache.shape[0], P, HKV))
    ref, reach = olc.key_mass(q, cache, windows(T), *table, old)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(windows(T)), *gpu(table), gm)
    assert not ref.isnan().any() and not gm.isnan().any()
    check_added(gm, ref, old, reach, D, max(T) * G)
    assert q35.device_status() == 0


@pytest.mark.parametrize("qo", [[0, 4, 40, 43], [0, 4, 3, 3], [0, 4, 50, 60], [0, 4, -1, 3]])
@pytest.mark.parametrize("accumulate", [False, True])
def test_a_refused_window_leaves_its_sequence_as_it_was(qo, accumulate):
    """a window longer than its sequence, one that ends before it begins, rows behind q: recorded, and the weights of that
    sequence stay; those of the others are right"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, ctxs = 16, 2, 4, 64, [200, 30, 150]
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 52)
    qo = torch.tensor(qo, dtype=torch.int32)
    fine = [b for b in range(3) if 0 <= qo[b] <= qo[b + 1] <= 43 and qo[b + 1] - qo[b] <= ctxs[b]]
    assert 0 in fine and 1 not in fine
    q = q_rows(43, HKV * G, D, g, 2.0)
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    want, base, reach = old.double(), old.clone(), 0.0
    for b in fine:
        one = (table[0][[b, b + 1]] - table[0][b], table[1][int(table[0][b]):int(table[0][b + 1])], table[2][b:b + 1])
        want, r = olc.key_mass(q[int(qo[b]):int(qo[b + 1])], cache, windows([int(qo[b + 1] - qo[b])]), *one, want, accumulate)
        reach = max(reach, r)
        if not accumulate:
            base[olc._places(*one, P, 0)] = 0.0
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(qo), *gpu(table), gm, accumulate=accumulate)
    assert q35.device_status() & 8
    for b in set(range(3)) - set(fine):
        page, row = olc._places(*table, P, b)
        assert torch.equal(gm.cpu()[page, row], old[page, row])
    check_added(gm, want, base, reach, D, 43 * G)


def test_first_pages_behind_the_end():
    """page_key_bounds from a page on that no sequence has, up to the largest number there is: nothing is looked at"""
    import ax_dsl_kernels_b200 as q35
    ctxs = [100, 1, 0, 64, 200]
    cache, table, _, g = make(ctxs, 16, 2, 64, "bf16", 53)
    old = torch.randn((cache.shape[0], 2, 2, 64), generator=g).to(torch.bfloat16)
    for first in ([2 ** 31 - 1] * 5, [7, 2 ** 31 - 1, 0, 2 ** 31 - 3, 2 ** 30], [2 ** 31 - 1, -2 ** 31, 5, 3, 2 ** 31 - 2]):
        first = torch.tensor(first, dtype=torch.int32)
        ref = olc.page_bounds(cache, *table, old, first_page=first)
        got = q35.page_key_bounds(gpu(cache), *gpu(table), gpu(old), first_page=gpu(first))
        assert torch.equal(got.cpu(), ref)
    assert q35.device_status() == 0


# ---------------------------------------------------------------------------------------------------- host threads
@pytest.mark.parametrize("role", ["key_mass", "key_mass int8", "all pages", "evict"])
def test_two_threads_on_one_stream(role):
    """roles of several launches, from two host threads whose calls share a stream and its scratch: every call's numbers are
    those that it gives alone"""
    import threading

    import ax_dsl_kernels_b200 as q35
    fmt = "int8" if "int8" in role else "bf16"
    HKV, G, D, P, ctxs = (16, 1, 64, 64, [57344]) if role == "all pages" else (2, 6, 128, 64, [900, 300, 77])
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 54)
    gc, gt, gs = gpu(cache), gpu(table), gpu_scales(scales)
    T, n = [20, 33, 5], 40
    qo = gpu(windows(T))
    rows = sum(T) if "key_mass" in role else len(ctxs)
    qs = [gpu(q_rows(rows, HKV * G, D, g, 2.0)) for _ in range(2)]
    masses = [torch.rand((cache.shape[0], P, HKV), generator=g).cuda() for _ in range(2)]

    def call(i):
        if role == "all pages":
            return q35.paged_attention_sparse(qs[i], gc, *gt)
        if role == "evict":
            mine, mass = caches[i].pop(), masses[i].clone()
            return torch.cat([q35.evict_keys(mine, mass, *gt, 200, keep_last=9).float().flatten(), mine.float().flatten(), mass.flatten()])
        gm = torch.zeros_like(masses[0])
        return q35.paged_key_mass(qs[i], gc, qo, *gt, gm, **gs)

    caches = [[gc.clone() for _ in range(n + 1)] for _ in range(2)] if role == "evict" else None
    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    got, errors, start = [[], []], [], threading.Barrier(2)

    def work(i):
        try:
            start.wait()
            for _ in range(n):
                got[i].append(call(i))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert not errors, errors
    for i in range(2):
        assert len(got[i]) == n and all(torch.equal(x, want[i]) for x in got[i])
    assert q35.device_status() == 0


# ---------------------------------------------------------------------------------------------------- streams by handle
def handle_case(seed):
    cache, table, _, g = make([700, 900], 64, 2, 128, "bf16", seed)
    return gpu(cache), dict(zip(("indptr", "indices", "last_page_len"), gpu(table))), gpu(q_rows(2, 16, 128, g, 2.0))


@pytest.mark.parametrize("current_captures", [False, True])
def test_capture_of_a_call_on_a_stream_by_its_handle(current_captures):
    """the stream named by the handle captures, the current one does not, or captures the same graph: scratch is the graph's.
    Later calls on that stream need more and write over what is not"""
    import ax_dsl_kernels_b200 as q35
    from ax_dsl_kernels_b200 import _lib
    gc, gt, q = handle_case(55)
    out, gm = torch.empty_like(q), torch.zeros((gc.shape[0], 64, 2), device="cuda")
    want, wm = torch.empty_like(q), torch.zeros_like(gm)
    q35.run("attn.sparse_decode", q=q, paged_kv_cache=gc, **gt, out=want, key_mass=wm)
    origin, side, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=origin):
        if current_captures:  # fork
            side.wait_stream(origin)
            target, current = side, origin
        else:
            target, current = origin, torch.cuda.Stream()
        with torch.cuda.stream(current):
            q35.run("attn.sparse_decode", target.cuda_stream, q=q, paged_kv_cache=gc, **gt, out=out, key_mass=gm)
        if current_captures:
            origin.wait_stream(side)
    assert (0, target.cuda_stream) not in _lib._ws_cache
    with torch.cuda.stream(target):
        for n in (1, 40):
            ids = torch.randint(0, 32, (64 * n, 4), dtype=torch.int32, device="cuda")
            q35.moe_permute(ids, torch.rand((64 * n, 4), device="cuda"), 32, 16)
        junk = [torch.full((1 << 18,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(gm, wm) and len(junk) == 8


def test_scratch_that_grows_on_a_stream_by_its_handle():
    """calls of growing size on another stream, with nothing waited for, while the current stream allocates and writes: the
    buffers that were outgrown stay the other stream's"""
    import ax_dsl_kernels_b200 as q35
    side, P, HKV, D = torch.cuda.Stream(), 64, 2, 128
    cases = []
    for i, ctx in enumerate((2000, 20000, 40000, 80000)):
        cache, table, _, g = make([ctx], P, HKV, D, "bf16", 56 + i)
        t = dict(zip(("indptr", "indices", "last_page_len"), gpu(table)), q=gpu(q_rows(1, 16, D, g, 2.0)), paged_kv_cache=gpu(cache))
        outs = [[torch.empty_like(t["q"]), torch.zeros((cache.shape[0], P, HKV), device="cuda")] for _ in range(2)]
        q35.run("attn.sparse_decode", **t, out=outs[0][0], key_mass=outs[0][1])
        cases.append((t, outs))
    torch.cuda.synchronize()
    for t, outs in cases:
        q35.run("attn.sparse_decode", side.cuda_stream, **t, out=outs[1][0], key_mass=outs[1][1])
        for n in (1 << 20, 1 << 21, 1 << 23):
            torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for _, (a, b) in cases:
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert q35.device_status() == 0


# ---------------------------------------------------------------------------------------------------- the documented loop
@pytest.mark.parametrize("fmt", ["bf16", "e4m3c", "int8"])
def test_decode_loop_as_documented(fmt):
    """prompt -> weights -> eviction -> steps that attend to the current token from its own rows, which stores its weight:
    what places in key_mass held before plays no part, neither behind an eviction nor in pages of another sequence.  Every
    step, and a second eviction by the weights that came together, against the oracle on the same state"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, K, W = 16, 2, 4, 64, 90, 8
    ctxs = [260, 85, 171]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 58, extra=9)
    pool = torch.arange(cache.shape[0], dtype=torch.int32)[~torch.isin(torch.arange(cache.shape[0]), table[1].long())].tolist()
    gc, gs = gpu(cache), gpu_scales(scales)
    row_scale = gs.get("paged_kv_scale")

    def now():  # what the oracle reads: the GPU's own state
        return gc.cpu(), {} if row_scale is None else {"row_scale": row_scale.cpu()}

    gm = torch.rand((cache.shape[0], P, HKV), generator=g).mul(1e4).cuda()  # of whoever had the pages before
    q = q_rows(3 * W, HKV * G, D, g, 2.0)
    q35.paged_key_mass(gpu(q), gc, gpu(windows([W] * 3)), *gpu(table), gm, **gs)
    mass = gm.cpu()
    kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=2, keep_last=W, **gs)
    rk, rc, rm, rs = olc.evict(cache, mass, *table, K, 2, W, scales.get("row_scale"))
    assert torch.equal(kept.cpu(), rk) and torch.equal(gc.cpu().view(torch.uint8), rc.view(torch.uint8)) and torch.equal(gm.cpu(), rm)
    ctxs = [min(c, K) for c in ctxs]
    pages_of = [table[1][int(table[0][b]):int(table[0][b + 1])].tolist()[:-(-ctxs[b] // P)] for b in range(3)]
    for b in range(3):
        pool += [p for p in table[1][int(table[0][b]):int(table[0][b + 1])].tolist() if p not in pages_of[b]]

    def listed():
        return (windows([len(p) for p in pages_of]), torch.tensor(sum(pages_of, []), dtype=torch.int32),
                torch.tensor([c - (len(p) - 1) * P for c, p in zip(ctxs, pages_of)], dtype=torch.int32))

    bounds = q35.page_key_bounds(gc, *gpu(listed()), paged_kv_scale=row_scale)
    for step in range(20):
        t, gt = listed(), gpu(listed())
        for b in range(3):
            if ctxs[b] == len(pages_of[b]) * P:
                pages_of[b].append(pool.pop(0))
        loc = torch.tensor([[pages_of[b][c // P], c % P] for b, c in enumerate(ctxs)], dtype=torch.int32)
        kn, vn, qs = q_rows(3, HKV, D, g), q_rows(3, HKV, D, g), q_rows(3, HKV * G, D, g, 2.0)
        c, s = now()
        sel = q35.select_pages(gpu(qs), bounds, *gt, 3, keep_first=1, keep_last=1)
        rb = olc.page_bounds(c, *t, torch.zeros(bounds.shape, dtype=torch.bfloat16), row_scale=s.get("row_scale"))
        assert torch.equal(sel.cpu(), olc.select_pages(qs, rb, *t, 3, 1, 1))
        before = gm.cpu()
        out = q35.paged_attention_sparse(gpu(qs), gc, *gt, sel, key_mass=gm, k_new=gpu(kn), v_new=gpu(vn), cache_location=gpu(loc), **gs)
        ref, rmass, size, reach = olc.sparse_decode(qs, c, *t, sel.cpu(), before, k_new=kn, v_new=vn, cache_location=loc, **s)
        check_out(out, ref, size, reach, D, fmt)
        before[loc[:, 0].long(), loc[:, 1].long()] = 0.0  # stored there
        check_added(gm, rmass, before, float(reach.max()), D, G)
        q35.kv_write(gc, gpu(loc), gpu(kn), gpu(vn), paged_kv_scale=row_scale)
        ctxs = [n + 1 for n in ctxs]
        q35.page_key_bounds(gc, *gpu(listed()), bounds, first_page=gpu(torch.tensor([len(p) - 1 for p in pages_of], dtype=torch.int32)),
                            paged_kv_scale=row_scale)
    (c, s), t, mass = now(), listed(), gm.cpu()
    kept = q35.evict_keys(gc, gm, *gpu(t), K - 20, keep_first=2, keep_last=4, **gs)
    assert torch.equal(kept.cpu(), olc.evict(c, mass, *t, K - 20, 2, 4, s.get("row_scale"))[0])
    page, row = olc._places(*t, P, 0)
    assert mass[page, row].max() < 40 * G * W  # no place kept what it held in the beginning
    assert q35.device_status() == 0
