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


# ---------------------------------------------------------------------------------------------------- added weights, row by row
@pytest.mark.parametrize("held", [0.0, 1.0])
@pytest.mark.parametrize("fmt,D,HKV,G,n", [("bf16", 256, 4, 2, 57344), ("int8", 128, 8, 3, 86016), ("e4m3c", 64, 16, 1, 57344)])
def test_weights_of_many_rows_one_by_one(fmt, D, HKV, G, n, held):
    """equal shares of all pages: a row's weight is about 1 / n, and every one of them is there, whatever the row held"""
    import ax_dsl_kernels_b200 as q35
    ctxs, P = [0, 1, n // 2, 33, n // 2 + 77], 64
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 59, extra=8)
    q, kn, vn = q_rows(5, HKV * G, D, g, 2.0), q_rows(5, HKV, D, g), q_rows(5, HKV, D, g)
    spare = torch.arange(cache.shape[0], dtype=torch.int32)[~torch.isin(torch.arange(cache.shape[0]), table[1].long())]
    loc = torch.stack([spare[:5], torch.arange(5, dtype=torch.int32)], 1).contiguous()
    old = torch.rand((cache.shape[0], P, HKV), generator=g) * held
    _, ref, _, reach = olc.sparse_decode(q, cache, *table, None, old, **scales, k_new=kn, v_new=vn, cache_location=loc)
    gm = gpu(old)
    q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), key_mass=gm, k_new=gpu(kn), v_new=gpu(vn), cache_location=gpu(loc),
                               **gpu_scales(scales))
    old[loc[:, 0].long(), loc[:, 1].long()] = 0.0
    check_added(gm, ref, old, float(reach.max()), D, G)
    assert q35.device_status() == 0


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("held", [0.0, 1.0])
def test_weights_added_to_shared_pages_one_by_one(fmt, held):
    """six sequences that share their first pages, from windows and from single queries"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, n = 16, 2, 6, 128, 6
    ctxs = [400 + 37 * i for i in range(n)]
    cache, (indptr, indices, last), scales, g = make(ctxs, P, HKV, D, fmt, 60)
    for b in range(1, n):
        indices[int(indptr[b]):int(indptr[b]) + 20] = indices[:20]
    table, T = (indptr, indices, last), [1, 30, 0, 60, 25, 130]
    q, old = q_rows(sum(T), HKV * G, D, g, 2.0), torch.rand((cache.shape[0], P, HKV), generator=g) * held
    ref, reach = olc.key_mass(q, cache, windows(T), *table, old, accumulate=True, **scales)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(windows(T)), *gpu(table), gm, accumulate=True, **gpu_scales(scales))
    check_added(gm, ref, old, reach, D, sum(T) * G, adds=n)
    q = q_rows(n, HKV * G, D, g, 2.0)
    _, ref, _, reach = olc.sparse_decode(q, cache, *table, None, old, **scales)
    gm = gpu(old)
    q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), key_mass=gm, **gpu_scales(scales))
    check_added(gm, ref, old, float(reach.max()), D, n * G, adds=n)


# ---------------------------------------------------------------------------------------------------- sizes
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("S", [32, 33, 64, 70])
def test_long_lists_of_chosen_pages(fmt, S):
    """lists that end inside a warp's 32 entries, at their border, and not at all"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D = 16, 2, 5, 64
    ctxs = [1200, 16 * 64, 16 * 32, 16 * 33 - 1, 16 * 31, 900, 5]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 61)
    cache, _ = poison_behind(cache, table, P)
    q, old = q_rows(len(ctxs), HKV * G, D, g, 2.0), torch.rand((cache.shape[0], P, HKV), generator=g)
    pages = random_pages(ctxs, P, HKV, S, g)
    for b, h, n in ((0, 0, 32), (0, 1, 31), (1, 0, 33), (5, 1, 0)):  # and lists of chosen lengths
        pages[b, h, min(n, S):] = -1
    ref, mass, size, reach = olc.sparse_decode(q, cache, *table, pages, old, **scales)
    gm = gpu(old)
    out = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), gpu(pages), key_mass=gm, **gpu_scales(scales))
    check_out(out, ref, size, reach, D, fmt)
    check_added(gm, mass, old, float(reach.max()), D, G)
    assert q35.device_status() == 0


@pytest.mark.parametrize("fmt,D", [("bf16", 256), ("e4m3", 128), ("int8", 64)])
def test_one_long_sequence(fmt, D):
    """the most CTAs to a row, the most ranges of keys to a window; chosen pages as many as there are"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, ctx, T = 64, 2, 4, 20011, 5
    cache, table, scales, g = make([ctx], P, HKV, D, fmt, 62)
    cache, _ = poison_behind(cache, table, P)
    q, old = q_rows(T, HKV * G, D, g, 2.0), torch.rand((cache.shape[0], P, HKV), generator=g)
    every = torch.arange(-(-ctx // P), dtype=torch.int32).expand(1, HKV, -1).contiguous()
    ref, mass, size, reach = olc.sparse_decode(q[:1], cache, *table, None, old, **scales)
    for pages in (None, gpu(every)):
        gm = gpu(old)
        out = q35.paged_attention_sparse(gpu(q[:1]), gpu(cache), *gpu(table), pages, key_mass=gm, **gpu_scales(scales))
        check_out(out, ref, size, reach, D, fmt)
        check_added(gm, mass, old, float(reach.max()), D, G)
    ref, reach = olc.key_mass(q, cache, windows([T]), *table, old, **scales)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(windows([T])), *gpu(table), gm, **gpu_scales(scales))
    base = old.clone()
    base[olc._places(*table, P, 0)] = 0.0
    check_added(gm, ref, base, reach, D, T * G)
    assert q35.device_status() == 0


@pytest.mark.parametrize("G", [43, 64, 65, 100, 128])
def test_key_mass_of_large_head_groups(G):
    import ax_dsl_kernels_b200 as q35
    P, HKV, D, ctxs, T = 32, 2, 64, [300, 130, 9], [12, 0, 9]
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 63)
    q, old = q_rows(sum(T), HKV * G, D, g, 2.0), torch.rand((cache.shape[0], P, HKV), generator=g)
    ref, reach = olc.key_mass(q, cache, windows(T), *table, old, accumulate=True)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(windows(T)), *gpu(table), gm, accumulate=True)
    check_added(gm, ref, old, reach, D, max(T) * G)
    assert q35.device_status() == 0


def test_more_sequences_than_a_warp_has_lanes():
    """70 sequences: the windows' and the equal shares' search goes around more than twice"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, B = 16, 2, 3, 64, 70
    g = torch.Generator().manual_seed(64)
    ctxs = torch.randint(0, 400, (B,), generator=g).tolist()
    T = [min(c, t) for c, t in zip(ctxs, torch.randint(0, 90, (B,), generator=g).tolist())]
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 65)
    q, old = q_rows(sum(T), HKV * G, D, g, 2.0), torch.rand((cache.shape[0], P, HKV), generator=g)
    ref, reach = olc.key_mass(q, cache, windows(T), *table, old, accumulate=True)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(windows(T)), *gpu(table), gm, accumulate=True)
    check_added(gm, ref, old, reach, D, max(T) * G)
    # equal shares: against every sequence by itself
    HKV, B = 16, 40
    ctxs = [0 if b % 9 == 4 else 9000 + 53 * b for b in range(B)]
    n = [-(-c // 64) for c in ctxs]
    cache = torch.randn((sum(n), 2, 64, HKV, D), device="cuda").to(torch.bfloat16)
    q = gpu(q_rows(B, HKV, D, g, 2.0))
    indptr, indices = gpu(windows(n)), torch.randperm(sum(n), device="cuda").to(torch.int32)
    last = gpu(torch.tensor([c - (m - 1) * 64 if m else 0 for c, m in zip(ctxs, n)], dtype=torch.int32))
    gm = torch.zeros((sum(n), 64, HKV), device="cuda")
    out = q35.paged_attention_sparse(q, cache, indptr, indices, last, key_mass=gm)
    one, gn = torch.empty_like(out), torch.zeros_like(gm)
    for b in range(B):
        lo, hi = sum(n[:b]), sum(n[:b + 1])
        q35.paged_attention_sparse(q[b:b + 1], cache, indptr[b:b + 2] - lo, indices[lo:hi].clone(), last[b:b + 1], out=one[b:b + 1],
                                   key_mass=gn)
    # two evaluations of scores with R <= 20 here (|q| |k| scale is 10 on average): weights differ by twice 2 (D + 4) 2^-23 R
    # < 2^-10 of themselves at most, outputs by that of sum p |v| < 1 and one step of bf16
    assert ((out.float() - one.float()).abs() <= one.float().abs() * 2.0 ** -7 + 2.0 ** -10).all()
    assert (out[4] == 0).all() and ((gm - gn).abs() <= gn * 2.0 ** -10).all()
    assert torch.allclose(gm.double().sum(), torch.tensor(float(HKV * (B - 4)), dtype=torch.float64, device="cuda"), rtol=2.0 ** -12)
    assert q35.device_status() == 0


@pytest.mark.parametrize("scale", [-0.07, 0.0, 1.5])
def test_other_scales(scale):
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, ctxs, T = 64, 2, 6, 64, [500, 200], [70, 3]
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 66)
    q, old = q_rows(sum(T), HKV * G, D, g), torch.rand((cache.shape[0], P, HKV), generator=g)
    for s in (scale, torch.tensor([scale], device="cuda")):
        ref, _ = olc.key_mass(q, cache, windows(T), *table, old, accumulate=True, sm_scale=scale)
        _, reach = olc.key_mass(q, cache, windows(T), *table, old, sm_scale=abs(scale))
        gm = gpu(old)
        q35.paged_key_mass(gpu(q), gpu(cache), gpu(windows(T)), *gpu(table), gm, accumulate=True, sm_scale=s)
        check_added(gm, ref, old, reach, D, max(T) * G)
        ref, mass, size, _ = olc.sparse_decode(q[:2], cache, *table, None, old, sm_scale=scale)
        _, _, _, reach = olc.sparse_decode(q[:2], cache, *table, sm_scale=abs(scale))
        gm = gpu(old)
        out = q35.paged_attention_sparse(gpu(q[:2]), gpu(cache), *gpu(table), key_mass=gm, sm_scale=s)
        check_out(out, ref, size, reach, D)
        check_added(gm, mass, old, float(reach.max()), D, G)


@pytest.mark.parametrize("fmt,D", [("bf16", 32), ("bf16", 96), ("bf16", 160), ("int8", 192), ("int8", 320), ("bf16", 512), ("bf16", 1024)])
@pytest.mark.parametrize("B,K", [(1, 600), (5, 100), (90, 130)])
def test_evict_rows_of_other_widths(fmt, D, B, K):
    """rows of 64 to 2048 bytes, among them those whose pieces do not divide a warp: K and V by a cluster each, by one, by
    one CTA"""
    import ax_dsl_kernels_b200 as q35
    P, HKV = 16, 2
    ctxs = [700, 0, 130, 101, 1][:B] if B <= 5 else [(37 * i) % 200 for i in range(B)]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 67)
    mass = torch.randn((cache.shape[0], P, HKV), generator=g).mul(2).exp()
    ref, rcache, rmass, rrs = olc.evict(cache, mass, *table, K, 2, 9, scales.get("row_scale"))
    gc, gm, gs = gpu(cache), gpu(mass), gpu_scales(scales)
    kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=2, keep_last=9, **gs)
    assert torch.equal(kept.cpu(), ref)
    assert torch.equal(gc.cpu().view(torch.uint8), rcache.view(torch.uint8)) and torch.equal(gm.cpu(), rmass)
    assert rrs is None or torch.equal(gs["paged_kv_scale"].cpu(), rrs)
    assert q35.device_status() == 0


def test_select_pages_of_more_than_fit_on_chip():
    """sequences of more than 16384 pages beside shorter ones; pages that differ, and pages that are all the same"""
    import ax_dsl_kernels_b200 as q35
    from test_gpu_long_context import select_case
    q, bounds, table = select_case([20000, 300, 16384, 17003], 2, 64, 2, 68)
    same = bounds.clone()
    same[table[1].long()] = bounds[table[1][0].long()]
    for b in (bounds, same):
        for S, first, last in ((100, 1, 2), (16500, 0, 1)):
            ref = olc.select_pages(q, b, *table, S, first, last)
            got = q35.select_pages(gpu(q), gpu(b), *gpu(table), S, keep_first=first, keep_last=last)
            assert torch.equal(got.cpu(), ref)
    assert q35.device_status() == 0


def test_nothing_cached_and_no_queries():
    """tables without an entry, sequences without a row, a window of no tokens, no sequence at all"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D = 16, 2, 4, 64
    cache, _, _, g = make([], P, HKV, D, "bf16", 69)
    gc, gm = gpu(cache), torch.full((cache.shape[0], P, HKV), 3.0, device="cuda")
    for B in (0, 2):
        t = gpu((torch.zeros(B + 1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)))
        q = gpu(q_rows(B, HKV * G, D, g))
        bounds = q35.page_key_bounds(gc, *t)
        assert (bounds == 0).all()
        assert (q35.select_pages(q, bounds, *t, 3, keep_first=1) == -1).all()
        for pages in (None, torch.full((B, HKV, 3), -1, dtype=torch.int32, device="cuda")):
            assert (q35.paged_attention_sparse(q, gc, *t, pages, key_mass=gm) == 0).all()
        q35.paged_key_mass(gpu(q_rows(0, HKV * G, D, g)), gc, torch.zeros(B + 1, dtype=torch.int32, device="cuda"), *t, gm)
        assert (q35.evict_keys(gc, gm, *t, 5, keep_last=2) == -1).all()
        assert (gm == 3.0).all() and torch.equal(gc.cpu(), cache)
    cache, table, _, g = make([40, 0, 20], P, HKV, D, "bf16", 70)  # rows, but no window: nobody gave them a weight
    gm = torch.full((cache.shape[0], P, HKV), 3.0, device="cuda")
    q35.paged_key_mass(gpu(q_rows(0, HKV * G, D, g)), gpu(cache), torch.zeros(4, dtype=torch.int32, device="cuda"), *gpu(table), gm)
    ref, _ = olc.key_mass(q_rows(0, HKV * G, D, g), cache, torch.zeros(4, dtype=torch.int32), *table, torch.full(gm.shape, 3.0))
    assert torch.equal(gm.cpu().double(), ref) and (ref == 0).sum() == 60 * HKV
    assert q35.device_status() == 0


@pytest.mark.parametrize("fmt", ["bf16", "e4m3c", "int8"])
def test_pages_far_into_a_large_cache(fmt):
    """the same rows in the last pages of a cache whose elements and bytes pass 2^31 and 2^32: the same results"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, total = 64, 2, 8, 256, 40000 if fmt == "bf16" else 70000
    ctxs, T = [900, 300, 65], [40, 3, 0]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 71)
    n = cache.shape[0]
    far = torch.arange(total - n, total, device="cuda")
    big = torch.empty((total, 2, P, HKV, D), dtype=torch.uint8 if fmt != "bf16" else torch.bfloat16, device="cuda")
    assert big.numel() > 2 ** 31 and big.numel() * big.element_size() > 2 ** 32
    big[far] = gpu(cache) if fmt == "bf16" else gpu(cache).view(torch.uint8)
    big = big if fmt == "bf16" else big.view(cache.dtype)
    mass = torch.rand((n, P, HKV), generator=g)
    qs, qw = gpu(q_rows(3, HKV * G, D, g, 2.0)), gpu(q_rows(sum(T), HKV * G, D, g, 2.0))
    results = []
    for c, shift in ((gpu(cache), 0), (big, total - n)):
        pages = c.shape[0]
        t = (gpu(table[0]), gpu(table[1]) + shift, gpu(table[2]))
        gm = torch.zeros((pages, P, HKV), device="cuda")
        gm[shift:shift + n] = gpu(mass)
        s = {}
        if "row_scale" in scales:
            s["paged_kv_scale"] = torch.zeros((pages, 2, P, HKV), dtype=torch.bfloat16, device="cuda")
            s["paged_kv_scale"][shift:shift + n] = gpu(scales["row_scale"])
        bounds = q35.page_key_bounds(c, *t, **s)
        sel = q35.select_pages(qs, bounds, *t, 4)
        out = q35.paged_attention_sparse(qs, c, *t, sel, key_mass=gm, **s)
        q35.paged_key_mass(qw, c, gpu(windows(T)), *t, gm, accumulate=True, **s)
        kept = q35.evict_keys(c, gm, *t, 200, keep_last=5, **s)
        results.append([x[shift:shift + n] if x.shape[0] == pages else x for x in (
            bounds, sel, out, gm, kept, c.view(torch.uint8) if fmt != "bf16" else c, *s.values())])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    assert q35.device_status() == 0


def test_last_pages_of_negative_length():
    """every role records one and takes the sequence for empty"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D = 16, 2, 4, 64
    cache, table, _, g = make([100, 60], P, HKV, D, "bf16", 72)
    q, mass = gpu(q_rows(2, HKV * G, D, g)), torch.rand((cache.shape[0], P, HKV), generator=g)
    fine = gpu(table)
    bounds = q35.page_key_bounds(gpu(cache), *fine)
    want = q35.select_pages(q, bounds, *fine, 3), q35.paged_attention_sparse(q, gpu(cache), *fine)
    t = (fine[0], fine[1], torch.tensor([-1, int(table[2][1])], dtype=torch.int32, device="cuda"))
    gc, gm = gpu(cache), gpu(mass)
    assert q35.device_status() == 0
    got = q35.select_pages(q, bounds, *t, 3)
    assert q35.device_status() & 1 and (got[0] == -1).all() and torch.equal(got[1], want[0][1])
    got = q35.paged_attention_sparse(q, gc, *t)
    assert q35.device_status() & 1 and (got[0] == 0).all() and torch.equal(got[1], want[1][1])
    q35.page_key_bounds(gc, *t, bounds.clone())
    assert q35.device_status() & 1
    q35.paged_key_mass(q, gc, gpu(windows([0, 2])), *t, gm)
    assert q35.device_status() & 1
    page, row = olc._places(*table, P, 0)
    assert torch.equal(gm.cpu()[page, row], mass[page, row])
    assert (q35.evict_keys(gc, gm, *t, 10)[0] == -1).all() and q35.device_status() & 1
    assert torch.equal(gc.cpu()[page, :, row], cache[page, :, row]) and torch.equal(gm.cpu()[page, row], mass[page, row])
