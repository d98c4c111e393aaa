"""The long-context operators on the GPU against their 64-bit oracle: bounds of pages, choice of pages, attention over
chosen pages, accumulated weights, eviction -- and a decode loop that uses them together.

Tolerances.  Whole numbers, bounds and moved rows are exact.  An attention output is rounded to bf16 once (half a step,
2^-8 of the value); before that, a weight is exp of an fp32 score.  A score is a sum of D products; any order of fp32
additions is off by at most D 2^-23 sum |q_d k_d| scale =: D 2^-23 R (2^-23: a tensor-core addition may truncate), its
scaling by 4 roundings more, so a weight, a quotient of two such exponentials, by 2 (D + 4) 2^-23 R + 2^-18 of itself
(2^-18: exp2, the running sums, the two 16-bit terms a weight is carried in, 2^-16 times 1 / 4 headroom for their
truncation).  Outputs are sums of weights times v: off by that fraction of sum p |v|.  With an E4M3 cache a weight meets
its v as one f16 number: 2^-11 of the weight more in the output (not in key_mass, which takes the fp32 weight)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import codecs  # noqa: E402
from oracle import long_context as olc  # noqa: E402


def make(ctxs, P, HKV, D, fmt, seed, extra=3):
    """cache, table (indptr, indices, last_page_len), kwargs of the scales; CPU tensors"""
    g = torch.Generator().manual_seed(seed)
    n_pages = [-(-c // P) for c in ctxs]
    total = sum(n_pages) + extra
    kv = torch.randn((total, 2, P, HKV, D), generator=g).to(torch.bfloat16)
    scales = {}
    if fmt == "bf16":
        cache = kv
    elif fmt == "e4m3":
        ks = (kv.float().abs().amax((0, 2, 4)) / 448.0).contiguous()
        cache = torch.stack([codecs.kv_quant_fp8(kv[:, i], ks[i]) for i in range(2)], 1).contiguous()
        scales["kv_scale"] = ks
    elif fmt == "e4m3c":
        cache = codecs.kv_quant_fp8(kv)
    else:
        rs = (kv.abs().amax(-1).float() / 127).to(torch.bfloat16).contiguous()
        cache = (kv.float() / rs.float().unsqueeze(-1)).round().clamp(-127, 127).to(torch.int8)
        scales["row_scale"] = rs
    perm = torch.randperm(total, generator=g).to(torch.int32)
    indptr = torch.tensor([0, *torch.tensor(n_pages).cumsum(0).tolist()], dtype=torch.int32)
    last = torch.tensor([c - (n - 1) * P if n else 0 for c, n in zip(ctxs, n_pages)], dtype=torch.int32)
    return cache, (indptr, perm[:sum(n_pages)].contiguous(), last), scales, g


def gpu(x):
    return x.cuda() if isinstance(x, torch.Tensor) else tuple(t.cuda() for t in x)


def gpu_scales(s):
    return {{"row_scale": "paged_kv_scale"}.get(k, k): v.cuda() for k, v in s.items()}


def poison_behind(cache, table, P):
    """NaN (0x7f / 0xff bytes) in every row behind a sequence's end and in every page that is not listed"""
    indptr, indices, last = table
    used = torch.zeros(cache.shape[0], P, dtype=torch.bool)
    for b in range(len(indptr) - 1):
        pg, row = olc._places(indptr, indices, last, P, b)
        used[pg, row] = True
    raw = cache.view(torch.uint8)
    bad = torch.full_like(raw, 0x7F if cache.dtype != torch.bfloat16 else 0xFF)
    cache = torch.where(used[:, None, :, None, None], raw, bad).view(cache.dtype)
    return cache, used


def q_rows(n, HQ, D, g, gain=1.0):
    return (torch.randn((n, HQ, D), generator=g) * gain).to(torch.bfloat16)


FMT = ["bf16", "e4m3", "e4m3c", "int8"]


# ---------------------------------------------------------------------------------------------------- bounds
@pytest.mark.parametrize("fmt", FMT[:1] + FMT[2:])
@pytest.mark.parametrize("P,HKV,D,ctxs", [(64, 2, 256, [1, 64, 65, 200, 0, 63]), (16, 5, 64, [33, 0, 16]), (7, 1, 128, [20, 7]),
                                          (128, 9, 256, [129, 300]), (1, 4, 64, [5, 1])])
def test_page_bounds(fmt, P, HKV, D, ctxs):
    import ax_dsl_kernels_b200 as q35
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 1)
    cache, _ = poison_behind(cache, table, P)
    old = torch.randn((cache.shape[0], 2, HKV, D), generator=g).to(torch.bfloat16)
    ref = olc.page_bounds(cache, *table, old, row_scale=scales.get("row_scale"))
    got = q35.page_key_bounds(gpu(cache), *gpu(table), gpu(old), paged_kv_scale=gpu_scales(scales).get("paged_kv_scale"))
    assert torch.equal(got.cpu(), ref)
    # from a page on: the others stay
    first = torch.tensor([max(0, -(-c // P) - 1 - b % 2) for b, c in enumerate(ctxs)], dtype=torch.int32)
    ref = olc.page_bounds(cache, *table, old, first_page=first, row_scale=scales.get("row_scale"))
    got = q35.page_key_bounds(gpu(cache), *gpu(table), gpu(old), first_page=gpu(first),
                              paged_kv_scale=gpu_scales(scales).get("paged_kv_scale"))
    assert torch.equal(got.cpu(), ref)
    assert q35.device_status() == 0


def test_page_bounds_special_values():
    import ax_dsl_kernels_b200 as q35
    cache, table, _, g = make([40, 30], 16, 2, 64, "bf16", 2)
    pg, row = olc._places(*table, 16, 0)
    cache[pg[3], 0, row[3], 0, 5] = float("nan")
    cache[pg[20], 0, row[20], 1, 7] = float("inf")
    cache[pg[35], 0, row[35], 1, 9] = float("-inf")
    ref = olc.page_bounds(cache, *table, torch.zeros((cache.shape[0], 2, 2, 64), dtype=torch.bfloat16))
    got = q35.page_key_bounds(gpu(cache), *gpu(table)).cpu()
    assert torch.equal(got.isnan(), ref.isnan()) and ref.isnan().sum() == 2
    assert torch.equal(got.nan_to_num(3.0), ref.nan_to_num(3.0))


# ---------------------------------------------------------------------------------------------------- selection
def select_case(n_pages, HKV, D, G, seed):
    g = torch.Generator().manual_seed(seed)
    total = sum(n_pages) + 2
    mid = torch.randn((total, HKV, D), generator=g)
    wide = torch.randn((total, HKV, D), generator=g).abs()
    bounds = torch.stack([mid - wide, mid + wide], 1).to(torch.bfloat16)
    perm = torch.randperm(total, generator=g).to(torch.int32)
    indptr = torch.tensor([0, *torch.tensor(n_pages).cumsum(0).tolist()], dtype=torch.int32)
    table = (indptr, perm[:sum(n_pages)].contiguous(), torch.tensor([3 if n else 0 for n in n_pages], dtype=torch.int32))
    return q_rows(len(n_pages), HKV * G, D, g), bounds, table


@pytest.mark.parametrize("HKV,G,D", [(2, 8, 256), (4, 6, 256), (1, 1, 64), (3, 16, 128), (2, 11, 64)])
@pytest.mark.parametrize("S,first,last", [(1, 0, 0), (5, 1, 2), (16, 0, 1), (40, 30, 30), (300, 2, 2)])
def test_select_pages(HKV, G, D, S, first, last):
    import ax_dsl_kernels_b200 as q35
    q, bounds, table = select_case([1, 0, 5, 16, 17, 130, 299, 300, 301], HKV, D, G, 3)
    ref = olc.select_pages(q, bounds, *table, S, first, last)
    got = q35.select_pages(gpu(q), gpu(bounds), *gpu(table), S, keep_first=first, keep_last=last)
    assert torch.equal(got.cpu(), ref)
    assert q35.device_status() == 0


@pytest.mark.parametrize("n,S", [(50, 7), (1100, 64), (2500, 200)])
def test_select_pages_ties_and_near_ties(n, S):
    """pages that are all the same; pages that differ in the last bit of one channel; blocks of equal pages"""
    import ax_dsl_kernels_b200 as q35
    q, bounds, table = select_case([n], 2, 128, 4, 4)
    page = table[1].long()
    same = bounds.clone()
    same[page] = bounds[page[0]]
    for case in ("same", "last bit", "blocks"):
        b = same.clone()
        if case == "last bit":
            for j in range(0, n, 3):  # one step of bf16 up or down in one channel of the maxima
                ch = j % 128
                bits = b[page[j], 1, :, ch].view(torch.int16)
                b[page[j], 1, :, ch] = (bits + (1 if j % 2 else -1)).view(torch.bfloat16)
        if case == "blocks":
            b[page] = bounds[page[torch.arange(n) // 9]]
        ref = olc.select_pages(q, b, *table, S, 1, 1)
        got = q35.select_pages(gpu(q), gpu(b), *gpu(table), S, keep_first=1, keep_last=1)
        assert torch.equal(got.cpu(), ref), case


def test_select_pages_special_values():
    import ax_dsl_kernels_b200 as q35
    q, bounds, table = select_case([40, 40, 40], 2, 64, 4, 5)
    page = table[1].long()
    bounds[page[3], 0, 0, 5] = float("nan")      # a NaN ranks last
    bounds[page[44], :, :, :] = float("nan")
    bounds[page[50], 1, 1, 2] = float("inf")
    bounds[page[51], :, 0, 1] = 3.0e38           # an fp32 sum overflows, the true one does not
    bounds[page[52], :, 0, 1] = 2.9e38
    bounds[page[53], 0, 0, :] = float("-inf")
    q[1, :, 1] = 100.0
    bounds[page[80:], :, :, :] = 0.0             # nothing but equal zeros, of either sign
    bounds[page[80::2], :, :, :] = -0.0
    for S in (1, 2, 8, 39):
        ref = olc.select_pages(q, bounds, *table, S)
        got = q35.select_pages(gpu(q), gpu(bounds), *gpu(table), S, keep_last=0)
        assert torch.equal(got.cpu(), ref)
    # keys masked by -inf in one channel: the page's other keys still count, by the sign of the query there
    q, bounds, table = select_case([60, 60], 1, 128, 3, 6)
    q[:, :, 7] = torch.tensor([1.0, -1.0]).reshape(2, 1).expand(2, 3).to(torch.bfloat16)
    page = table[1].long()
    bounds[page[5:110:4], 0, 0, 7] = float("-inf")
    for S in (3, 20):
        assert torch.equal(q35.select_pages(gpu(q), gpu(bounds), *gpu(table), S).cpu(), olc.select_pages(q, bounds, *table, S, 0, 1))
    # a last page without rows is no page
    table[2][0] = 0
    assert torch.equal(q35.select_pages(gpu(q), gpu(bounds), *gpu(table), 8).cpu(), olc.select_pages(q, bounds, *table, 8, 0, 1))


# ---------------------------------------------------------------------------------------------------- attention
def check_out(got, ref, size, reach, D, fmt="bf16"):
    got = got.double().cpu()
    carried = 2.0 ** -11 if fmt.startswith("e4m3") else 0.0
    tol = ref.abs() * 2.0 ** -8 + size * (2 * (D + 4) * 2.0 ** -23 * reach + 2.0 ** -18 + carried)
    assert torch.equal(got.isnan(), ref.isnan())
    bad = ((got - ref).abs() > tol) & ~ref.isnan()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - ref).abs() / tol).nan_to_num(0).max():.3g} of the tolerance"


def check_mass(got, ref, old, reach, D, n_add=1):
    """weights to 2 (D + 4) 2^-23 R + 2^-18 of themselves, plus fp32 additions to what was there and to each other"""
    got = got.double().cpu()
    w = (ref - old.double()).abs() + ref.abs()
    tol = w * (2 * (D + 4) * 2.0 ** -23 * reach + 2.0 ** -18 + n_add * 2.0 ** -23) + 1e-30
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {((got - ref).abs() / tol).max():.3g} of the tolerance"


def random_pages(ctxs, P, HKV, S, g):
    out = torch.full((len(ctxs), HKV, S), -1, dtype=torch.int32)
    for b, c in enumerate(ctxs):
        n = -(-c // P)
        for h in range(HKV):
            k = min(S, n) if h % 2 == 0 else int(torch.randint(0, min(S, n) + 1, (1,), generator=g))
            out[b, h, :k] = torch.randperm(n, generator=g)[:k].sort().values.to(torch.int32)
    return out


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("D,HKV,G,P", [(256, 2, 8, 64), (128, 4, 6, 16), (64, 1, 1, 48), (64, 3, 5, 128)])
@pytest.mark.parametrize("S", [0, 1, 5])
def test_sparse_decode(fmt, D, HKV, G, P, S):
    import ax_dsl_kernels_b200 as q35
    ctxs = [1, 0, 16, 15, P + 1, 5 * P, 700, 1501]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 7)
    cache, _ = poison_behind(cache, table, P)
    q = q_rows(len(ctxs), HKV * G, D, g, 2.0)
    pages = random_pages(ctxs, P, HKV, S, g) if S else None
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    ref, mass, size, reach = olc.sparse_decode(q, cache, *table, pages, old, **scales)
    gp = gpu(pages) if S else None
    out = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), gp, **gpu_scales(scales))
    check_out(out, ref, size, reach, D, fmt)
    gm = gpu(old)
    out2 = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), gp, key_mass=gm, **gpu_scales(scales))
    assert torch.equal(out.view(torch.int16), out2.view(torch.int16))
    check_mass(gm, mass, old, reach.max(), D, n_add=8)
    assert torch.equal(gm.cpu()[mass == old.double()], old[mass == old.double()])  # rows that were not attended to
    assert q35.device_status() == 0


@pytest.mark.parametrize("fmt,D,HKV,G,n", [("bf16", 256, 4, 2, 57344), ("int8", 128, 8, 3, 86016), ("e4m3c", 64, 16, 1, 57344)])
def test_sparse_decode_of_many_rows_of_all_lengths(fmt, D, HKV, G, n):
    """all pages of so many rows that every CTA gets an equal share of them, from none to half of them in one sequence"""
    import ax_dsl_kernels_b200 as q35
    ctxs, P = [0, 1, n // 2, 0, 33, n // 2 + 77, 0], 64
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 23, extra=10)
    q = q_rows(len(ctxs), HKV * G, D, g, 2.0)
    kn, vn = q_rows(len(ctxs), HKV, D, g), q_rows(len(ctxs), HKV, D, g)
    spare = torch.arange(cache.shape[0], dtype=torch.int32)[~torch.isin(torch.arange(cache.shape[0]), table[1].long())]
    loc = torch.stack([spare[:len(ctxs)], torch.arange(len(ctxs), dtype=torch.int32)], 1).contiguous()
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    need = q35.workspace_bytes("attn.sparse_decode", q=q, paged_kv_cache=cache, indptr=table[0], indices=table[1],
                               last_page_len=table[2], out=q, **{{"row_scale": "paged_kv_scale"}.get(k, k): v for k, v in scales.items()})
    assert need > 0  # the form with partial results in memory
    ref, mass, size, reach = olc.sparse_decode(q, cache, *table, None, old, **scales, k_new=kn, v_new=vn, cache_location=loc)
    gm = gpu(old)
    args = (gpu(q), gpu(cache), *gpu(table))
    kw = dict(k_new=gpu(kn), v_new=gpu(vn), **gpu_scales(scales))
    out = q35.paged_attention_sparse(*args, key_mass=gm, cache_location=gpu(loc), **kw)
    check_out(out, ref, size, reach, D, fmt)
    check_mass(gm, mass, torch.zeros_like(old), reach.max(), D, n_add=8)
    assert torch.equal(out, q35.paged_attention_sparse(*args, **kw))
    # without the current token the empty sequences give zeros; the others agree with chosen pages that are all of them
    out = q35.paged_attention_sparse(*args, **gpu_scales(scales))
    every = torch.full((len(ctxs), HKV, max(-(-c // P) for c in ctxs)), -1, dtype=torch.int32)
    for b, c in enumerate(ctxs):
        every[b, :, :-(-c // P)] = torch.arange(-(-c // P), dtype=torch.int32)
    other = q35.paged_attention_sparse(*args, gpu(every), **gpu_scales(scales))
    assert (out[[0, 3, 6]] == 0).all()
    assert ((out.float() - other.float()).abs() <= other.float().abs() * 2.0 ** -7 + 1e-5).all()
    assert q35.device_status() == 0


@pytest.mark.parametrize("fmt", ["bf16", "e4m3c", "int8"])
def test_sparse_decode_current_token(fmt):
    import ax_dsl_kernels_b200 as q35
    ctxs, P, HKV, G, D = [0, 1, 64, 130, 500], 64, 2, 8, 128
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 8, extra=8)
    q = q_rows(len(ctxs), HKV * G, D, g, 2.0)
    kn, vn = q_rows(len(ctxs), HKV, D, g), q_rows(len(ctxs), HKV, D, g)
    spare = torch.arange(cache.shape[0], dtype=torch.int32)[~torch.isin(torch.arange(cache.shape[0]), table[1].long())]
    loc = torch.stack([spare[:len(ctxs)], torch.arange(len(ctxs), dtype=torch.int32)], 1).contiguous()
    pages = random_pages(ctxs, P, HKV, 3, g)
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    for pg in (None, pages):
        ref, mass, size, reach = olc.sparse_decode(q, cache, *table, pg, old, k_new=kn, v_new=vn, cache_location=loc,
                                                   sm_scale=0.11, **scales)
        gm = gpu(old)
        out = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), None if pg is None else gpu(pg), key_mass=gm,
                                         k_new=gpu(kn), v_new=gpu(vn), cache_location=gpu(loc), sm_scale=0.11,
                                         **gpu_scales(scales))
        check_out(out, ref, size, reach, D, fmt)
        check_mass(gm, mass, torch.zeros_like(old), reach.max(), D, n_add=8)
        out2 = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), None if pg is None else gpu(pg),
                                          k_new=gpu(kn), v_new=gpu(vn), sm_scale=0.11, **gpu_scales(scales))
        assert torch.equal(out, out2)


def test_sparse_decode_special_values():
    """scores of -inf (a masked key), the lowest and largest finite values, all rows -inf, a NaN in an attended row"""
    import ax_dsl_kernels_b200 as q35
    ctxs, P, HKV, G, D = [40, 40, 40, 40], 16, 1, 4, 64
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 9)
    q = q_rows(4, G, D, g)
    q[:, :, 0] = 1.0
    place = [olc._places(*table, P, b) for b in range(4)]
    for b, rows in ((0, [0, 1, 17, 39]), (1, range(40))):
        for i in rows:
            cache[place[b][0][i], 0, place[b][1][i], 0] = 0.0
            cache[place[b][0][i], 0, place[b][1][i], 0, 0] = float("-inf")
    cache[place[2][0][5], 0, place[2][1][5], 0] = 0.0
    cache[place[2][0][5], 0, place[2][1][5], 0, 0] = -3.3e38
    cache[place[3][0][7], 1, place[3][1][7], 0, 3] = float("nan")
    # q * 0 stays 0 and q * -inf is -inf: no NaN from other channels
    old = torch.zeros((cache.shape[0], P, HKV))
    ref, mass, size, reach = olc.sparse_decode(q, cache, *table, None, old)
    assert (ref[1] == 0).all() and not ref[0].isnan().any()
    gm = gpu(old)
    out = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table), key_mass=gm)
    fine = reach.where(reach.isfinite() & (reach < 1e6), torch.full_like(reach, 40.0))  # masked keys carry no weight
    check_out(out, ref, size, fine, D)
    assert (gm.cpu()[place[1][0], place[1][1]] == 0).all()
    check_mass(gm, mass, old, 40.0, D, n_add=8)


def test_sparse_decode_of_all_pages_equals_dense_decode():
    import ax_dsl_kernels_b200 as q35
    ctxs, P, HKV, G, D = [5000, 1, 333], 64, 2, 8, 256
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 10)
    q = q_rows(3, HKV * G, D, g)
    dense = q35.paged_attention_decode(gpu(q), gpu(cache), *gpu(table)).float()
    got = q35.paged_attention_sparse(gpu(q), gpu(cache), *gpu(table)).float()
    # both round nearly the same fp32 value: at most one step apart
    assert ((got - dense).abs() <= dense.abs() * 2.0 ** -7 + 1e-5).all()


# ---------------------------------------------------------------------------------------------------- key mass
@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("D,HKV,G,P", [(256, 2, 8, 64), (128, 1, 16, 16), (64, 4, 1, 7), (64, 2, 5, 100)])
def test_key_mass(fmt, D, HKV, G, P):
    import ax_dsl_kernels_b200 as q35
    ctxs, T = [300, 64, 1, 0, 77, 513], [33, 64, 1, 0, 0, 130]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 11)
    cache, used = poison_behind(cache, table, P)
    q = q_rows(sum(T), HKV * G, D, g, 2.0)
    qo = torch.tensor([0, *torch.tensor(T).cumsum(0).tolist()], dtype=torch.int32)
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    for acc in (False, True):
        ref, reach = olc.key_mass(q, cache, qo, *table, old, accumulate=acc, **scales)
        gm = gpu(old)
        q35.paged_key_mass(gpu(q), gpu(cache), gpu(qo), *gpu(table), gm, accumulate=acc, **gpu_scales(scales))
        check_mass(gm, ref, torch.zeros_like(old), reach, D, n_add=max(T) * G)
        assert torch.equal(gm.cpu()[~used], old[~used])
    assert q35.device_status() == 0


@pytest.mark.parametrize("HKV,G,D,T", [(40, 1, 64, [3, 0, 130, 1]), (24, 8, 128, [20, 37, 0, 16]), (16, 6, 256, [5, 40, 64, 0])])
def test_key_mass_of_many_tiles(HKV, G, D, T):
    """several tiles to a CTA: of other sequences and heads, with windows of other lengths, and none"""
    import ax_dsl_kernels_b200 as q35
    ctxs, P = [1300, 400, 700, 1000], 64
    cache, table, scales, g = make(ctxs, P, HKV, D, "bf16", 32)
    cache, used = poison_behind(cache, table, P)
    q = q_rows(sum(T), HKV * G, D, g, 2.0)
    qo = torch.tensor([0, *torch.tensor(T).cumsum(0).tolist()], dtype=torch.int32)
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    for acc in (False, True):
        ref, reach = olc.key_mass(q, cache, qo, *table, old, accumulate=acc)
        gm = gpu(old)
        q35.paged_key_mass(gpu(q), gpu(cache), gpu(qo), *gpu(table), gm, accumulate=acc)
        check_mass(gm, ref, torch.zeros_like(old), reach, D, n_add=max(T) * G)
        assert torch.equal(gm.cpu()[~used], old[~used])
    assert q35.device_status() == 0


@pytest.mark.parametrize("T", [1, 2, 17, 700])
def test_key_mass_weights_sum_to_the_number_of_query_rows(T):
    import ax_dsl_kernels_b200 as q35
    ctx, P, HKV, G, D = 1900, 64, 2, 8, 256
    cache, table, _, g = make([ctx], P, HKV, D, "bf16", 12)
    q = q_rows(T, HKV * G, D, g, 2.0)
    qo = torch.tensor([0, T], dtype=torch.int32)
    gm = torch.zeros((cache.shape[0], P, HKV), device="cuda")
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(qo), *gpu(table), gm)
    # reach: |q| . |k| scale <= 2 * 256 * (2 / pi) / 16 on average, below 40 for every pair of these seeds' normal rows
    assert torch.allclose(gm.double().sum((0, 1)).cpu(), torch.full((HKV,), float(T * G), dtype=torch.float64),
                          rtol=2 * 260 * 2.0 ** -23 * 40 + 2.0 ** -18 + 2.0 ** -14)
    one = q35.paged_attention_sparse(gpu(q[-1:]), gpu(cache), *gpu(table), key_mass=(gn := torch.zeros_like(gm)))
    assert one.isfinite().all()
    if T == 1:  # one query: both operators state the same weights
        ref, _, _, reach = olc.sparse_decode(q, cache, *table, None, None)
        assert ((gm - gn).abs() <= gn * 2 * (2 * 260 * 2.0 ** -23 * float(reach.max()) + 2.0 ** -18) + 1e-30).all()


def test_weights_of_shared_pages_add_up():
    """eight sequences that share their first pages: every row gets the weight of all of them.  Eight terms in any order:
    seven roundings of 2^-24 more than check_mass counts"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, n = 16, 2, 4, 128, 8
    ctxs = [200 + 7 * i for i in range(n)]
    cache, (indptr, indices, last), _, g = make(ctxs, P, HKV, D, "bf16", 31)
    for b in range(1, n):  # the first ten pages are the first sequence's
        indices[int(indptr[b]):int(indptr[b]) + 10] = indices[:10]
    table = (indptr, indices, last)
    T = [5 + b for b in range(n)]
    q, qo = q_rows(sum(T), HKV * G, D, g, 2.0), torch.tensor([0, *torch.tensor(T).cumsum(0).tolist()], dtype=torch.int32)
    old = torch.rand((cache.shape[0], P, HKV), generator=g)
    ref, reach = olc.key_mass(q, cache, qo, *table, old, accumulate=True)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(qo), *gpu(table), gm, accumulate=True)
    check_mass(gm, ref, torch.zeros_like(old), reach, D, n_add=sum(T) * G)
    q1 = q_rows(n, HKV * G, D, g, 2.0)
    _, ref, _, reach = olc.sparse_decode(q1, cache, *table, None, old)
    gm = gpu(old)
    q35.paged_attention_sparse(gpu(q1), gpu(cache), *gpu(table), key_mass=gm)
    check_mass(gm, ref, torch.zeros_like(old), float(reach.max()), D, n_add=n * G)


def test_key_mass_special_values():
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D = 16, 1, 4, 64
    cache, table, _, g = make([50, 50], P, HKV, D, "bf16", 13)
    q = q_rows(20, G, D, g)
    q[:, :, 0] = 1.0
    qo = torch.tensor([0, 10, 20], dtype=torch.int32)
    place = [olc._places(*table, P, b) for b in range(2)]
    for b, rows in ((0, [0, 3, 49]), (1, range(50))):
        for i in rows:
            cache[place[b][0][i], 0, place[b][1][i], 0] = 0.0
            cache[place[b][0][i], 0, place[b][1][i], 0, 0] = float("-inf")
    cache[place[0][0][48], 0, place[0][1][48], 0, 5] = float("nan")  # masked for all queries but the last two
    old = torch.zeros((cache.shape[0], P, HKV))
    ref, _ = olc.key_mass(q[:], cache, qo, *table, old)
    gm = gpu(old)
    q35.paged_key_mass(gpu(q), gpu(cache), gpu(qo), *gpu(table), gm)
    assert torch.equal(gm.cpu().isnan(), ref.isnan()) and ref.isnan().any()
    assert (gm.cpu()[place[1][0], place[1][1]] == 0).all()


# ---------------------------------------------------------------------------------------------------- eviction
@pytest.mark.parametrize("fmt", FMT[:1] + FMT[2:])
@pytest.mark.parametrize("P,HKV,D", [(64, 2, 256), (16, 3, 64), (7, 1, 128)])
@pytest.mark.parametrize("K,first,last", [(1, 0, 0), (63, 4, 16), (100, 0, 7), (100, 90, 90), (2000, 3, 3)])
def test_evict(fmt, P, HKV, D, K, first, last):
    import ax_dsl_kernels_b200 as q35
    ctxs = [1, 0, 63, 64, 100, 101, 700, 1300]
    cache, table, scales, g = make(ctxs, P, HKV, D, fmt, 14)
    mass = torch.randn((cache.shape[0], P, HKV), generator=g).mul(2).exp()
    ref, rcache, rmass, rrs = olc.evict(cache, mass, *table, K, first, last, scales.get("row_scale"))
    gc, gm, gs = gpu(cache), gpu(mass), gpu_scales(scales)
    kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=first, keep_last=last, **gs)
    assert torch.equal(kept.cpu(), ref)
    assert torch.equal(gc.cpu().view(torch.uint8), rcache.view(torch.uint8))
    assert torch.equal(gm.cpu(), rmass)
    if rrs is not None:
        assert torch.equal(gs["paged_kv_scale"].cpu(), rrs)
    assert q35.device_status() == 0


def test_evict_from_more_rows_than_fit_on_chip():
    """60001 rows: the choice works from scratch memory, the moves take many rounds; a whole number of them and not"""
    import ax_dsl_kernels_b200 as q35
    for ctx, K in ((60001, 50000), (60001, 3 * 6144), (49152, 49151), (50000, 7)):
        cache, table, scales, g = make([ctx, 300], 64, 1, 64, "int8", 21)
        mass = torch.randn((cache.shape[0], 64, 1), generator=g).mul(2).exp()
        ref, rcache, rmass, rrs = olc.evict(cache, mass, *table, K, 4, 100, scales["row_scale"])
        gc, gm, gs = gpu(cache), gpu(mass), gpu_scales(scales)
        kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=4, keep_last=100, **gs)
        assert torch.equal(kept.cpu(), ref)
        assert torch.equal(gc.cpu(), rcache) and torch.equal(gm.cpu(), rmass) and torch.equal(gs["paged_kv_scale"].cpu(), rrs)
    assert q35.device_status() == 0


@pytest.mark.parametrize("n,long,K", [(76, 60001, 40000), (76, 20000, 1500), (40, 60001, 900), (40, 130000, 100000), (16, 9000, 333)])
def test_evict_of_many_rows_of_all_lengths(n, long, K):
    """one, two and four blocks to a row's choice: keys in registers, in shared memory, in scratch memory; equal weights
    across the blocks' borders"""
    import ax_dsl_kernels_b200 as q35
    ctxs = [long] + [(97 * i) % 2000 for i in range(n - 1)]
    cache, table, scales, g = make(ctxs, 64, 1, 64, "int8", 24)
    for mass in (torch.randn((cache.shape[0], 64, 1), generator=g).mul(2).exp(),
                 torch.randint(0, 5, (cache.shape[0], 64, 1), generator=g).float()):
        ref, rcache, rmass, rrs = olc.evict(cache, mass, *table, K, 3, 60, scales["row_scale"])
        gc, gm, gs = gpu(cache), gpu(mass), gpu_scales(scales)
        kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=3, keep_last=60, **gs)
        assert torch.equal(kept.cpu(), ref)
        assert torch.equal(gc.cpu(), rcache) and torch.equal(gm.cpu(), rmass) and torch.equal(gs["paged_kv_scale"].cpu(), rrs)
    assert q35.device_status() == 0


@pytest.mark.parametrize("ctx,K", [(5000, 4096), (9000, 1100)])
def test_evict_ties_and_special_values(ctx, K):
    import ax_dsl_kernels_b200 as q35
    cache, table, _, g = make([ctx, 300], 64, 2, 64, "bf16", 15)
    mass = torch.randint(0, 3, (cache.shape[0], 64, 2), generator=g).float()  # three values only
    pg, row = olc._places(*table, 64, 0)
    mass[pg[::7], row[::7]] = float("nan")
    mass[pg[5], row[5]] = float("inf")
    mass[pg[6], row[6]] = float("-inf")
    mass[pg[11::13], row[11::13]] = -0.0
    ref, rcache, rmass, _ = olc.evict(cache, mass, *table, K, 2, 5)
    gc, gm = gpu(cache), gpu(mass)
    kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=2, keep_last=5)
    assert torch.equal(kept.cpu(), ref)
    assert torch.equal(gc.cpu(), rcache)
    assert torch.equal(gm.cpu().view(torch.int32), rmass.view(torch.int32))


# ---------------------------------------------------------------------------------------------------- together
def test_decode_loop_with_all_of_them():
    """prompt -> weights of its last queries -> eviction -> bounds -> steps that choose pages, attend, add weights and
    look at the last page again; every step against the oracle on the same state"""
    import ax_dsl_kernels_b200 as q35
    P, HKV, G, D, K = 16, 2, 4, 64, 100
    ctxs = [260, 90, 171]
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 16)
    W = 8
    q = q_rows(3 * W, HKV * G, D, g, 2.0)
    qo = torch.tensor([0, W, 2 * W, 3 * W], dtype=torch.int32)
    gc, gm = gpu(cache), torch.zeros((cache.shape[0], P, HKV), device="cuda")
    q35.paged_key_mass(gpu(q), gc, gpu(qo), *gpu(table), gm)
    ref, reach = olc.key_mass(q, cache, qo, *table, torch.zeros(gm.shape))
    check_mass(gm, ref, torch.zeros(gm.shape), reach, D, n_add=W * G)
    mass = gm.cpu()  # the choice is checked on the GPU's own weights
    rk, cache, mass, _ = olc.evict(cache, mass, *table, K, 2, W)
    kept = q35.evict_keys(gc, gm, *gpu(table), K, keep_first=2, keep_last=W)
    assert torch.equal(kept.cpu(), rk) and torch.equal(gc.cpu(), cache) and torch.equal(gm.cpu(), mass)
    ctxs = [min(c, K) for c in ctxs]
    indptr, indices, _ = table
    pages_of = [indices[int(indptr[b]):int(indptr[b + 1])] for b in range(3)]
    bounds = None
    for step in range(3):
        n = [-(-(c + 1) // P) for c in ctxs]
        loc = torch.tensor([[int(pages_of[b][c // P]), c % P] for b, c in enumerate(ctxs)], dtype=torch.int32)
        kn, vn = q_rows(3, HKV, D, g), q_rows(3, HKV, D, g)
        q35.kv_write(gc, gpu(loc), gpu(kn), gpu(vn))
        for b in range(3):
            cache[loc[b, 0], 0, loc[b, 1]], cache[loc[b, 0], 1, loc[b, 1]] = kn[b], vn[b]
            gm[loc[b, 0].item(), loc[b, 1].item()] = 0
        ctxs = [c + 1 for c in ctxs]
        now = (torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32),
               torch.cat([pages_of[b][:n[b]] for b in range(3)]).contiguous(),
               torch.tensor([c - (m - 1) * P for c, m in zip(ctxs, n)], dtype=torch.int32))
        gt = gpu(now)
        if bounds is None:
            bounds = q35.page_key_bounds(gc, *gt)
        else:
            q35.page_key_bounds(gc, *gt, bounds, first_page=gpu(torch.tensor([m - 1 for m in n], dtype=torch.int32)))
        rb = olc.page_bounds(cache, *now, torch.zeros(bounds.shape, dtype=torch.bfloat16))
        listed = now[1].long()
        assert torch.equal(bounds.cpu()[listed], rb[listed])
        qs = q_rows(3, HKV * G, D, g, 2.0)
        sel = q35.select_pages(gpu(qs), bounds, *gt, 3, keep_first=1, keep_last=1)
        assert torch.equal(sel.cpu(), olc.select_pages(qs, rb, *now, 3, 1, 1))
        before = gm.cpu()
        out = q35.paged_attention_sparse(gpu(qs), gc, *gt, sel, key_mass=gm)
        ref, rmass, size, reach = olc.sparse_decode(qs, cache, *now, sel.cpu(), before)
        check_out(out, ref, size, reach, D)
        check_mass(gm, rmass, before, reach.max(), D, n_add=8)
    assert q35.device_status() == 0


def test_captured_and_replayed_and_on_another_stream():
    import ax_dsl_kernels_b200 as q35
    ctxs, P, HKV, G, D, S = [900, 64, 1, 431], 64, 2, 8, 128, 4
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 17)
    q, q2 = q_rows(4, HKV * G, D, g, 2.0), q_rows(4, HKV * G, D, g, 2.0)
    T = [3, 64, 1, 20]
    qo = gpu(torch.tensor([0, *torch.tensor(T).cumsum(0).tolist()], dtype=torch.int32))
    qw = gpu(q_rows(sum(T), HKV * G, D, g, 2.0))
    gt, gc = gpu(table), gpu(cache)
    gq, out = gpu(q), torch.empty((4, HKV * G, D), dtype=torch.bfloat16, device="cuda")
    sel = torch.empty((4, HKV, S), dtype=torch.int32, device="cuda")
    bounds = torch.zeros((cache.shape[0], 2, HKV, D), dtype=torch.bfloat16, device="cuda")
    gm = torch.zeros((cache.shape[0], P, HKV), device="cuda")
    kept = torch.empty((4, HKV, 50), dtype=torch.int32, device="cuda")

    def step():
        q35.paged_key_mass(qw, gc, qo, *gt, gm)
        q35.page_key_bounds(gc, *gt, bounds)
        q35.select_pages(gq, bounds, *gt, S, sel, keep_first=1, keep_last=1)
        q35.paged_attention_sparse(gq, gc, *gt, sel, out, key_mass=gm)
        q35.evict_keys(gc, gm, *gt, 50, kept, keep_last=4)

    def state():
        return [t.clone() for t in (out, sel, bounds, gm, kept, gc)]

    def reset(x):
        gc.copy_(cache)
        gq.copy_(x)
        gm.zero_()

    want = []
    for x in (q, q2):
        reset(x)
        step()
        want.append(state())
    side = torch.cuda.Stream()
    reset(q)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(state(), want[0]))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]  # two graphs, one scratch buffer
    for gr in graphs:
        reset(q)
        with torch.cuda.graph(gr):
            step()
    for i in (0, 1, 1, 0):
        reset((q, q2)[i])
        graphs[i].replay()
        assert all(torch.equal(a, b) for a, b in zip(state(), want[i]))
    assert q35.device_status() == 0


def test_first_calls_inside_a_capture():
    """counts and scales that no call has used yet: nothing is copied from the host"""
    import ax_dsl_kernels_b200 as q35
    cache, table, _, g = make([700, 300], 16, 2, 128, "bf16", 23)
    gt, gc, q = gpu(table), gpu(cache), gpu(q_rows(2, 16, 128, g))
    bounds, qo = q35.page_key_bounds(gc, *gt), gpu(torch.tensor([0, 1, 2], dtype=torch.int32))

    def step(first, last, scale):
        pages = q35.select_pages(q, bounds, *gt, 9, keep_first=first, keep_last=last)
        gm = torch.zeros((cache.shape[0], 16, 2), device="cuda")
        out = q35.paged_attention_sparse(q, gc, *gt, pages, key_mass=gm, sm_scale=scale)
        q35.paged_key_mass(q, gc, qo, *gt, gm, accumulate=True, sm_scale=scale)
        return pages, out, gm

    step(0, 1, None)  # the library itself is loaded
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(6, 2, 0.0625)
    graph.replay()
    assert not any(k[:2] == (6, 2) for k in q35.long_context._keep)
    for a, b in zip(got, step(6, 2, 0.0625)):
        assert torch.equal(a, b)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], step(6, 2, 0.0625)[0]) and q35.device_status() == 0


def test_a_captured_graph_keeps_its_own_scratch():
    """a call that needs more scratch, made after the capture on the stream of the capture, replaces the eager buffer; the
    graph's addresses stay valid and nobody else's"""
    import ax_dsl_kernels_b200 as q35
    cache, table, _, g = make([700, 900], 64, 2, 128, "bf16", 20)
    gt, gc = gpu(table), gpu(cache)
    q, gm = gpu(q_rows(2, 16, 128, g, 2.0)), torch.zeros((cache.shape[0], 64, 2), device="cuda")
    want = q35.paged_attention_sparse(q, gc, *gt, key_mass=gm)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    out, gm2 = torch.empty_like(want), torch.zeros_like(gm)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        q35.paged_attention_sparse(q, gc, *gt, out=out, key_mass=gm2)
    assert (q.get_device(), stream.cuda_stream) not in q35._lib._ws_cache
    with torch.cuda.stream(stream):
        for n in (1, 40):  # the second needs 40 times the first's
            big = [torch.randn((64 * n, 4), device="cuda").sort().values for _ in range(2)]
            ids, rw = torch.randint(0, 32, (64 * n, 4), dtype=torch.int32, device="cuda"), big[0].contiguous()
            q35.moe_permute(ids, rw, 32, 16)
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(gm, gm2)


def test_both_host_paths_issue_the_same_call():
    """the binding's fast path and the checked one, on a stream given by its handle too; what neither takes is refused"""
    import ax_dsl_kernels_b200 as q35
    from ax_dsl_kernels_b200 import _lib
    cache, table, _, g = make([700, 90], 64, 2, 128, "bf16", 22)
    gt, gc, q = dict(zip(("indptr", "indices", "last_page_len"), gpu(table))), gpu(cache), gpu(q_rows(2, 16, 128, g, 2.0))
    got = []
    side = torch.cuda.Stream()
    for run, kw in ((_lib.run_checked, {}), (_lib.run, {}), (_lib.run, dict(stream=side.cuda_stream))):
        out, gm = torch.empty_like(q), torch.zeros((cache.shape[0], 64, 2), device="cuda")
        torch.cuda.synchronize()
        run("attn.sparse_decode", q=q, paged_kv_cache=gc, **gt, out=out, key_mass=gm, **kw)
        torch.cuda.synchronize()
        got.append((out, gm))
    for out, gm in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(gm, got[0][1])
    bad = dict(q=q, paged_kv_cache=gc, **gt, out=torch.empty_like(q))
    for run in (_lib.run_checked, _lib.run):
        for change, error in ((dict(q=q.cpu()), ValueError), (dict(q=q.transpose(0, 1)), ValueError), (dict(out=3), Exception),
                              (dict(q=q.double()), TypeError), (dict(out=q[:1].clone()), q35.Q35Error)):
            with pytest.raises(error):
                run("attn.sparse_decode", **dict(bad, **change))
        with pytest.raises(q35.Q35Error):
            run("attn.no_such_role", q=q)


# ---------------------------------------------------------------------------------------------------- bad tables
def test_bad_tables_are_recorded_and_touch_nothing():
    """page ids outside the cache, ranges outside the table, lists of pages that are not ascending"""
    import ax_dsl_kernels_b200 as q35
    ctxs, P, HKV, G, D = [100, 100], 16, 2, 4, 64
    cache, table, _, g = make(ctxs, P, HKV, D, "bf16", 18)
    q = gpu(q_rows(2, HKV * G, D, g))
    indptr, indices, last = table
    mass = torch.rand((cache.shape[0], P, HKV), generator=g)
    qo = gpu(torch.tensor([0, 1, 2], dtype=torch.int32))

    def everything(t, pages=None):
        gc, gm = gpu(cache), gpu(mass)
        bounds = q35.page_key_bounds(gc, *t)
        bits = [q35.device_status()]
        q35.select_pages(q, bounds, *t, 3)
        bits.append(q35.device_status())
        q35.paged_attention_sparse(q, gc, *t, pages, key_mass=gm)
        bits.append(q35.device_status())
        q35.paged_key_mass(q, gc, qo, *t, gm)
        bits.append(q35.device_status())
        gm = gpu(mass)
        q35.evict_keys(gc, gm, *t, 40)
        bits.append(q35.device_status())
        return bits, gc, gm

    bad_ids = indices.clone()
    bad_ids[[1, 9]] = torch.tensor([cache.shape[0], -1], dtype=torch.int32)
    bits, _, _ = everything(gpu((indptr, bad_ids, last)))
    assert all(b & 1 for b in bits)
    bad_range = indptr.clone()
    bad_range[2] = 1000
    bits, gc, _ = everything(gpu((bad_range, indices, last)))
    assert all(b & 1 for b in bits)
    rows = olc._places(indptr, indices, last, P, 1)  # the sequence with the bad range counts as empty: its rows stay
    assert torch.equal(gc.cpu()[rows[0], :, rows[1]], cache[rows[0], :, rows[1]])
    bits, gc, _ = everything(gpu((indptr, indices, torch.tensor([P + 1, 4], dtype=torch.int32))))
    assert all(b & 1 for b in bits[:1] + bits[2:])
    # chosen pages: the list ends before the first entry that does not ascend or is no page
    pages = torch.tensor([[[0, 2, 2, 5], [3, 1, -1, -1]], [[0, 6, 7, -1], [-5, 1, 2, 3]]], dtype=torch.int32)
    cut = torch.tensor([[[0, 2, -1, -1], [3, -1, -1, -1]], [[0, 6, -1, -1], [-1, -1, -1, -1]]], dtype=torch.int32)
    got = q35.paged_attention_sparse(q, gpu(cache), *gpu(table), gpu(pages))
    assert q35.device_status() & 1
    assert torch.equal(got, q35.paged_attention_sparse(q, gpu(cache), *gpu(table), gpu(cut)))
    assert q35.device_status() == 0
    # a window longer than its sequence
    long = gpu(torch.tensor([0, 1, 102], dtype=torch.int32))
    gm = gpu(mass)
    q35.paged_key_mass(gpu(q_rows(102, HKV * G, D, g)), gpu(cache), long, *gpu(table), gm)
    assert q35.device_status() & 8
