"""The long-context roles without a GPU: what their contract refuses, what scratch they ask for, and their 64-bit oracle
against independent statements of the same operators."""
import math

import pytest
import torch

from ax_dsl_kernels_b200 import _lib
from ax_dsl_kernels_b200 import long_context as lc
from oracle import long_context as olc

B, HQ, HKV, D, P, PAGES, N = 2, 8, 2, 128, 16, 9, 7
bf16, i32, f32 = torch.bfloat16, torch.int32, torch.float32


def z(*shape, dtype=bf16):
    return torch.zeros(shape, dtype=dtype)


TABLE = dict(indptr=z(B + 1, dtype=i32), indices=z(N, dtype=i32), last_page_len=z(B, dtype=i32))
CACHE = z(PAGES, 2, P, HKV, D)
MASS = z(PAGES, P, HKV, dtype=f32)
ROLES = {
    "attn.page_bounds": dict(TABLE, paged_kv_cache=CACHE, page_bounds=z(PAGES, 2, HKV, D)),
    "attn.select_pages": dict(TABLE, q=z(B, HQ, D), page_bounds=z(PAGES, 2, HKV, D), pages=z(B, HKV, 3, dtype=i32)),
    "attn.sparse_decode": dict(TABLE, q=z(B, HQ, D), paged_kv_cache=CACHE, out=z(B, HQ, D)),
    "attn.key_mass": dict(TABLE, q=z(5, HQ, D), paged_kv_cache=CACHE, qo_indptr=z(B + 1, dtype=i32), key_mass=MASS),
    "attn.evict": dict(TABLE, paged_kv_cache=CACHE, key_mass=MASS, kept=z(B, HKV, 20, dtype=i32)),
}
E4M3 = CACHE.to(torch.float8_e4m3fn)
INT8 = CACHE.to(torch.int8)
ROWS = z(PAGES, 2, P, HKV)
MISSING, DTYPE, SHAPE, UNSUPPORTED = 2, 3, 4, 8


@pytest.mark.parametrize("role", sorted(ROLES))
def test_the_contract_accepts_and_describes(role):
    assert role in _lib.roles()
    table = _lib.io_table(role)
    named = {e[0] for e in table["in"] + table["out"]}
    assert set(ROLES[role]) <= named
    need = _lib.workspace_bytes(role, **ROLES[role])
    assert need >= 0 and need % 256 == 0
    assert (need > 0) == (role in ("attn.select_pages", "attn.key_mass"))
    empty = dict(ROLES[role], indptr=z(1, dtype=i32), last_page_len=z(0, dtype=i32), indices=z(0, dtype=i32))
    for n in ("q", "out", "pages", "kept"):
        if n in empty and not (role == "attn.key_mass" and n == "q"):
            empty[n] = empty[n][:0]
    if "qo_indptr" in empty:
        empty["qo_indptr"] = z(1, dtype=i32)
    assert _lib.workspace_bytes(role, **empty) >= 0


def test_scratch_of_an_eviction_from_a_long_table():
    t = dict(ROLES["attn.evict"], indices=z(5000, dtype=i32))
    assert _lib.workspace_bytes("attn.evict", **t) == 5000 * P * HKV * 4


@pytest.mark.parametrize("role", sorted(r for r in ROLES if r != "attn.select_pages"))
def test_tables_of_more_than_2_30_positions_are_refused(role):
    for n, ok in ((2 ** 30 // P - 1, True), (2 ** 30 // P, False)):
        t = dict(ROLES[role], indices=torch.empty(n, dtype=i32, device="meta"))
        if ok:
            assert _lib.workspace_bytes(role, **t) >= 0
            continue
        with pytest.raises(_lib.Q35Error) as e:
            _lib.workspace_bytes(role, **t)
        assert e.value.status == UNSUPPORTED


def test_scratch_of_the_weights():
    with_mass = dict(ROLES["attn.sparse_decode"], key_mass=MASS)
    assert _lib.workspace_bytes("attn.sparse_decode", **with_mass) == HKV * N * P * 32
    assert _lib.workspace_bytes("attn.sparse_decode", **dict(with_mass, pages=z(B, HKV, 4, dtype=i32))) == B * HKV * 4 * P * 32


@pytest.mark.parametrize("role,change,status", [
    *[(r, {"indptr": None}, MISSING) for r in sorted(ROLES)],
    *[(r, {"last_page_len": z(B - 1, dtype=i32)}, SHAPE) for r in sorted(ROLES)],
    *[(r, {"indices": z(N, dtype=f32)}, DTYPE) for r in sorted(ROLES)],
    *[(r, {"paged_kv_cache": CACHE.float()}, DTYPE) for r in sorted(ROLES) if r != "attn.select_pages"],
    # an int8 cache without its row scales, scales without an int8 cache, of another size
    *[(r, {"paged_kv_cache": INT8}, DTYPE) for r in sorted(ROLES) if r != "attn.select_pages"],
    *[(r, {"paged_kv_scale": ROWS}, DTYPE) for r in sorted(ROLES) if r != "attn.select_pages"],
    *[(r, {"paged_kv_cache": E4M3, "paged_kv_scale": ROWS}, DTYPE) for r in sorted(ROLES) if r != "attn.select_pages"],
    *[(r, {"paged_kv_cache": INT8, "paged_kv_scale": ROWS[:-1]}, SHAPE) for r in sorted(ROLES) if r != "attn.select_pages"],
    *[(r, {"paged_kv_cache": CACHE[:0]}, SHAPE) for r in sorted(ROLES) if r != "attn.select_pages"],
    ("attn.page_bounds", {"page_bounds": z(PAGES, 2, HKV, D // 2)}, SHAPE),
    ("attn.page_bounds", {"page_bounds": z(PAGES - 1, 2, HKV, D)}, SHAPE),
    ("attn.page_bounds", {"first_page": z(B - 1, dtype=i32)}, SHAPE),
    ("attn.page_bounds", {"paged_kv_cache": z(PAGES, 2, P, HKV, 24), "page_bounds": z(PAGES, 2, HKV, 24)}, UNSUPPORTED),
    ("attn.select_pages", {"q": z(B, HQ + 1, D)}, SHAPE),
    ("attn.select_pages", {"q": z(B, HQ, D, dtype=f32)}, DTYPE),
    ("attn.select_pages", {"pages": z(B, HKV, 0, dtype=i32)}, SHAPE),
    ("attn.select_pages", {"pages": z(B, HKV + 1, 3, dtype=i32)}, SHAPE),
    ("attn.select_pages", {"keep": z(3, dtype=i32)}, SHAPE),
    ("attn.select_pages", {"q": z(B, HQ, 96), "page_bounds": z(PAGES, 2, HKV, 96)}, UNSUPPORTED),
    ("attn.sparse_decode", {"q": z(B, 18, D), "out": z(B, 18, D)}, UNSUPPORTED),  # nine query heads per KV head
    ("attn.sparse_decode", {"q": z(B, HQ, 64), "out": z(B, HQ, 64)}, SHAPE),
    ("attn.sparse_decode", {"out": z(B, HQ, D // 2)}, SHAPE),
    ("attn.sparse_decode", {"paged_kv_cache": z(PAGES, 2, 24, HKV, D)}, UNSUPPORTED),
    ("attn.sparse_decode", {"pages": z(B, HKV, dtype=i32)}, SHAPE),
    ("attn.sparse_decode", {"sm_scale": z(2, dtype=f32)}, SHAPE),
    ("attn.sparse_decode", {"kv_scale": z(2, HKV, dtype=f32)}, DTYPE),
    ("attn.sparse_decode", {"paged_kv_cache": E4M3, "kv_scale": z(2, HKV + 1, dtype=f32)}, SHAPE),
    ("attn.sparse_decode", {"k_new": z(B, HKV, D)}, MISSING),
    ("attn.sparse_decode", {"k_new": z(B, HKV, D), "v_new": z(B, HKV, D // 2)}, SHAPE),
    ("attn.sparse_decode", {"k_new": z(B, HKV, D), "v_new": z(B, HKV, D), "key_mass": MASS}, MISSING),
    ("attn.sparse_decode", {"cache_location": z(B, 2, dtype=i32)}, MISSING),
    ("attn.sparse_decode", {"key_mass": MASS[:-1]}, SHAPE),
    ("attn.sparse_decode", {"key_mass": MASS.to(bf16)}, DTYPE),
    ("attn.key_mass", {"key_mass": MASS[:-1]}, SHAPE),
    ("attn.key_mass", {"qo_indptr": None}, MISSING),
    ("attn.key_mass", {"qo_indptr": z(B, dtype=i32)}, SHAPE),
    ("attn.key_mass", {"q": z(5, HQ, 96), "paged_kv_cache": z(PAGES, 2, P, HKV, 96)}, UNSUPPORTED),
    ("attn.evict", {"kept": z(B, HKV, 0, dtype=i32)}, SHAPE),
    ("attn.evict", {"kept": z(B, HKV + 1, 20, dtype=i32)}, SHAPE),
    ("attn.evict", {"key_mass": None}, MISSING),
    ("attn.evict", {"key_mass": MASS[:-1]}, SHAPE),
    ("attn.evict", {"paged_kv_cache": z(PAGES, 2, P, HKV, 16)}, UNSUPPORTED),
])
def test_the_contract_refuses(role, change, status):
    t = dict(ROLES[role], **change)
    t = {k: v for k, v in t.items() if v is not None}
    with pytest.raises(_lib.Q35Error) as e:
        _lib.workspace_bytes(role, **t)
    assert e.value.status == status, str(e.value)


def test_host_functions_refuse():
    table = tuple(TABLE.values())
    with pytest.raises(ValueError):  # no CPU path
        lc.page_key_bounds(CACHE, *table)
    with pytest.raises(ValueError):
        lc.select_pages(z(B, HQ, D), z(PAGES, 2, HKV, D), *table, 3, keep_first=-1)
    with pytest.raises(ValueError):
        lc.select_pages(z(B, HQ, D), z(PAGES, 2, HKV, D), *table, 3, out=z(B, HKV, 4, dtype=i32))
    with pytest.raises(ValueError):
        lc.evict_keys(CACHE, MASS, *table, 3, kept=z(B, HKV, 4, dtype=i32))
    with pytest.raises(ValueError):  # strided views are not bound
        lc.paged_attention_sparse(z(B, D, HQ).transpose(1, 2), CACHE, *table)


# ------------------------------------------------------------------------------------------------------ the oracle
def _case(ctxs, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = [-(-c // P) for c in ctxs]
    cache = torch.randn((sum(n) + 2, 2, P, HKV, D), generator=g).to(bf16)
    perm = torch.randperm(sum(n) + 2, generator=g).to(i32)
    table = (torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=i32), perm[:sum(n)],
             torch.tensor([c - (m - 1) * P if m else 0 for c, m in zip(ctxs, n)], dtype=i32))
    return cache, table, torch.randn((len(ctxs), HQ, D), generator=g).to(bf16), g


def test_oracle_attention_and_weights_against_torch():
    ctxs = [1, 50, 33]
    cache, table, q, _ = _case(ctxs)
    out, mass, size, _ = olc.sparse_decode(q, cache, *table, None, torch.zeros((cache.shape[0], P, HKV)))
    for b, c in enumerate(ctxs):
        pg = table[1][int(table[0][b]):int(table[0][b + 1])].long()
        k, v = (cache[pg, i].reshape(-1, HKV, D)[:c].double().transpose(0, 1) for i in (0, 1))
        want = torch.nn.functional.scaled_dot_product_attention(q[b].double().unsqueeze(1), k.repeat_interleave(HQ // HKV, 0),
                                                                v.repeat_interleave(HQ // HKV, 0)).squeeze(1)
        assert torch.allclose(out[b], want, atol=1e-12)
        assert mass[pg].sum().item() == pytest.approx(HQ, rel=1e-12)
    assert (size >= out.abs() - 1e-12).all()
    some = torch.tensor([[[0, -1], [0, -1]], [[1, 3], [0, 2]], [[-1, -1], [2, -1]]], dtype=i32)
    out, mass, _, _ = olc.sparse_decode(q, cache, *table, some, torch.zeros((cache.shape[0], P, HKV)))
    assert (out[2, :HQ // HKV] == 0).all() and (out[2, HQ // HKV:] != 0).any()
    assert mass.sum().item() == pytest.approx(HQ * 3 - HQ // HKV, rel=1e-12)


def test_oracle_window_weights_are_those_of_single_queries():
    ctxs = [40, 20]
    cache, table, _, g = _case(ctxs, 1)
    q = torch.randn((5, HQ, D), generator=g).to(bf16)
    mass, _ = olc.key_mass(q, cache, torch.tensor([0, 3, 5], dtype=i32), *table, torch.zeros((cache.shape[0], P, HKV)))
    want = torch.zeros_like(mass)
    for b, (t0, T) in enumerate(((0, 3), (3, 2))):
        for t in range(T):  # the sequence cut off behind the query's own row
            n = ctxs[b] - T + t + 1
            pages = -(-n // P)
            lo = int(table[0][b])
            cut = (torch.tensor([0, pages], dtype=i32), table[1][lo:lo + pages], torch.tensor([n - (pages - 1) * P], dtype=i32))
            want += olc.sparse_decode(q[t0 + t:t0 + t + 1], cache, *cut, None, torch.zeros_like(mass))[1]
    assert torch.allclose(mass, want, atol=1e-12)


def test_oracle_bounds_hold_and_choose():
    cache, table, q, _ = _case([100, 16, 64], 2)
    bounds = olc.page_bounds(cache, *table, torch.zeros((cache.shape[0], 2, HKV, D), dtype=bf16))
    for b in range(3):
        k, _ = olc._rows(cache, *table, b)
        for h in range(HKV):
            s = olc.page_scores(q, bounds, *table, b, h)
            real = (q[b, h * 4:h * 4 + 4].double() @ k[:, h].T).amax(0)
            for i in range(len(s)):
                assert s[i] >= real[i * P:(i + 1) * P].max()
    assert olc.best([3.0, 5.0, 5.0, math.nan, 5.0, -math.inf], 2, 0, 0) == [1, 2]
    assert olc.best([3.0, 5.0, 5.0, math.nan, 5.0, -math.inf], 3, 1, 1) == [0, 1, 5]
    assert olc.best([0.0, 1.0, 2.0, 3.0], 2, 3, 3) == [2, 3]
    assert olc.best([0.0, -0.0, 0.0], 2, 0, 0) == [0, 1]


def test_oracle_eviction_moves_rows_in_order():
    cache, table, _, g = _case([50, 20, 0], 3)
    mass = torch.rand((cache.shape[0], P, HKV), generator=g)
    kept, new, new_mass, _ = olc.evict(cache, mass, *table, 24, 2, 3)
    assert (kept[2] == -1).all() and (kept[1, :, 20:] == -1).all() and (kept[1, :, :20] == torch.arange(20)).all()
    for h in range(HKV):
        assert kept[0, h, :2].tolist() == [0, 1] and kept[0, h, -3:].tolist() == [47, 48, 49]
        pg, row = olc._places(*table, P, 0)
        j = kept[0, h].long()
        assert torch.equal(new[pg[:24], :, row[:24], h], cache[pg[j], :, row[j], h])
        assert torch.equal(new_mass[pg[:24], row[:24], h], mass[pg[j], row[j], h])
        assert torch.equal(new[pg[24:], :, row[24:], h], cache[pg[24:], :, row[24:], h])
