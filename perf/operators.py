"""Long contexts over the paged KV cache, as measured work: bounds of every page's keys, choice of the pages a query
attends to, attention over the chosen pages (with the softmax weights added up per cached row), the weights a window of
queries gives to every cached row, and the eviction of the rows that got least.

`run` computes an operator in its plain form (elementary torch operations in fp32, in fp64 where a choice depends on the
order of the sums), or, with `own`, by the calls a user of the package makes.

All operators share one page table, as in the package: sequence b owns the pages indices[indptr[b]] ..
indices[indptr[b + 1] - 1] of a cache [pages, 2, P, HKV, D] (K rows, V rows) and has ctx_b cached rows, the last page
holding last_page_len[b] of them.  Row i of sequence b and KV head h is row i % P of its page i // P.
Formats: "bf16"; "e4m3" with one scale per head and K / V; "e4m3c", the constant form (stored = 8 x value); "int8", one
bf16 scale per cached row and head, value = bf16(int8 * scale)."""
import math
import random

import torch

own = False

HEADS = ((16, 2, 256), (24, 4, 256), (8, 2, 128), (16, 2, 128), (4, 4, 64), (8, 1, 256), (10, 2, 64))


def listed():
    return [
        # a decode step of 64 sequences: each has just filled in a row of its last page, only that page is looked at again
        dict(name="bounds_decode", op="bounds", B=64, ctx=4096, ragged=True, HQ=16, HKV=2, D=256, P=64, kv="bf16", last_only=True),
        # a batch of prompts has just been written
        dict(name="bounds_prompt", op="bounds", B=16, ctx=16384, ragged=True, HQ=16, HKV=2, D=256, P=64, kv="bf16", last_only=False),
        # one user's decode step at 16k: 256 pages, 16 of them chosen -- latency
        dict(name="select_one", op="select", B=1, ctx=16384, ragged=False, HQ=16, HKV=2, D=256, P=64, S=16, first=1, last=2),
        # the decode group of 8 sequences at 131072
        dict(name="select_group", op="select", B=8, ctx=131072, ragged=False, HQ=24, HKV=4, D=256, P=64, S=64, first=1, last=4),
        # one user's decode step over 16 chosen pages -- latency
        dict(name="attend_one", op="attend", B=1, ctx=16384, ragged=False, HQ=16, HKV=2, D=256, P=64, kv="bf16", S=16, mass=False),
        # 64 sequences at 16k, 4096 of their rows each
        dict(name="attend_batch", op="attend", B=64, ctx=16384, ragged=False, HQ=16, HKV=2, D=256, P=64, kv="bf16", S=64, mass=False),
        # decode over a cache that eviction holds near 4096 rows: every row is read, the weights are added up
        dict(name="attend_mass_e4m3", op="attend", B=32, ctx=4161, ragged=True, HQ=24, HKV=4, D=256, P=64, kv="e4m3", S=0, mass=True),
        # small pages, int8 rows, chosen pages and weights together
        dict(name="attend_int8", op="attend", B=24, ctx=9001, ragged=True, HQ=8, HKV=2, D=128, P=16, kv="int8", S=100, mass=True),
        # the last 32 queries of four prompts look back over 8192 rows
        dict(name="mass_window", op="mass", B=4, ctx=8192, ragged=True, HQ=16, HKV=2, D=256, P=64, kv="bf16", T=32),
        # a long window: 2047 queries over 8192 rows
        dict(name="mass_prompt", op="mass", B=1, ctx=8192, ragged=False, HQ=16, HKV=2, D=256, P=64, kv="e4m3", T=2047),
        # one sequence is one page over its budget of 4096 rows -- latency
        dict(name="evict_one", op="evict", B=1, ctx=4160, ragged=False, HQ=16, HKV=2, D=256, P=64, kv="bf16", K=4096, first=4, last=64),
        # 16 prompts of up to 16k cut to 4000 rows each
        dict(name="evict_prompt", op="evict", B=16, ctx=16384, ragged=True, HQ=16, HKV=2, D=256, P=64, kv="bf16", K=4000, first=4, last=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("bounds", "select", "attend", "attend", "mass", "evict"))
    HQ, HKV, D = rng.choice(HEADS)
    P = rng.choice((16, 32, 64, 64, 128))
    case = dict(op=op, ragged=rng.random() < 0.6, HQ=HQ, HKV=HKV, D=D, P=P)
    row = HKV * D * 4  # bytes of K and V of one bf16 row
    if op == "select":
        B = _log(rng, 1, 48)
        n = _log(rng, 32, max(40, min(4096, 40_000_000 // (B * HKV * D * 4))))
        first, last = rng.randrange(0, 3), rng.randrange(0, 4)
        S = _log(rng, first + last + 3, min(256, n // 2))
        return dict(case, B=B, ctx=n * P - rng.randrange(P), S=S, first=first, last=last)
    if op == "bounds":
        B = _log(rng, 1, 64)
        return dict(case, B=B, ctx=_log(rng, 1, max(64, min(131072, 400_000_000 // (B * row)))), last_only=rng.random() < 0.4,
                    kv=rng.choice(("bf16", "e4m3", "e4m3c", "int8")))
    if op == "attend":
        B = _log(rng, 1, 64)
        ctx = _log(rng, 1, max(64, min(32768, 1_000_000_000 // (B * row))))
        S = _log(rng, 1, min(256, max(2, ctx // P))) if rng.random() < 0.6 or ctx * B * row > 300_000_000 else 0
        while S * P * B * row > 400_000_000:
            S = max(1, S // 2)
        return dict(case, B=B, ctx=ctx, kv=rng.choice(("bf16", "bf16", "e4m3", "e4m3c", "int8")), S=S, mass=rng.random() < 0.5)
    if op == "mass":
        B = _log(rng, 1, 8)
        T = _log(rng, 1, 600)
        ctx = _log(rng, max(T, 16), max(T + 16, min(32768, 250_000_000 // (B * T * HQ))))
        return dict(case, B=B, T=T, ctx=ctx, kv=rng.choice(("bf16", "bf16", "e4m3", "e4m3c", "int8")))
    B = _log(rng, 1, 32)
    ctx = _log(rng, 16, max(64, min(65536, 400_000_000 // (B * row))))
    K = max(1, int(ctx * rng.uniform(0.1, 1.1)))
    return dict(case, B=B, ctx=ctx, kv=rng.choice(("bf16", "bf16", "e4m3c")), K=K, first=rng.randrange(0, 8), last=rng.randrange(0, min(K, 256)))


def _lens(case):
    """cached rows of every sequence: ctx, or for a ragged batch ctx, 1 and lengths between ctx / 8 and ctx"""
    B, ctx = case["B"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * B
    r = random.Random(B * 1_000_003 + ctx)
    low = max(case.get("T", 1), ctx // 8, 1)
    got = [ctx] + [r.randint(min(low, ctx), ctx) for _ in range(B - 1)]
    if B >= 6 and "T" not in case:
        got[2] = 1
    return got


def _pages(case):
    return [-(-n // case["P"]) for n in _lens(case)]


def work(case):
    lens, HQ, HKV, D, P, B = _lens(case), case["HQ"], case["HKV"], case["D"], case["P"], case["B"]
    elt = 2 if case.get("kv", "bf16") == "bf16" else 1
    rs = 2 if case.get("kv") == "int8" else 0  # row scale
    op = case["op"]
    if op == "bounds":
        rows = sum((n - 1) % P + 1 for n in lens) if case["last_only"] else sum(lens)
        pages = B if case["last_only"] else sum(_pages(case))
        return {"bytes": rows * HKV * (D * elt + rs) + pages * 4 * HKV * D, "flops": 2 * rows * HKV * D}
    if op == "select":
        pages = sum(_pages(case))
        return {"bytes": pages * 4 * HKV * D + 2 * B * HQ * D + 4 * B * HKV * case["S"], "flops": 4 * pages * HQ * D}
    if op == "attend":
        rows = sum(min(n, case["S"] * P) for n in lens) if case["S"] else sum(lens)
        return {"bytes": rows * HKV * (2 * (D * elt + rs) + (8 if case["mass"] else 0)) + 4 * B * HQ * D, "flops": 4 * rows * HQ * D}
    if op == "mass":
        T = case["T"]
        pairs = sum(T * (n - T) + T * (T + 1) // 2 for n in lens)
        return {"bytes": sum(lens) * HKV * (D * elt + rs + 4) + 2 * B * T * HQ * D, "flops": 2 * pairs * HQ * D}
    moved = sum(max(0, min(case["K"], n) - min(case["first"], n)) for n in lens if n > case["K"])
    return {"bytes": sum(lens) * HKV * 4 + moved * HKV * (4 * D * elt + 4) + 4 * B * HKV * case["K"], "flops": 0}


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    lens, n_pages = _lens(case), _pages(case)
    B, HQ, HKV, D, P = (case[k] for k in ("B", "HQ", "HKV", "D", "P"))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    total = sum(n_pages) + 3  # three pages belong to nobody
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    indptr = [0]
    for n in n_pages:
        indptr.append(indptr[-1] + n)
    st = dict(case=case, B=B, HQ=HQ, HKV=HKV, D=D, P=P, lens=lens, n_pages=n_pages, indptr=i32(indptr),
              indices=perm[:-3].contiguous(), spare=perm[-1:].contiguous(),
              last_page_len=i32([n - (p - 1) * P for n, p in zip(lens, n_pages)]), op=case["op"])
    rand = lambda *shape: torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=g)  # noqa: E731
    if case["op"] == "select":  # neighbouring keys resemble each other: every page has a centre and a width
        mid, wide = rand(total, HKV, D), rand(total, HKV, D).abs()
        st["page_bounds"] = torch.stack([mid - wide, mid + wide], 1).contiguous()
        st["keep_first"], st["keep_last"] = case["first"], case["last"]
    else:
        kv = case["kv"]
        cache = rand(total, 2, P, HKV, D)
        st["kv_scale"] = st["row_scale"] = None
        if kv == "e4m3":
            st["kv_scale"] = (torch.rand((2, HKV), generator=g, device=dev) * 0.01 + 0.008).float()
            cache = (cache / st["kv_scale"].reshape(1, 2, 1, HKV, 1).to(torch.bfloat16)).clamp(-448, 448).to(torch.float8_e4m3fn)
        elif kv == "e4m3c":
            cache = (cache * 8).clamp(-448, 448).to(torch.float8_e4m3fn)
        elif kv == "int8":
            st["row_scale"] = (cache.abs().amax(-1).float() / 127).to(torch.bfloat16).contiguous()
            cache = (cache / st["row_scale"].unsqueeze(-1)).round().clamp(-127, 127).to(torch.int8)
        st["cache"] = cache
    if case["op"] == "bounds":
        st["page_bounds"] = torch.zeros((total, 2, HKV, D), dtype=torch.bfloat16, device=dev)
        st["first_page"] = i32([p - 1 for p in n_pages]) if case["last_only"] else None
    if case["op"] in ("select", "attend"):
        st["q"] = rand(B, HQ, D) * 2
    if case["op"] == "attend" and case["S"]:  # distinct pages in order, the last page among them
        S, M = case["S"], max(n_pages)
        score = torch.rand((B, HKV, M), generator=g, device=dev)
        page = torch.arange(M, device=dev)
        n = torch.tensor(n_pages, device=dev).reshape(B, 1, 1)
        score = torch.where(page >= n, -1.0, torch.where(page == n - 1, 2.0, score))
        took = score.sort(dim=-1, descending=True, stable=True).indices[..., :S]
        took = torch.where(took < n, took, 1 << 30).sort(dim=-1).values
        took = torch.where(took < n, took, -1).to(torch.int32)
        st["pages"] = torch.nn.functional.pad(took, (0, S - took.shape[-1]), value=-1).contiguous()
    if case["op"] == "mass" or case.get("mass"):
        st["key_mass"] = torch.rand((total, P, HKV), generator=g, device=dev)
    if case["op"] == "mass":
        T = case["T"]
        st["q"] = rand(B * T, HQ, D) * 2
        st["qo_indptr"] = i32([T * b for b in range(B + 1)])
    if case["op"] == "evict":  # accumulated weights are heavy-tailed
        st["key_mass"] = torch.randn((total, P, HKV), generator=g, device=dev).mul_(2).exp_()
        st["keep_first"], st["keep_last"] = case["first"], case["last"]
    return st


# ------------------------------------------------------------------------------------------------- plain forms
def _table(st):
    """ctx [B, 1, 1] and a function (position [B, HKV, N]) -> flat (page, row, head) index of the position's row, a row of a
    page that belongs to nobody where the position is outside the sequence, and whether it is inside"""
    P, HKV = st["P"], st["HKV"]
    first = st["indptr"][:-1].long().reshape(-1, 1, 1)
    n = st["indptr"][1:].long().reshape(-1, 1, 1) - first
    ctx = torch.where(n > 0, (n - 1) * P + st["last_page_len"].long().reshape(-1, 1, 1), 0)
    head = torch.arange(HKV, device=ctx.device).reshape(1, -1, 1)

    def at(pos):
        ok = (pos >= 0) & (pos < ctx)
        page = st["indices"].long()[torch.where(ok, first + pos // P, 0)]
        page = torch.where(ok, page, st["spare"].long())
        row = torch.where(ok, pos % P, 0)
        return (page, row, head), ok

    return ctx, at


def _rows(st, where, kv):
    """values [B, HKV, N, D] fp32 of the cached K (kv 0) or V (kv 1) rows"""
    page, row, head = where
    D, P, HKV = st["D"], st["P"], st["HKV"]
    flat = ((page * 2 + kv) * P + row) * HKV + head
    cache = st["cache"]
    if cache.dtype == torch.bfloat16:
        return cache.view(-1, D)[flat].float()
    if st["row_scale"] is not None:
        got = cache.view(-1, D)[flat].float() * st["row_scale"].view(-1)[flat].float().unsqueeze(-1)
        return got.to(torch.bfloat16).float()
    got = cache.view(torch.uint8).view(-1, D)[flat].view(torch.float8_e4m3fn).float()
    return got * (0.125 if st["kv_scale"] is None else st["kv_scale"][kv].reshape(1, HKV, 1, 1))


def _plain_bounds(st):
    case, P, HKV, D = st["case"], st["P"], st["HKV"], st["D"]
    ctx, at = _table(st)
    M = max(st["n_pages"])
    if case["last_only"]:
        pos = ((st["first_page"].long().reshape(-1, 1) * P) + torch.arange(P, device=ctx.device)).unsqueeze(1)
    else:
        pos = torch.arange(M * P, device=ctx.device).reshape(1, 1, -1)
    pos = pos.expand(st["B"], HKV, -1)
    where, ok = at(pos)
    raw = dict(st, kv_scale=None)  # bounds of an E4M3 cache are those of the stored codes
    k = _rows(raw, where, 0) * (8.0 if st["cache"].dtype == torch.float8_e4m3fn else 1.0)
    k = k.reshape(st["B"], HKV, -1, P, D)
    ok = ok.reshape(st["B"], HKV, -1, P, 1)
    lo = torch.where(ok, k, torch.inf).amin(-2)
    hi = torch.where(ok, k, -torch.inf).amax(-2)
    page = where[0].reshape(st["B"], HKV, -1, P)[..., 0]
    some = ok[..., 0, 0].unsqueeze(-1)
    head = torch.arange(HKV, device=ctx.device).reshape(1, -1, 1).expand_as(page)
    out = st["page_bounds"]
    spare = out[st["spare"].long()].clone()
    out[page, 0, head] = torch.where(some, lo, 0.0).to(torch.bfloat16)
    out[page, 1, head] = torch.where(some, hi, 0.0).to(torch.bfloat16)
    out[st["spare"].long()] = spare
    return out


def _choose(score, n, first, last, S):
    """the S highest of score [.., M] fp64 among the first n, ties to the lowest index, the first and the last ones always,
    ascending, -1 behind"""
    i = torch.arange(score.shape[-1], device=score.device)
    score = torch.nan_to_num(score, nan=-torch.inf, posinf=1e308, neginf=-torch.inf)
    last = min(last, S)
    first = min(first, S - last)
    score = torch.where((i < first) | (i >= n - last), torch.inf, score)
    score = torch.where(i < n, score, -torch.inf)
    took = score.sort(dim=-1, descending=True, stable=True).indices[..., :S]
    took = torch.where(took < n, took, 1 << 40).sort(dim=-1).values
    took = torch.where(took < n, took, -1).to(torch.int32)
    return torch.nn.functional.pad(took, (0, S - took.shape[-1]), value=-1)


def _plain_select(st):
    B, HQ, HKV, D, case = st["B"], st["HQ"], st["HKV"], st["D"], st["case"]
    n = (st["indptr"][1:] - st["indptr"][:-1]).long().reshape(B, 1, 1)
    i = torch.arange(max(st["n_pages"]), device=n.device).reshape(1, 1, -1)
    page = st["indices"].long()[torch.where(i < n, st["indptr"][:-1].long().reshape(B, 1, 1) + i, 0)].squeeze(1)
    lo = st["page_bounds"][:, 0][page].double().permute(0, 2, 3, 1)  # [B, HKV, D, M]
    hi = st["page_bounds"][:, 1][page].double().permute(0, 2, 3, 1)
    q = st["q"].double().reshape(B, HKV, HQ // HKV, D)
    score = (q.clamp(min=0) @ hi + q.clamp(max=0) @ lo).amax(2)
    return _choose(score, n, case["first"], case["last"], case["S"])


def _plain_attend(st):
    B, HQ, HKV, D, P, case = st["B"], st["HQ"], st["HKV"], st["D"], st["P"], st["case"]
    ctx, at = _table(st)
    if case["S"]:
        pages = st["pages"].long().unsqueeze(-1)
        pos = torch.where(pages >= 0, pages * P + torch.arange(P, device=ctx.device), -1).reshape(B, HKV, -1)
    else:
        pos = torch.arange(max(st["lens"]), device=ctx.device).reshape(1, 1, -1).expand(B, HKV, -1)
    where, ok = at(pos)
    q = st["q"].float().reshape(B, HKV, HQ // HKV, D)
    s = (q @ _rows(st, where, 0).transpose(-1, -2)) * D ** -0.5
    s = torch.where(ok.unsqueeze(2), s, -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, 0.0)
    v = torch.where(ok.unsqueeze(-1), _rows(st, where, 1), 0.0)
    out = (p @ v).reshape(B, HQ, D).to(torch.bfloat16)
    if not case["mass"]:
        return out
    page, row, head = where
    st["key_mass"].view(-1).index_add_(0, ((page * P + row) * HKV + head).reshape(-1), p.sum(2).reshape(-1))
    return out, st["key_mass"]


def _plain_mass(st):
    B, HQ, HKV, D, P, T = st["B"], st["HQ"], st["HKV"], st["D"], st["P"], st["case"]["T"]
    ctx, at = _table(st)
    N = max(st["lens"])
    pos = torch.arange(N, device=ctx.device).reshape(1, 1, -1).expand(B, HKV, -1)
    where, ok = at(pos)
    q = st["q"].float().reshape(B, T, HKV, HQ // HKV, D).permute(0, 2, 3, 1, 4).reshape(B, HKV, -1, D)
    s = (q @ _rows(st, where, 0).transpose(-1, -2)) * D ** -0.5
    s = s.reshape(B, HKV, HQ // HKV, T, N)
    mine = ctx.reshape(B, 1, 1, 1, 1) - T + torch.arange(T, device=ctx.device).reshape(1, 1, 1, T, 1)  # the queries' positions
    s = s.masked_fill_(pos.reshape(B, HKV, 1, 1, N) > mine, -torch.inf)
    s = torch.exp_(s.sub_(s.amax(-1, keepdim=True)))
    w = (s / s.sum(-1, keepdim=True)).sum((2, 3))
    page, row, head = where
    old = st["key_mass"]
    flat = ((page * P + row) * HKV + head).reshape(-1)
    new = torch.zeros_like(old).view(-1).index_add_(0, flat, torch.where(ok, w, 0.0).reshape(-1))
    hit = torch.zeros_like(old).view(-1).index_add_(0, flat, ok.float().reshape(-1))
    return old.copy_(torch.where(hit.view_as(old) > 0, new.view_as(old), old))


def _plain_evict(st):
    B, HKV, D, P, case, K = st["B"], st["HKV"], st["D"], st["P"], st["case"], st["case"]["K"]
    ctx, at = _table(st)
    pos = torch.arange(max(st["lens"]), device=ctx.device).reshape(1, 1, -1).expand(B, HKV, -1)
    (page, row, head), ok = at(pos)
    mass = st["key_mass"].view(-1)
    kept = _choose(mass[(page * P + row) * HKV + head].double(), ctx, case["first"], case["last"], K)
    src, ok = at(kept.long())
    j = torch.arange(K, device=ctx.device).reshape(1, 1, -1).expand(B, HKV, -1)
    dst, _ = at(torch.where(ok, j, -1))
    cache = st["cache"].view(torch.uint8).view(-1, D * st["cache"].element_size())
    flat = lambda w, kv: ((w[0] * 2 + kv) * P + w[1]) * HKV + w[2]  # noqa: E731
    k, v = cache[flat(src, 0)], cache[flat(src, 1)]
    m = mass[(src[0] * P + src[1]) * HKV + src[2]]
    cache[flat(dst, 0)] = k
    cache[flat(dst, 1)] = v
    mass[(dst[0] * P + dst[1]) * HKV + dst[2]] = m
    return kept, st["cache"], st["key_mass"]


def run(st):
    op, case = st["op"], st["case"]
    if not own:
        return {"bounds": _plain_bounds, "select": _plain_select, "attend": _plain_attend, "mass": _plain_mass, "evict": _plain_evict}[op](st)
    import ax_dsl_kernels_b200 as q35
    table = (st["indptr"], st["indices"], st["last_page_len"])
    if op == "bounds":
        return q35.page_key_bounds(st["cache"], *table, st["page_bounds"], first_page=st["first_page"], paged_kv_scale=st["row_scale"])
    if op == "select":
        return q35.select_pages(st["q"], st["page_bounds"], *table, case["S"], keep_first=st["keep_first"], keep_last=st["keep_last"])
    scales = dict(kv_scale=st["kv_scale"], paged_kv_scale=st["row_scale"])
    if op == "attend":
        out = q35.paged_attention_sparse(st["q"], st["cache"], *table, st.get("pages"), key_mass=st.get("key_mass"), **scales)
        return (out, st["key_mass"]) if case["mass"] else out
    if op == "mass":
        return q35.paged_key_mass(st["q"], st["cache"], st["qo_indptr"], *table, st["key_mass"], **scales)
    kept = q35.evict_keys(st["cache"], st["key_mass"], *table, case["K"], keep_first=st["keep_first"], keep_last=st["keep_last"])
    return kept, st["cache"], st["key_mass"]


# ------------------------------------------------------------------- the definitions in 64 bits, sequence by sequence
def _value(st, b, kv):
    """[rows, HKV, D] fp64 of sequence b, its pages, and the (page, row) of every position"""
    n, lo = st["lens"][b], int(sum(st["n_pages"][:b]))
    pages = st["indices"][lo:lo + st["n_pages"][b]].long()
    got = st["cache"][pages, kv] if st["cache"].dtype != torch.float8_e4m3fn else \
        st["cache"].view(torch.uint8)[pages, kv].view(torch.float8_e4m3fn)
    x = got.to(torch.float64)
    if st["row_scale"] is not None:
        x = (x * st["row_scale"][pages, kv].double().unsqueeze(-1)).to(torch.bfloat16).double()
    elif st["cache"].dtype == torch.float8_e4m3fn:
        x = x / 8 if st["kv_scale"] is None else x * st["kv_scale"][kv].double().reshape(1, 1, -1, 1)
    return x.reshape(-1, st["HKV"], st["D"])[:n], pages


def _best(score, n, first, last, S):
    """Python's own sort: (forced, score, lowest index)"""
    last = min(last, S)
    first = min(first, S - last)
    rank = sorted(range(n), key=lambda i: (0 if i < first or i >= n - last else 1, -score[i], i))
    return sorted(rank[:S]) + [-1] * (S - min(S, n))


def exact(case, seed):
    st = prepare(case, seed)
    B, HQ, HKV, D, P, op = st["B"], st["HQ"], st["HKV"], st["D"], st["P"], st["op"]
    G = HQ // HKV
    if op == "bounds":
        out = st["page_bounds"].double()
        for b in range(B):
            raw = dict(st, kv_scale=torch.ones((2, HKV), device="cuda"))
            k, pages = _value(raw, b, 0)
            for i in range(st["n_pages"][b] - 1 if case["last_only"] else 0, st["n_pages"][b]):
                rows = k[i * P:(i + 1) * P]
                out[pages[i], 0], out[pages[i], 1] = rows.min(0).values, rows.max(0).values
        return out
    if op == "select":
        got = []
        for b in range(B):
            lo = int(sum(st["n_pages"][:b]))
            bound = st["page_bounds"][st["indices"][lo:lo + st["n_pages"][b]].long()].double()
            for h in range(HKV):
                q = st["q"][b, h * G:(h + 1) * G].double()
                best = None
                for g in range(G):
                    s = torch.maximum(q[g] * bound[:, 0, h], q[g] * bound[:, 1, h]).sum(-1)
                    best = s if best is None else torch.maximum(best, s)
                got.append(_best(best.tolist(), st["n_pages"][b], case["first"], case["last"], case["S"]))
        return torch.tensor(got, dtype=torch.int32).reshape(B, HKV, -1)
    if op in ("attend", "mass"):
        mass = st["key_mass"].double() if "key_mass" in st else None
        out = torch.zeros((B, HQ, D), dtype=torch.float64, device="cuda")
        for b in range(B):
            k, pages = _value(st, b, 0)
            v = _value(st, b, 1)[0] if op == "attend" else None
            pos = torch.arange(st["lens"][b], device="cuda")
            for h in range(HKV):
                if op == "attend":
                    use = pos
                    if case["S"]:
                        took = torch.zeros(st["n_pages"][b] + 1, dtype=torch.bool, device="cuda")
                        took[st["pages"][b, h].long()] = True
                        use = pos[took[:-1][pos // P]]
                    p = torch.softmax(st["q"][b, h * G:(h + 1) * G].double() @ k[use, h].T / math.sqrt(D), -1)
                    out[b, h * G:(h + 1) * G] = p @ v[use, h]
                    if mass is not None:
                        mass[pages[use // P], use % P, h] += p.sum(0)
                    continue
                T = case["T"]
                total = torch.zeros_like(pos, dtype=torch.float64)
                later = pos > (st["lens"][b] - T + torch.arange(T, device="cuda")).reshape(-1, 1)
                for g in range(G):
                    s = st["q"][b * T:(b + 1) * T, h * G + g].double() @ k[:, h].T / math.sqrt(D)
                    total += torch.softmax(s.masked_fill(later, -math.inf), -1).sum(0)
                mass[pages[pos // P], pos % P, h] = total
        return mass if op == "mass" else (out, mass) if mass is not None else out
    kept = []
    cache, mass = st["cache"].clone(), st["key_mass"].clone()
    for b in range(B):
        lo = int(sum(st["n_pages"][:b]))
        pages = st["indices"][lo:lo + st["n_pages"][b]].long()
        for h in range(HKV):
            own_mass = st["key_mass"][pages, :, h].reshape(-1)[:st["lens"][b]].tolist()
            best = _best(own_mass, st["lens"][b], case["first"], case["last"], case["K"])
            kept.append(best)
            src = torch.tensor([i for i in best if i >= 0], device="cuda")
            dst = torch.arange(len(src), device="cuda")
            for old, new in ((st["cache"].view(torch.uint8), cache.view(torch.uint8)),):
                new[pages[dst // P], :, dst % P, h] = old[pages[src // P], :, src % P, h]
            mass[pages[dst // P], dst % P, h] = st["key_mass"][pages[src // P], src % P, h]
    return torch.tensor(kept, dtype=torch.int32).reshape(B, HKV, -1), cache.double() if cache.dtype == torch.bfloat16 else cache.to(torch.float64), mass.double()
