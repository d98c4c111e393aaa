"""How exactly attn.sparse_decode carries its weights and sums, seen through outputs in which the large terms cancel: the
output's own rounding to bf16 is then far below what a weight of too few bits, or a sum that loses on every addition, costs.

Inputs are exact in every cache format, and a score is one product, so that fp32 holds it exactly."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from oracle import long_context as olc  # noqa: E402
from test_gpu_long_context import gpu, gpu_scales  # noqa: E402

FMT = ["bf16", "e4m3", "e4m3c", "int8"]
UNIT = 1 / 64  # int8: every row's scale


def stored(x, fmt):
    """values -> the nearest ones the format holds (fp64) and their stored form"""
    if fmt == "bf16":
        s = x.to(torch.bfloat16)
        return s.double(), s
    if fmt == "int8":
        s = (x / UNIT).round().clamp(-127, 127)
        return s * UNIT, s.to(torch.int8)
    s = (x * 8).float().clamp(-448, 448).to(torch.float8_e4m3fn)
    return s.double() / 8, s


def cache_of(k, v, P, fmt):
    """one page per sequence of k, v [B, n, HKV, D] (fp64, exact in the format): cache, table, scales"""
    B, n, HKV, D = k.shape
    pages = -(-n // P)
    kv = torch.zeros((B, pages * P, 2, HKV, D), dtype=torch.float64)
    kv[:, :n, 0], kv[:, :n, 1] = k, v
    values, s = stored(kv, fmt)
    assert torch.equal(values, kv)
    cache = s.view(torch.uint8) if fmt.startswith("e4m3") else s
    cache = cache.reshape(B * pages, P, 2, HKV, D).transpose(1, 2).contiguous()
    cache = cache.view(torch.float8_e4m3fn) if fmt.startswith("e4m3") else cache
    table = (torch.arange(B + 1, dtype=torch.int32) * pages, torch.arange(B * pages, dtype=torch.int32),
             torch.full((B,), n - (pages - 1) * P, dtype=torch.int32))
    scales = {}
    if fmt == "e4m3":
        scales["kv_scale"] = torch.full((2, HKV), 0.125)
    if fmt == "int8":
        scales["row_scale"] = torch.full((B * pages, 2, P, HKV), UNIT, dtype=torch.bfloat16)
    return cache, table, scales


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_weights_meet_v_with_all_their_bits(fmt, D):
    """Row 1 has weight exp(-x), 1 / 2 to 1; row 0, of weight 1, and rows of weights 2^-4, 2^-8, ... take its term away as
    far as their values allow.  What is left of the largest term, about 2^-20 of it, is the output.

    Tolerance: the output's rounding; exp2 2^-22 and the score's scaling and subtraction 3 x 2^-24 of numbers up to 2^4 log2 e
    for rows whose share is 2^-4 of the sum at most, of numbers up to 1 for the others; the weight's own bits 2^-22; three
    truncated additions of a step and the merges' roundings, 2^-21: 2^-20 of sum p |v| in all."""
    import ax_dsl_kernels_b200 as q35
    B, HKV, n, P, step = 12, 2, 8, 16, 2.75
    g = torch.Generator().manual_seed(41)
    x = torch.linspace(0.03, 0.67, B * HKV).to(torch.bfloat16).double().reshape(B, HKV)
    q = torch.zeros((B, HKV, D), dtype=torch.float64)
    q[..., 0], q[..., 1] = -x, -step
    k, v = torch.zeros((B, n, HKV, D), dtype=torch.float64), torch.zeros((B, n, HKV, D), dtype=torch.float64)
    k[:, 1, :, 0] = 1.0
    for j in range(2, n):
        k[:, j, :, 1] = (j - 1) / 4 if fmt == "int8" else j - 1
    if fmt == "int8":
        q[..., 1] *= 4
    weight = torch.exp(torch.einsum("bhd,bnhd->bnh", q, k))
    v[:, 1] = stored(torch.rand((B, HKV, D), generator=g, dtype=torch.float64) * 0.7 + 0.7, fmt)[0]
    left = weight[:, 1, :, None] * v[:, 1]
    for j in (0, *range(2, n)):
        w = weight[:, j, :, None]
        v[:, j] = stored(-left / w, fmt)[0]
        left = left + w * v[:, j]
    cache, table, scales = cache_of(k, v, P, fmt)
    qb = q.to(torch.bfloat16)
    assert torch.equal(qb.double(), q)
    ref, _, size, _ = olc.sparse_decode(qb, cache, *table, sm_scale=1.0, **scales)
    assert (ref.abs() / size).median() < 2.0 ** -15
    got = q35.paged_attention_sparse(gpu(qb), gpu(cache), *gpu(table), sm_scale=1.0, **gpu_scales(scales)).double().cpu()
    tol = ref.abs() * 2.0 ** -8 + size * 2.0 ** -20
    assert ((got - ref).abs() <= tol).all(), f"worst {((got - ref).abs() / tol).max():.3g} of the tolerance"
    assert q35.device_status() == 0


@pytest.mark.parametrize("fmt", FMT[:2] + FMT[3:])
def test_long_sums_lose_nothing_on_the_way(fmt):
    """16384 rows whose second half takes the first half's terms away again, at one CTA per (sequence, KV head): the output
    is 0, and what comes out instead is what the sums lost while they rose and fell.

    Tolerance: a warp adds up 128 steps, rounded to nearest, 2^-24 of running sums that are half their peak on average, and
    the peaks are half of sum p |v|: 2^-19 of it; within a step six products, each cut off at 2^-23 of the step's own sum,
    2^-20.  A rounding to nearest goes either way: the mean over 512 channels has to be 1 / 8 of that (the mean of 512
    errors of one bound has a 75th of it as its deviation); one that always goes towards zero shows there."""
    import ax_dsl_kernels_b200 as q35
    HKV, D, P, n, B = 2, 256, 64, 16384, 80
    g = torch.Generator().manual_seed(43)
    k, v = torch.zeros((1, n, HKV, D), dtype=torch.float64), torch.zeros((1, n, HKV, D), dtype=torch.float64)
    k[0, :n // 2, :, 0] = -torch.randint(0, 12, (n // 2, HKV), generator=g).double() / 8
    k[0, ::32, :, 0] = 0.0  # the largest score is in every step: no rescaling
    v[0, :n // 2] = stored(1 + torch.rand((n // 2, HKV, D), generator=g, dtype=torch.float64) * 0.9, fmt)[0]
    k[0, n // 2:], v[0, n // 2:] = k[0, :n // 2], -v[0, :n // 2]
    cache, (indptr, indices, last), scales = cache_of(k, v, P, fmt)
    q = torch.zeros((1, HKV, D), dtype=torch.bfloat16)
    q[..., 0] = 1.0
    ref, _, size, _ = olc.sparse_decode(q, cache, indptr, indices, last, sm_scale=1.0, **scales)
    assert (ref.abs() < 1e-12).all()
    table = (torch.arange(B + 1, dtype=torch.int32) * (n // P), indices.repeat(B), last.repeat(B))  # all read the same pages
    pages = torch.arange(n // P, dtype=torch.int32).expand(B, HKV, -1).contiguous()
    got = q35.paged_attention_sparse(gpu(q.expand(B, -1, -1).contiguous()), gpu(cache), *gpu(table), gpu(pages), sm_scale=1.0,
                                     **gpu_scales(scales)).double().cpu()
    tol = size * (2.0 ** -19 + 2.0 ** -20)
    assert torch.equal(got, got[:1].expand_as(got))
    assert (got[:1].abs() <= tol).all(), f"worst {(got[:1].abs() / tol).max():.3g} of the tolerance"
    assert (got[0] / tol[0]).mean().abs() <= 1 / 8, f"mean {(got[0] / tol[0]).mean():.3g} of the tolerance"
    assert q35.device_status() == 0
