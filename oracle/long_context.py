"""The long-context operators in 64 bits, one sequence and KV head at a time (CPU oracle; test infrastructure only).

Written from the definitions: bounds of a page's keys, choice of pages by them, attention over chosen rows with the
weight every row gets, the weight a window of queries gives, eviction by weight.  The reference has no counterpart."""
import math

import torch

from .attention import gather_kv, valid_kv_len


def _rows(cache, indptr, indices, last_page_len, b, kv_scale=None, row_scale=None):
    k, v = gather_kv(cache, indptr, indices, last_page_len, b, kv_scale, row_scale)
    return k.double(), v.double()


def _places(indptr, indices, last_page_len, P, b):
    """(page id, row in page) of every position of sequence b"""
    n = int(valid_kv_len(indptr, last_page_len, P)[b])
    pos = torch.arange(n)
    return indices[int(indptr[b]) + pos // P].long(), pos % P


def page_bounds(cache, indptr, indices, last_page_len, out, first_page=None, row_scale=None):
    out = out.clone()
    P = cache.shape[2]
    for b in range(len(indptr) - 1):
        k, _ = _rows(cache, indptr, indices, last_page_len, b, None, row_scale)
        if cache.dtype == torch.float8_e4m3fn:  # the stored codes' values (gather_kv takes out the constant 1 / 8)
            k = k * 8
        for i in range(0 if first_page is None else max(0, int(first_page[b])), -(-k.shape[0] // P)):
            rows = k[i * P:(i + 1) * P]
            page = int(indices[int(indptr[b]) + i])
            out[page, 0] = rows.amin(0).to(torch.bfloat16)
            out[page, 1] = rows.amax(0).to(torch.bfloat16)
    return out


def best(score, n_keep, first, last):
    """positions of the n_keep highest of a list, the first and last ones always (the last before the first when they do
    not all fit), ties to the lower position, NaN lowest; ascending"""
    n = len(score)
    last = min(last, n_keep)
    first = min(first, n_keep - last)
    rank = sorted(range(n), key=lambda i: (0 if i < first or i >= n - last else 1,
                                           math.inf if math.isnan(score[i]) else -score[i], i))
    return sorted(rank[:n_keep])


def page_scores(q, bounds, indptr, indices, last_page_len, b, h):
    """fp64 scores of the pages of (sequence b, KV head h)"""
    HKV = bounds.shape[2]
    G = q.shape[1] // HKV
    n = int(indptr[b + 1]) - int(indptr[b])
    n -= int(n > 0 and last_page_len[b] == 0)
    page = indices[int(indptr[b]):int(indptr[b]) + n].long()
    lo, hi = bounds[page, 0, h].double(), bounds[page, 1, h].double()
    out = []
    for g in range(G):
        qg = q[b, h * G + g].double()
        out.append(torch.maximum(qg * lo, qg * hi).sum(-1))
    return torch.stack(out).amax(0)


def select_pages(q, bounds, indptr, indices, last_page_len, S, first=0, last=0):
    B, HKV = q.shape[0], bounds.shape[2]
    out = torch.full((B, HKV, S), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(HKV):
            got = best(page_scores(q, bounds, indptr, indices, last_page_len, b, h).tolist(), S, first, last)
            out[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
    return out


def _weights(s):
    """softmax along the last dim in 64 bits; a row that is all -inf has no weights"""
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.zeros((*s.shape[:-1], 1), dtype=s.dtype)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.where(total == 0, torch.zeros_like(p), p / total)


def sparse_decode(q, cache, indptr, indices, last_page_len, pages=None, key_mass=None, sm_scale=None, kv_scale=None,
                  row_scale=None, k_new=None, v_new=None, cache_location=None):
    """out [B, HQ, D] fp64, key_mass fp64, and for the tolerance of an fp32 evaluation sum_i p_i |v_i| and the largest
    sum_d |q_d k_id| * scale of every query head"""
    B, HQ, D = q.shape
    P, HKV = cache.shape[2], cache.shape[3]
    G = HQ // HKV
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    out = torch.zeros((B, HQ, D), dtype=torch.float64)
    size, reach = torch.zeros_like(out), torch.zeros((B, HQ, 1), dtype=torch.float64)
    mass = None if key_mass is None else key_mass.double().clone()
    for b in range(B):
        k_all, v_all = _rows(cache, indptr, indices, last_page_len, b, kv_scale, row_scale)
        page, row = _places(indptr, indices, last_page_len, P, b)
        for h in range(HKV):
            use = torch.arange(k_all.shape[0])
            if pages is not None:
                chosen = {int(p) for p in pages[b, h] if p >= 0}
                use = use[torch.tensor([int(i) // P in chosen for i in use], dtype=torch.bool)]
            k, v = k_all[use, h], v_all[use, h]
            if k_new is not None:
                k = torch.cat([k, k_new[b, h].double()[None]], 0)
                v = torch.cat([v, v_new[b, h].double()[None]], 0)
            if k.shape[0] == 0:
                continue
            qg = q[b, h * G:(h + 1) * G].double()
            p = _weights(qg @ k.T * scale)
            out[b, h * G:(h + 1) * G] = p @ v
            size[b, h * G:(h + 1) * G] = p @ v.abs()
            reach[b, h * G:(h + 1) * G] = (qg.abs() @ k.abs().T * scale).amax(-1, keepdim=True)
            if mass is not None:
                mass[page[use], row[use], h] += p[:, :len(use)].sum(0)
                if k_new is not None:
                    mass[int(cache_location[b, 0]), int(cache_location[b, 1]), h] = p[:, -1].sum()
    return out, mass, size, reach


def key_mass(q, cache, qo_indptr, indptr, indices, last_page_len, mass, accumulate=False, sm_scale=None, kv_scale=None,
             row_scale=None):
    """mass fp64 and the largest sum_d |q_d k_id| * scale of the call"""
    HQ, D = q.shape[1:]
    P, HKV = cache.shape[2], cache.shape[3]
    G = HQ // HKV
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    mass = mass.double().clone()
    reach = 0.0
    for b in range(len(indptr) - 1):
        k, _ = _rows(cache, indptr, indices, last_page_len, b, kv_scale, row_scale)
        page, row = _places(indptr, indices, last_page_len, P, b)
        n, q0, T = k.shape[0], int(qo_indptr[b]), int(qo_indptr[b + 1]) - int(qo_indptr[b])
        later = torch.arange(n)[None] > (n - T + torch.arange(T))[:, None]
        for h in range(HKV):
            total = torch.zeros(n, dtype=torch.float64)
            for g in range(G):
                qg = q[q0:q0 + T, h * G + g].double()
                total += _weights((qg @ k[:, h].T * scale).masked_fill(later, -math.inf)).sum(0)
                if T and n:
                    r = (qg.abs() @ k[:, h].abs().T * scale).masked_fill(later, 0.0)
                    reach = max(reach, float(r[r.isfinite()].max()))
            mass[page, row, h] = mass[page, row, h] + total if accumulate else total
    return mass, reach


def evict(cache, mass, indptr, indices, last_page_len, K, first=0, last=0, row_scale=None):
    """kept, and copies of cache, mass and row scales after the moves"""
    B, (P, HKV) = len(indptr) - 1, cache.shape[2:4]
    kept = torch.full((B, HKV, K), -1, dtype=torch.int32)
    raw = cache.view(torch.uint8)
    new, new_mass = raw.clone(), mass.clone()
    new_rs = None if row_scale is None else row_scale.clone()
    for b in range(B):
        page, row = _places(indptr, indices, last_page_len, P, b)
        for h in range(HKV):
            got = best(mass[page, row, h].tolist(), K, first, last) if len(page) > K else list(range(len(page)))
            kept[b, h, :len(got)] = torch.tensor(got, dtype=torch.int32)
            s = torch.tensor(got, dtype=torch.long)
            d = torch.arange(len(got))
            new[page[d], :, row[d], h] = raw[page[s], :, row[s], h]
            new_mass[page[d], row[d], h] = mass[page[s], row[s], h]
            if row_scale is not None:
                new_rs[page[d], :, row[d], h] = row_scale[page[s], :, row[s], h]
    return kept, new.view(cache.dtype), new_mass, new_rs
