"""Host side of the long-context operators: attending to, and keeping, less than the whole paged cache.

    page_key_bounds         per page and channel, the minimum and maximum of its keys (made as the cache is written)
    select_pages            the pages whose keys can score highest with a query
    paged_attention_sparse  decode attention over those pages (or all), optionally adding up the weight every row gets
    paged_key_mass          the weight a window of queries (a prompt's last tokens) gives to every cached row
    evict_keys              keeps the rows that got most and moves them together, in place

All of them take the page table of paged_attention_decode: indptr [B + 1], indices, last_page_len [B] int32; sequence b
has (pages - 1) * P + last_page_len[b] cached rows.  Rows and pages behind a sequence's end are neither read nor written.
Pages that hold another sequence's rows too (a shared prefix) can be read by all of them.  Weights that are added to
key_mass (paged_attention_sparse, paged_key_mass with accumulate) then add up over all their queries, in no fixed order;
stored ones are those of one of the sequences; eviction, which moves rows, wants pages of its own.
The reference has no counterpart of these operators; they extend its page-table form of decode attention
(models/qwen35_35b_a3b/sgl/python/sgl_kernel_axera/attention/flash_attn.py:2549-2665)."""
import torch

from . import _lib

_keep = {}


def _keep_pair(first, last, device):
    """int32 [2] tensor (first, last) on `device`, made once per pair of values; a pair first used inside a graph capture,
    where nothing can be copied from the host, is set by the graph itself"""
    if first < 0 or last < 0:
        raise ValueError("keep_first and keep_last count pages or rows: not negative")
    key = (int(first), int(last), device.index)
    t = _keep.get(key)
    if t is not None:
        return t
    with torch.cuda.device(device.index if device.type == "cuda" else -1):  # the device whose stream the call goes to
        if torch.cuda.is_current_stream_capturing():
            t = torch.full((2,), int(first), dtype=torch.int32, device=device)
            t[1:].fill_(int(last))
        else:
            t = _keep[key] = torch.tensor([int(first), int(last)], dtype=torch.int32, device=device)
    return t


def _scale(kw, sm_scale, device):
    if sm_scale is not None:
        kw["sm_scale"] = sm_scale if isinstance(sm_scale, torch.Tensor) else torch.full(
            (1,), float(sm_scale), dtype=torch.float32, device=device)


def page_key_bounds(paged_kv_cache, indptr, indices, last_page_len, out=None, *, first_page=None, paged_kv_scale=None):
    """Bounds of every listed page's keys: out [pages, 2, HKV, D] bf16, out[page, 0] the minimum and out[page, 1] the
    maximum of the page's valid K rows per head and channel.  Exact in the stored format; an E4M3 cache gives the bounds
    of its stored codes (a head's scale does not change the order of its pages), an int8 cache those of
    bf16(int8 * scale).  first_page [B] int32: only the pages of sequence b from that one on -- after a decode step its
    last page, after a chunk of tokens the page it began in.  Pages not listed stay as they were in `out`."""
    if out is None:
        pages, _, _, HKV, D = paged_kv_cache.shape
        out = torch.zeros((pages, 2, HKV, D), dtype=torch.bfloat16, device=paged_kv_cache.device)
    kw = dict(paged_kv_cache=paged_kv_cache, indptr=indptr, indices=indices, last_page_len=last_page_len, page_bounds=out)
    if first_page is not None:
        kw["first_page"] = first_page
    if paged_kv_scale is not None:
        kw["paged_kv_scale"] = paged_kv_scale
    _lib.run("attn.page_bounds", **kw)
    return out


def select_pages(q, page_bounds, indptr, indices, last_page_len, n_select, out=None, *, keep_first=0, keep_last=1):
    """The n_select pages of every (sequence, KV head) to attend to: [B, HKV, n_select] int32 positions in the
    sequence's page list (not page ids), ascending, -1 behind when it has fewer.  A page scores
    max over the KV head's query heads of sum_d max(q_d * min_d, q_d * max_d), the most any of its keys can score;
    pages are ordered by these sums in fp64, ties go to the lower position, a NaN ranks last.  The keep_first first and the
    keep_last last pages are chosen whatever they score (keep_last before keep_first when they do not all fit).  q [B, HQ, D] bf16."""
    if out is None:
        out = torch.empty((q.shape[0], page_bounds.shape[2], int(n_select)), dtype=torch.int32, device=q.device)
    elif out.shape[-1] != n_select:
        raise ValueError("select_pages: out must be [B, HKV, n_select]")
    kw = dict(q=q, page_bounds=page_bounds, indptr=indptr, indices=indices, last_page_len=last_page_len, pages=out)
    if keep_first or keep_last:
        kw["keep"] = _keep_pair(keep_first, keep_last, q.device)
    _lib.run("attn.select_pages", **kw)
    return out


def paged_attention_sparse(q, paged_kv_cache, indptr, indices, last_page_len, pages=None, out=None, *, key_mass=None,
                           sm_scale=None, kv_scale=None, k_new=None, v_new=None, cache_location=None,
                           paged_kv_scale=None):
    """paged_attention_decode over the chosen pages of every (sequence, KV head): pages [B, HKV, S] int32 as select_pages
    gives them (None: all pages).  key_mass [pages, P, HKV] fp32, when given, gets the softmax weight of every attended
    row added, summed over the query heads of the row's KV head.  k_new / v_new [B, HKV, D]: the current token, attended
    to from its own rows whatever the pages; with key_mass, cache_location [B, 2] says where its own weight is stored
    (stored, not added: the row is new; the table does not hold it yet).  Without them, a row that is new in the table
    starts from whatever its place in key_mass held -- after an eviction or in a page used again, another row's weight --
    and the caller clears it first.  Unlike paged_attention_decode nothing is written into the cache.
    A row without any page and without a current token gives zeros; a NaN or an infinity in an attended row of V gives NaN.
    At most 8 query heads per KV head, head_dim 64, 128
    or 256, page size a multiple of 16.  Formats and scales as in paged_attention_decode."""
    out = torch.empty_like(q) if out is None else out
    kw = dict(q=q, paged_kv_cache=paged_kv_cache, indptr=indptr, indices=indices, last_page_len=last_page_len, out=out)
    if pages is not None:
        kw["pages"] = pages
    if key_mass is not None:
        kw["key_mass"] = key_mass
        if cache_location is not None and k_new is not None:
            kw["cache_location"] = cache_location
    if kv_scale is not None:
        kw["kv_scale"] = kv_scale
    if paged_kv_scale is not None:
        kw["paged_kv_scale"] = paged_kv_scale
    if k_new is not None:
        kw["k_new"], kw["v_new"] = k_new, v_new
    _scale(kw, sm_scale, q.device)
    _lib.run("attn.sparse_decode", **kw)
    return out


def paged_key_mass(q, paged_kv_cache, qo_indptr, indptr, indices, last_page_len, key_mass, *, accumulate=False,
                   sm_scale=None, kv_scale=None, paged_kv_scale=None):
    """The softmax weight that a window of queries gives to every cached row: q [T_total, HQ, D] bf16 holds the last
    qo_indptr[b + 1] - qo_indptr[b] tokens of every sequence, whose K rows are in the cache already (the page table
    includes them, as in paged_attention_prefill); each sees the rows up to its own.  key_mass [pages, P, HKV] fp32: the
    sum over the window's queries and over the query heads of the KV head, stored for every row of every sequence
    (accumulate: added; the form for pages that several sequences list).  Up to 128 query heads per KV head, any page size;
    head_dim 64, 128 or 256."""
    kw = dict(q=q, paged_kv_cache=paged_kv_cache, qo_indptr=qo_indptr, indptr=indptr, indices=indices,
              last_page_len=last_page_len, key_mass=key_mass)
    if accumulate:
        kw["accumulate"] = _keep_pair(1, 1, q.device)
    if kv_scale is not None:
        kw["kv_scale"] = kv_scale
    if paged_kv_scale is not None:
        kw["paged_kv_scale"] = paged_kv_scale
    _scale(kw, sm_scale, q.device)
    _lib.run("attn.key_mass", **kw)
    return key_mass


def evict_keys(paged_kv_cache, key_mass, indptr, indices, last_page_len, n_keep, kept=None, *, keep_first=0, keep_last=0,
               paged_kv_scale=None):
    """Keeps min(n_keep, rows) rows of every (sequence, KV head) and moves them, in order, to the sequence's first
    positions, in place, together with their key_mass (and int8 row scales).  Kept are the keep_first first and the
    keep_last last rows (keep_last before keep_first when they do not all fit) and, of the rest, those with the highest
    key_mass; ties go to the lower position, a NaN ranks last.  Returns kept [B, HKV, n_keep] int32: the old position of
    every new row, -1 behind.  Afterwards a sequence has min(n_keep, rows) rows -- the caller shortens its page table --
    and what lies behind them is left as it was.  Keys keep the rotation of their old positions, so later tokens go on
    counting positions as if nothing had been evicted; bounds of pages have to be made again."""
    if kept is None:
        kept = torch.empty((indptr.numel() - 1, paged_kv_cache.shape[3], int(n_keep)), dtype=torch.int32,
                           device=paged_kv_cache.device)
    elif kept.shape[-1] != n_keep:
        raise ValueError("evict_keys: kept must be [B, HKV, n_keep]")
    kw = dict(paged_kv_cache=paged_kv_cache, key_mass=key_mass, indptr=indptr, indices=indices,
              last_page_len=last_page_len, kept=kept)
    if keep_first or keep_last:
        kw["keep"] = _keep_pair(keep_first, keep_last, kept.device)
    if paged_kv_scale is not None:
        kw["paged_kv_scale"] = paged_kv_scale
    _lib.run("attn.evict", **kw)
    return kept
