"""A serving step over the paged cache: ``extend_block_table``,
``paged_append``, ``update_page_means``, ``select_pages`` and
``scaled_dot_product_attention_paged_sparse`` against float64, and all of
them in a row.

Tables, slots, means and selected pages are compared exactly (means: the
64-bit sum rounded through fp32 to the cache's type, on both sides).

Sparse attention's tolerance, with u half a step of the operand type, A the
attention of |v| and n the number of keys: every weight is rounded to the type
before the second product (u A; fp16 weights below 2^-14 of their row's
maximum to within 2^-25, n 2^-25 max |v|), the result once more (u |o|).
Scores are fp32 sums of exact products: up to D 2^-23 of their terms' sum, some
10, so 2e-4 in a weight at worst, twice (2 x 1e-4 A allows for the ratio).
"""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import triton_flash_attention_b200 as fa
from oracle import fa2_oracle as orc
from triton_flash_attention_b200 import _abi

F16, BF16 = torch.float16, torch.bfloat16


def _i32(a):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32)


def _f64(t):
    return t.detach().double().cpu().numpy()


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def _rounded_mean(ref, dtype):
    return torch.from_numpy(ref).float().to(dtype)


class Case:
    """Sequences of ``lens_k`` keys, the last ``lens_q`` of them new, in a
    shuffled cache; every row no sequence has a key in holds ``junk``."""

    def __init__(self, lens_q, lens_k, page, hq, hkv, d, dtype, seed, junk=float("nan"), pad=0, spare=3, width=None):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.page, self.hq, self.hkv, self.d, self.dtype = page, hq, hkv, d, dtype
        pages = [-(-n // page) for n in lens_k]
        n_pages = sum(pages) + spare
        perm = rng.permutation(n_pages)
        self.table = np.full((len(lens_k), width or max(max(pages), 1)), -1, np.int32)
        at = 0
        for b, p in enumerate(pages):
            self.table[b, :p] = perm[at:at + p]
            at += p
        self.cu = np.concatenate([[0], np.cumsum(lens_q)]).astype(np.int32)
        self.lens = np.asarray(lens_k, np.int32)
        self.q = _randn(g, int(self.cu[-1]) + pad, hq, d, dtype=dtype)
        self.kc, self.vc = (_randn(g, n_pages, page, hkv, d, dtype=dtype) for _ in range(2))
        own = np.zeros((n_pages, page), bool)
        for b, n in enumerate(lens_k):
            for p in range(pages[b]):
                own[self.table[b, p], :min(page, n - p * page)] = True
        self.kc[torch.from_numpy(~own)] = junk
        self.vc[torch.from_numpy(~own)] = junk

    def cuda(self):
        return [t.cuda() for t in (self.q, self.kc, self.vc, _i32(self.table), _i32(self.cu), _i32(self.lens))]

    def refs(self):
        return _f64(self.q), _f64(self.kc), _f64(self.vc), self.table, self.cu, self.lens


def _check_sparse(c, pages, scale=None, **kw):
    q, kc, vc, table, cu, lens = c.cuda()
    scale = c.d ** -0.5 if scale is None else scale
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, lens, _i32(pages).cuda(), scale=scale,
                                                       enable_gqa=True, **kw)
    o, a = orc.sparse_paged_reference(*c.refs(), pages, scale)
    u = torch.finfo(c.dtype).eps / 2
    n = pages.shape[2] * c.page
    vmax = float(c.vc[~c.vc.isnan()].abs().max())
    tol = u * (a + np.abs(o)) * 1.01 + 2e-4 * a + (n * 2.0 ** -25 * vmax if c.dtype == F16 else 0.0) + 2.0 ** -25
    diff = np.abs(_f64(got) - o)
    assert (diff <= tol).all(), (float((diff - tol).max()), int((diff > tol).sum()))
    assert _abi.device_status() == 0
    return got


def _random_pages(c, n, seed, keep_own=True):
    """Ascending distinct pages up to each row's own, -1 behind them."""
    rng = np.random.default_rng(seed)
    out = np.full((c.q.shape[0], c.hkv, n), -1, np.int32)
    for t, b, pos in orc._rows(c.cu, c.lens):
        for h in range(c.hkv):
            have = pos // c.page + 1
            if have <= 0:
                continue
            m = min(n, have)
            p = rng.permutation(have - 1)[:m - 1] if keep_own else rng.permutation(have)[:m]
            p = np.append(p, have - 1) if keep_own else p
            out[t, h, :m] = np.sort(p)
    return out


# ---------------------------------------------------------------- CPU
def test_oracle_sparse_over_all_pages_is_the_paged_reference():
    c = Case([1, 3, 0, 2], [40, 17, 5, 64], 16, 4, 2, 32, F16, 0, junk=0.0)
    pages = np.tile(np.arange(4, dtype=np.int32), (6, 2, 1))
    o, a = orc.sparse_paged_reference(*c.refs(), pages, 0.2)
    q, kc, vc, table, cu, lens = c.refs()
    ref = orc.sdpa_paged_reference(q, kc, vc, table, cu, lens, causal=True, scale=0.2)["o"]
    assert np.abs(o - ref).max() < 1e-12 and (a >= np.abs(o) - 1e-12).all()


def test_oracle_selection_keeps_the_best_pages():
    c = Case([2], [16 * 9 + 5], 16, 2, 1, 32, F16, 1, junk=0.0)
    q, kc, _, table, cu, lens = c.refs()
    means = orc.page_means_reference(kc, np.zeros((kc.shape[0], 1, 32)), table, [0, int(lens[0])], lens)
    got = orc.select_pages_reference(q, means, table, cu, lens, 16, 4, 1, 2)
    for t in range(2):
        s = np.array([max(q[t, g] @ means[table[0, p], 0] for g in range(2)) for p in range(1, 8)])
        best = 1 + np.argsort(-s)[:1]
        assert list(got[t, 0]) == sorted([0, 8, 9, *best])


def test_refusals_on_cpu():
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bt, one = i(2, 4), i(2)
    good = dict(block_table=bt, seqlens_cached=one, seqlens_new=one, free_pages=i(5), free_start=i(1))
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        fa.extend_block_table(**good, page_size=16, total_q=4)
    for kw, message in [
        (dict(block_table=bt.long()), "int32"), (dict(block_table=i(2)), "2-D int32"), (dict(block_table=i(0, 4)), "zero"),
        (dict(block_table=i(4, 2).t()), "contiguous"), (dict(seqlens_new=i(3)), "one entry per row"),
        (dict(free_start=i(2)), "one entry"), (dict(free_pages=i(5).float()), "int32"),
    ]:
        with pytest.raises(ValueError, match=message):
            fa.extend_block_table(**{**good, **kw}, page_size=16, total_q=4)
    for page in (0, 8, 24, 16.0, True):
        with pytest.raises(ValueError, match="page_size"):
            fa.extend_block_table(**good, page_size=page, total_q=4)
    for total in (-1, 1.5, True):
        with pytest.raises(ValueError, match="total_q"):
            fa.extend_block_table(**good, page_size=16, total_q=total)

    q, kv = torch.randn(3, 4, 32).half(), torch.randn(3, 2, 32).half()
    cache, t = torch.zeros(5, 16, 2, 32).half(), fa.rotary_table(8, 32)
    args = [q, kv, kv, cache, cache.clone(), i(3), t, i(3)]
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        fa.paged_append(*args)
    for at, bad, message in [
        (0, q[0], "must have shape"), (1, kv[:2], "key and value"), (2, kv.float(), "same dtype"),
        (3, cache[:, :, :, :16], "contiguous"), (4, cache[:4], "same shape"), (3, cache[0], "num_pages"),
        (5, i(2), "one entry per row"), (5, i(3).long(), "int32"), (6, t.half(), "float32"), (7, i(3, 1), "1-D int32"),
    ]:
        with pytest.raises(ValueError, match=message):
            fa.paged_append(*[bad if j == at else a for j, a in enumerate(args)])
    with pytest.raises(RuntimeError, match="forward only"):
        fa.paged_append(q.clone().requires_grad_(), *args[1:])

    means, cu, lens = torch.zeros(5, 2, 32).half(), i(3), i(2)
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        fa.update_page_means(cache, means, bt, cu, lens)
    for bad, message in [((cache, means[:4], bt, cu, lens), "page_means"), ((cache, means, bt, i(2), lens), "one row"),
                         ((cache, means.float(), bt, cu, lens), "page_means"), ((cache, means, bt, cu, i(3)), "one row")]:
        with pytest.raises(ValueError, match=message):
            fa.update_page_means(*bad)
    with pytest.raises(ValueError, match="total_q"):
        fa.update_page_means(cache, means, bt, cu, lens, total_q=0)

    ok = dict(page_size=16, num_selected=3)
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        fa.select_pages(q, means, bt, cu, lens, **ok)
    for kw, message in [(dict(num_selected=0), "num_selected"), (dict(local_pages=0), "local_pages"),
                        (dict(sink_pages=-1), "sink_pages"), (dict(sink_pages=2, local_pages=2), "not be above"),
                        (dict(page_size=17), "page_size")]:
        with pytest.raises(ValueError, match=message):
            fa.select_pages(q, means, bt, cu, lens, **{**ok, **kw})
    with pytest.raises(ValueError, match="pages wide"):
        fa.select_pages(q, means, i(2, 16385), cu, lens, **ok)
    with pytest.raises(ValueError, match="divisible"):
        fa.select_pages(q[:, :3], means, bt, cu, lens, **ok)

    idx = i(3, 2, 4)
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        fa.scaled_dot_product_attention_paged_sparse(q, cache, cache, bt, cu, lens, idx, enable_gqa=True)
    with pytest.raises(ValueError, match="enable_gqa=True"):
        fa.scaled_dot_product_attention_paged_sparse(q, cache, cache, bt, cu, lens, idx)
    for bad, message in [(idx[:2], "page_indices"), (i(3, 2, 0), "page_indices"), (idx.long(), "int32")]:
        with pytest.raises(ValueError, match=message):
            fa.scaled_dot_product_attention_paged_sparse(q, cache, cache, bt, cu, lens, bad, enable_gqa=True)
    with pytest.raises(ValueError, match="scale"):
        fa.scaled_dot_product_attention_paged_sparse(q, cache, cache, bt, cu, lens, idx, enable_gqa=True,
                                                     scale=float("inf"))


def test_abi_refuses_before_any_cuda_call():
    lib, p = _abi.lib(), 16
    s, odd = _abi.strides_of((4096, 64, 64)), _abi.strides_of((4096, 60, 64))
    E = _abi
    # fa_extend_block_table(..., requests, max_pages, n_free, page_size, total_q, stream)
    for bad in ((0, 4, 5, 16, 4), (2, 0, 5, 16, 4), (2, 4, -1, 16, 4), (2, 4, 5, 12, 4), (2, 4, 5, 16, -1),
                (2, 1 << 28, 5, 16, 4)):
        assert lib.fa_extend_block_table(*[p] * 11, *bad, None) == E.FA_ERR_BAD_SHAPE, bad
    assert lib.fa_extend_block_table(None, *[p] * 10, 2, 4, 5, 16, 4, None) == E.FA_ERR_BAD_SHAPE

    def append(total=4, hq=4, hkv=2, d=64, slots=160, rd=64, q=p, kc=p, vs=s):
        return lib.fa_paged_append(q, p, p, p, kc, p, p, p, p, p, p, total, hq, hkv, d, slots, 8, rd, 0, 0, s, s, vs,
                                   1e-6, None)
    assert append(d=96) == E.FA_ERR_UNSUPPORTED_HEAD_DIM
    for bad in (dict(total=0), dict(slots=0), dict(rd=8), dict(q=None), dict(hkv=0)):
        assert append(**bad) == E.FA_ERR_BAD_SHAPE, bad
    for bad in (dict(kc=24), dict(vs=odd)):
        assert append(**bad) == E.FA_ERR_MISALIGNED, bad
    # fa_page_means(..., B, Hkv, D, num_pages, page_size, width, total_q, stream)
    assert lib.fa_page_means(*[p] * 5, 2, 2, 48, 5, 16, 4, 4, None) == E.FA_ERR_UNSUPPORTED_HEAD_DIM
    for bad in ((0, 2, 64, 5, 16, 4, 4), (2, 2, 64, 5, 20, 4, 4), (2, 2, 64, 1 << 27, 16, 4, 4), (2, 2, 64, 5, 16, 4, 0)):
        assert lib.fa_page_means(*[p] * 5, *bad, None) == E.FA_ERR_BAD_SHAPE, bad

    def select(b=2, hq=4, hkv=2, d=64, total=4, page=16, width=4, top=3, sink=1, local=1, qs=s):
        return lib.fa_select_pages(p, p, p, p, p, p, b, hq, hkv, d, total, 5, page, width, top, sink, local, qs, None)
    assert select(d=16) == E.FA_ERR_UNSUPPORTED_HEAD_DIM
    for bad in (dict(hkv=3), dict(total=0), dict(page=4), dict(width=16385), dict(top=0), dict(sink=-1), dict(local=0),
                dict(sink=2, local=2), dict(sink=3), dict(sink=0x7fffffff, local=0x7fffffff)):
        assert select(**bad) == E.FA_ERR_BAD_SHAPE, bad
    assert select(qs=odd) == E.FA_ERR_MISALIGNED

    def sparse(hq=4, hkv=2, d=64, page=16, top=3, scale=0.1, o=p):
        return lib.fa_fwd_paged_sparse(p, p, p, o, p, p, p, p, 2, hq, hkv, d, 4, 5, page, 4, top, scale, s, None)
    assert sparse(d=256) == E.FA_ERR_UNSUPPORTED_HEAD_DIM
    for bad in (dict(hkv=3), dict(page=8), dict(top=0), dict(scale=float("nan")), dict(o=None), dict(top=1 << 27)):
        assert sparse(**bad) == E.FA_ERR_BAD_SHAPE, bad
    assert sparse(o=20) == E.FA_ERR_MISALIGNED


# ---------------------------------------------------------------- tables
def _check_tables(table, cached, new, free, start, page, total):
    ref = orc.extend_block_table_reference(table, cached, new, free, start, page, total)
    bt = _i32(table).cuda()
    got = fa.extend_block_table(bt, _i32(cached).cuda(), _i32(new).cuda(), _i32(free).cuda(), _i32([start]).cuda(),
                                page_size=page, total_q=total)
    for name in got._fields:
        assert np.array_equal(getattr(got, name).cpu().numpy(), ref[name]), name
    assert np.array_equal(bt.cpu().numpy(), ref["block_table"])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("requests,page,most,width,pool,pad,seed", [
    (1, 16, 1, 1, 4, 0, 0), (1, 64, 300, 8, 9, 3, 1), (5, 16, 40, 6, 100, 0, 2), (513, 32, 20, 9, 3000, 7, 3),
    (1500, 16, 33, 5, 3500, 0, 4), (40, 16, 64, 8, 60, 0, 5), (300, 128, 3000, 60, 100000, 1, 6), (7, 16, 0, 3, 0, 2, 7)])
def test_extend_block_table(requests, page, most, width, pool, pad, seed):
    """Ragged requests, empty ones, ones too long for their row (the lengths
    run past width * page) and free lists that run out."""
    rng = np.random.default_rng(seed)
    cached = rng.integers(0, width * page + 1, requests)
    new = rng.integers(0, most + 1, requests)
    new[rng.random(requests) < 0.2] = 0
    ids = rng.permutation(requests * width + pool)
    table = np.full((requests, width), -7, np.int32)
    at = 0
    for r in range(requests):
        have = -(-int(cached[r]) // page)
        table[r, :have] = ids[at:at + have]
        at += have
    free = ids[at:at + pool]
    start = min(2, pool)
    _check_tables(table, cached, new, free, start, page, int(new.sum()) + pad)
    _check_tables(table, cached, new, free, start, page, max(0, int(new.sum()) - 5))  # rows for not all of them


@pytest.mark.gpu
def test_extend_block_table_odd_values():
    table = np.array([[5, 6], [7, -1], [8, 9]], np.int32)
    # negative lengths count as 0, a start behind the list leaves nothing, a page of -1 gives no slot
    _check_tables(table, [-4, 16, 20], [3, 2, -1], [1, 2, 3], 0, 16, 9)
    _check_tables(table, [17, 16, 20], [3, 2, 1], [1, 2, 3], 3, 16, 6)
    _check_tables(table, [17, 20, 20], [3, 2, 1], [1, 2, 3], 7, 16, 6)
    _check_tables(table, [17, 20, 0], [3, 2, 1], [1, 2, 3], -2, 16, 6)
    _check_tables(table, [2 ** 31 - 1, 1, 0], [2 ** 31 - 1, 1, 1], [1, 2, 3], 0, 16, 2)
    _check_tables(table, [0, 0, 0], [0, 0, 0], [], 0, 16, 0)


# ---------------------------------------------------------------- append
@pytest.mark.gpu
@pytest.mark.parametrize("total,hq,hkv,d,rd,interleaved,norm,wdt,dt", [
    (1, 1, 1, 32, 32, False, True, F16, F16), (9, 4, 2, 64, 32, True, True, torch.float32, F16),
    (130, 7, 1, 128, 128, False, True, BF16, BF16), (77, 5, 5, 128, 64, False, False, None, BF16)])
def test_paged_append(total, hq, hkv, d, rd, interleaved, norm, wdt, dt):
    """The queries and keys are those of ``qk_norm_rotary`` bit for bit, the
    values unchanged, and every other row of the caches is left alone."""
    g = torch.Generator().manual_seed(total)
    page, n_pages = 16, total // 16 + 4
    x = _randn(g, total, hq + 2 * hkv, d, dtype=dt).cuda()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    table = fa.rotary_table(total + 3, rd).cuda()
    pos = torch.randperm(total + 3, generator=g)[:total].int().cuda()
    slots = torch.randperm(n_pages * page, generator=g)[:total].int().cuda()
    slots[::4] = -1
    wq, wk = ((1 + 0.5 * _randn(g, d)).to(wdt).cuda() if norm else None for _ in range(2))
    kc, vc = (torch.full((n_pages, page, hkv, d), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    kw = dict(query_weight=wq, key_weight=wk, interleaved=interleaved)
    out = fa.paged_append(q, k, v, kc, vc, slots, table, pos, **kw)
    zq, zk = fa.qk_norm_rotary(q, k, table, pos, **kw)
    assert torch.equal(out, zq)
    want_k, want_v = torch.full_like(kc, float("nan")), torch.full_like(vc, float("nan"))
    at = slots[slots >= 0].long()
    want_k.view(-1, hkv, d)[at] = zk[slots >= 0]
    want_v.view(-1, hkv, d)[at] = v[slots >= 0]
    assert torch.equal(kc.view(torch.int16), want_k.view(torch.int16))
    assert torch.equal(vc.view(torch.int16), want_v.view(torch.int16))
    assert _abi.device_status() == 0
    # a slot behind the cache writes nothing and is reported
    before = kc.clone()
    fa.paged_append(q[:1], k[:1], v[:1], kc, vc, _i32([n_pages * page]).cuda(), table, pos[:1], **kw)
    assert torch.equal(kc.view(torch.int16), before.view(torch.int16))
    assert _abi.device_status(reset=True) & 0xff == _abi.FA_ERR_BAD_INDEX


# ---------------------------------------------------------------- means and selection
SHAPES = [
    # lens_q, lens_k, page, hq, hkv, d, dtype
    ([1], [1], 16, 1, 1, 32, F16),
    ([1, 1, 1], [700, 33, 48], 16, 4, 2, 64, F16),
    ([4, 0, 2, 1], [260, 90, 700, 16], 16, 14, 2, 128, BF16),
    ([5, 3], [1000, 3], 64, 8, 8, 64, BF16),
    ([1, 130], [900, 130], 32, 6, 3, 32, F16),
    ([2], [5000], 128, 20, 1, 128, F16),
    ([1, 1], [3001, 2049], 16, 12, 4, 128, BF16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens_q,lens_k,page,hq,hkv,d,dt", SHAPES)
def test_page_means_and_selection(lens_q, lens_k, page, hq, hkv, d, dt):
    c = Case(lens_q, lens_k, page, hq, hkv, d, dt, len(lens_k) * 100 + lens_k[0], pad=2)
    q, kc, _, table, cu, lens = c.cuda()
    start = torch.full((kc.shape[0], hkv, d), 0.5, dtype=dt)
    # the step's pages only
    means = start.clone().cuda()
    assert fa.update_page_means(kc, means, table, cu, lens) is means
    ref = orc.page_means_reference(_f64(c.kc), _f64(start), c.table, c.cu, c.lens)
    assert torch.equal(means.cpu(), _rounded_mean(ref, dt))
    # all of them: a step that brought every key
    full = np.concatenate([[0], np.cumsum(lens_k)]).astype(np.int32)
    fa.update_page_means(kc, means, table, _i32(full).cuda(), lens, total_q=int(full[-1]))
    ref = orc.page_means_reference(_f64(c.kc), ref, c.table, full, c.lens)
    assert torch.equal(means.cpu(), _rounded_mean(ref, dt))
    most = max(-(-n // page) for n in lens_k)
    for top, sink, local in ((1, 0, 1), (3, 1, 1), (4, 0, 3), (max(2, most // 3), 1, 1), (most, 1, 1), (most + 3, 2, 1)):
        if sink + local > top:
            continue
        got = fa.select_pages(q, means, table, cu, lens, page_size=page, num_selected=top, sink_pages=sink,
                              local_pages=local)
        want = orc.select_pages_reference(_f64(c.q), _f64(means), c.table, c.cu, c.lens, page, top, sink, local)
        assert np.array_equal(got.cpu().numpy(), want), (top, sink, local)
    assert _abi.device_status() == 0


@pytest.mark.gpu
def test_selection_ties_nan_and_infinite_scores():
    """Equal scores go to the lower page, NaN ranks below everything, and one
    page's infinity above."""
    page, n = 16, 600
    c = Case([2], [page * n - 3], page, 2, 1, 32, BF16, 3, junk=0.0)
    q, kc, _, table, cu, lens = c.cuda()
    q[:] = 1.0
    means = torch.zeros(kc.shape[0], 1, 32, dtype=BF16, device="cuda")
    order = torch.from_numpy(c.table[0].astype(np.int64)).cuda()
    means[order] = (torch.arange(n, device="cuda") % 7).to(BF16)[:, None, None]
    means[order[100]] = float("nan")
    means[order[200]] = float("inf")
    means[order[300]] = -float("inf")
    for top in (3, 40, 300, 599):
        got = fa.select_pages(q, means, table, cu, lens, page_size=page, num_selected=top)
        want = orc.select_pages_reference(_f64(q), _f64(means), c.table, c.cu, c.lens, page, top, 1, 1)
        if top == 599:  # the one page left out is NaN's, behind -inf
            want[:] = np.delete(np.arange(n), 100)
        assert np.array_equal(got.cpu().numpy(), want), top


@pytest.mark.gpu
@pytest.mark.parametrize("n,d,dt,group", [(120, 128, BF16, 2), (700, 64, F16, 1), (2500, 128, F16, 3), (5000, 32, BF16, 6)])
def test_selection_where_fp32_sums_do_not_decide(n, d, dt, group):
    """Large terms that cancel: the scores differ by far less than the
    roundings of an fp32 sum, and the pages are those of the 64-bit ones."""
    page = 16
    c = Case([1], [page * n - 3], page, group, 1, d, dt, n, junk=0.0)
    q, kc, _, table, cu, lens = c.cuda()
    g = torch.Generator().manual_seed(n)
    half = d // 2
    q[:, :, :half] = 900.0 + torch.randint(0, 8, (1, group, half), generator=g).to(q)
    q[:, :, half:] = -q[:, :, :half]
    k = _randn(g, n, half)
    k = torch.cat([k, k + 2.0 ** -7 * torch.randint(-1, 2, (n, half), generator=g)], 1).to(dt)
    means = torch.zeros(kc.shape[0], 1, d, dtype=dt, device="cuda")
    means[torch.from_numpy(c.table[0].astype(np.int64)).cuda(), 0] = k.cuda()
    for top in (3, n // 4, n // 2, n - 1):
        got = fa.select_pages(q, means, table, cu, lens, page_size=page, num_selected=top)
        want = orc.select_pages_reference(_f64(q), _f64(means), c.table, c.cu, c.lens, page, top, 1, 1)
        assert np.array_equal(got.cpu().numpy(), want), top
    # all scores equal: the first pages
    means[:] = means[0]
    got = fa.select_pages(q, means, table, cu, lens, page_size=page, num_selected=n // 2)
    assert got[0, 0].tolist() == [*range(n // 2 - 1), n - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["huge", "tiny", "zero", "nan", "inf"])
def test_selection_with_queries_and_means_at_the_edges(what):
    page, n = 16, 900
    c = Case([1], [page * n - 3], page, 2, 1, 64, BF16, 5, junk=0.0)
    q, kc, _, table, cu, lens = c.cuda()
    g = torch.Generator().manual_seed(6)
    means = _randn(g, kc.shape[0], 1, 64, dtype=BF16).cuda()
    if what == "huge":  # squares and products past the fp32 range, with both signs
        q, means = q * 2.0 ** 90, means * 2.0 ** 60
    elif what == "tiny":  # products below it
        q, means = q * 2.0 ** -90, means * 2.0 ** -60
    elif what == "zero":
        means[:] = 0
    elif what == "nan":
        q[0, 1, 3] = float("nan")
    else:
        q[0, 0, 3] = float("inf")
    got = fa.select_pages(q, means, table, cu, lens, page_size=page, num_selected=100)
    with np.errstate(all="ignore"):
        want = orc.select_pages_reference(_f64(q), _f64(means), c.table, c.cu, c.lens, page, 100, 1, 1)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 5, 8, 9, 17, 40])
def test_selection_groups_and_scores_in_heaps(group):
    """Groups on both sides of 8 heads; then a few scores a million times the
    others', and scores in two heaps, so that nearly all lie close together."""
    page, n = 16, 1500
    for d, dt in ((32, F16), (64, BF16), (128, F16)):
        c = Case([1], [page * n - 3], page, 2 * group, 2, d, dt, group + d, junk=0.0)
        q, kc, _, table, cu, lens = c.cuda()
        g = torch.Generator().manual_seed(group * d)
        means = _randn(g, kc.shape[0], 2, d, dtype=dt).cuda() * 0.125
        for what in ("plain", "outliers", "heaps"):
            if what == "outliers":
                means[:: means.shape[0] // 5] *= 2.0 ** 14
                means *= 2.0 ** -6
            elif what == "heaps":
                means = (means[:1] * 2.0 ** -8).expand(means.shape).clone()
                means[: means.shape[0] // 2] *= -1.0
                means[:, :, 0] += (torch.arange(means.shape[0]) % 16 * 2.0 ** -6).to(means)[:, None]
            for top in (3, 64, 700, n - 1):
                got = fa.select_pages(q, means, table, cu, lens, page_size=page, num_selected=top)
                want = orc.select_pages_reference(_f64(q), _f64(means), c.table, c.cu, c.lens, page, top, 1, 1)
                assert np.array_equal(got.cpu().numpy(), want), (d, what, top)


@pytest.mark.gpu
def test_selection_over_the_widest_table():
    n = 16384
    c = Case([1], [16 * n], 16, 2, 1, 32, F16, 4, junk=0.0)
    q, kc, _, table, cu, lens = c.cuda()
    means = torch.zeros(kc.shape[0], 1, 32, dtype=F16, device="cuda")
    fa.update_page_means(kc, means, table, _i32([0, 16 * n]).cuda(), lens)
    got = fa.select_pages(q, means, table, cu, lens, page_size=16, num_selected=1000)
    want = orc.select_pages_reference(_f64(q), _f64(means), c.table, c.cu, c.lens, 16, 1000, 1, 1)
    assert np.array_equal(got.cpu().numpy(), want)


# ---------------------------------------------------------------- attention
@pytest.mark.gpu
@pytest.mark.parametrize("lens_q,lens_k,page,hq,hkv,d,dt", SHAPES)
@pytest.mark.parametrize("n", [1, 3, 17, 64])
def test_sparse_attention(lens_q, lens_k, page, hq, hkv, d, dt, n):
    c = Case(lens_q, lens_k, page, hq, hkv, d, dt, len(lens_k) * 100 + lens_k[0], pad=2)
    got = _check_sparse(c, _random_pages(c, n, 7))
    assert (got[int(c.cu[-1]):] == 0).all()
    _check_sparse(c, _random_pages(c, n, 8, keep_own=False))


@pytest.mark.gpu
@pytest.mark.parametrize("group", [1, 8, 9, 16, 17, 40])
def test_sparse_attention_groups_and_scales(group):
    for d, dt in ((32, F16), (64, BF16), (128, F16)):
        c = Case([1, 2], [333, 100], 16, 2 * group, 2, d, dt, group)
        _check_sparse(c, _random_pages(c, 9, 1), scale=0.5 * d ** -0.5)
        _check_sparse(c, _random_pages(c, 9, 2), scale=-0.25)
        _check_sparse(c, _random_pages(c, 9, 2), scale=0.0)


@pytest.mark.gpu
def test_sparse_attention_of_all_pages_is_the_paged_call():
    c = Case([1, 1, 1], [777, 64, 3000], 64, 8, 2, 128, F16, 11, junk=0.0)
    q, kc, vc, table, cu, lens = c.cuda()
    pages = torch.arange(table.shape[1], dtype=torch.int32, device="cuda").expand(3, 2, -1)
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table.clamp(min=0), cu, lens, pages, enable_gqa=True)
    want = fa.scaled_dot_product_attention_paged(q, kc, vc, table.clamp(min=0), cu, lens, 1, 3000, is_causal=True,
                                                 enable_gqa=True)
    # both within the bar of 2e-3 of float64
    assert float((got.float() - want.float()).abs().max()) <= 4e-3


@pytest.mark.gpu
def test_sparse_attention_lists_out_of_order_repeated_empty_and_ahead():
    c = Case([2, 1], [500, 40], 16, 4, 2, 64, F16, 12)
    pages = _random_pages(c, 6, 3)
    pages[0, 0] = [9, 2, -1, 2, 31, 0]  # out of order, one twice, one behind the row's own page (30)
    pages[1, 1] = -1
    pages[2, 0] = [2, 2, 2, 2, -1, 2]
    pages[2, 1] = [3, 5, 100, 2 ** 31 - 1, -5, -2 ** 31]  # nothing that the row sees
    got = _check_sparse(c, pages)
    assert (got[1, 2:] == 0).all() and (got[2, 2:] == 0).all()


@pytest.mark.gpu
def test_sparse_attention_with_infinities_and_peaked_scores():
    c = Case([1], [640], 16, 2, 1, 64, BF16, 13)
    c.q[0] *= 60  # scores in the hundreds: one key takes all
    _check_sparse(c, np.arange(40, dtype=np.int32)[None, None])
    c = Case([1], [640], 16, 2, 1, 64, F16, 14)
    c.kc[c.table[0, 3], 2, 0] = 0
    c.q[0, :, 0], c.kc[c.table[0, 3], 2, 0, 0] = 1.0, -float("inf")  # a score of -inf among finite ones
    _check_sparse(c, np.arange(40, dtype=np.int32)[None, None])
    c.vc[c.table[0, 5], 1, 0, 7] = float("nan")  # a seen NaN stays one
    q, kc, vc, table, cu, lens = c.cuda()
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, lens,
                                                       torch.arange(40).int().cuda()[None, None], enable_gqa=True)
    assert got[0, :, 7].isnan().all() and not got[0, :, :7].isnan().any()


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_refused_on_the_device():
    c = Case([1, 1], [200, 100], 16, 4, 2, 64, F16, 15)
    pages = _random_pages(c, 5, 1)
    ref, _ = orc.sparse_paged_reference(*c.refs(), pages[1:][[0, 0]], c.d ** -0.5)
    q, kc, vc, table, cu, lens = c.cuda()
    means = torch.zeros(kc.shape[0], 2, 64, dtype=F16, device="cuda")
    for bad in (-1, -2 ** 31, kc.shape[0], 2 ** 31 - 1):
        t = table.clone()
        t[0] = bad
        out = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, t, cu, lens, _i32(pages).cuda(), enable_gqa=True)
        assert (out[0] == 0).all() and out[1].isfinite().all() and (out[1] != 0).any()
        assert _abi.device_status(reset=True) & 0xff == _abi.FA_ERR_BAD_INDEX
        fa.select_pages(q, means, t, cu, lens, page_size=16, num_selected=4)
        assert _abi.device_status(reset=True) & 0xff == _abi.FA_ERR_BAD_INDEX
        before = means.clone()
        fa.update_page_means(kc, means, t, _i32([0, 200, 201]).cuda(), _i32([200, 100]).cuda())
        assert torch.equal(means, before)
        assert _abi.device_status(reset=True) & 0xff == _abi.FA_ERR_BAD_INDEX
    # more keys than the table's row holds; fewer keys than rows
    for lens_bad in ([100_000, 100], [-3, 100], [0, 100]):
        out = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, _i32(lens_bad).cuda(),
                                                           _i32(pages).cuda(), enable_gqa=True)
        assert (out[0] == 0).all()
        sel = fa.select_pages(q, means, table, cu, _i32(lens_bad).cuda(), page_size=16, num_selected=4)
        assert (sel[0] == -1).all()
        code = _abi.device_status(reset=True) & 0xff
        assert code == (_abi.FA_ERR_BAD_INDEX if lens_bad[0] > 0 else 0)


@pytest.mark.gpu
def test_cache_offsets_past_32_bits():
    """Slots whose element offsets pass 2^31 in the caches (and 2^32 bytes)."""
    page, hkv, d = 64, 8, 128
    n_pages = (1 << 31) // (page * hkv * d) + 40
    kc, vc = (torch.empty(n_pages, page, hkv, d, dtype=F16, device="cuda") for _ in range(2))
    n, hq = 300, 16
    ids = torch.tensor([n_pages - 1 - i for i in range(5)], dtype=torch.int32)
    g = torch.Generator().manual_seed(1)
    x = _randn(g, n, hq + 2 * hkv, d, dtype=F16).cuda()
    slots = (ids.repeat_interleave(page) * page + torch.arange(5 * page) % page)[:n].int().cuda()
    pos = torch.arange(n, dtype=torch.int32).cuda()
    table = fa.rotary_table(n, d).cuda()
    q = fa.paged_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], kc, vc, slots, table, pos)
    means = torch.zeros(n_pages, hkv, d, dtype=F16, device="cuda")
    bt, cu, lens = ids[None].cuda(), _i32([0, n]).cuda(), _i32([n]).cuda()
    fa.update_page_means(kc, means, bt, cu, lens)
    pages = fa.select_pages(q, means, bt, cu, lens, page_size=page, num_selected=3)
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, bt, cu, lens, pages, enable_gqa=True)
    # the same in a small cache
    kc2, vc2 = (torch.zeros(5, page, hkv, d, dtype=F16, device="cuda") for _ in range(2))
    bt2 = torch.arange(5, dtype=torch.int32, device="cuda")[None]
    q2 = fa.paged_append(x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], kc2, vc2, pos, table, pos)
    means2 = torch.zeros(5, hkv, d, dtype=F16, device="cuda")
    fa.update_page_means(kc2, means2, bt2, cu, lens)
    pages2 = fa.select_pages(q2, means2, bt2, cu, lens, page_size=page, num_selected=3)
    got2 = fa.scaled_dot_product_attention_paged_sparse(q2, kc2, vc2, bt2, cu, lens, pages2, enable_gqa=True)
    assert torch.equal(q, q2) and torch.equal(pages, pages2) and torch.equal(got, got2)
    assert _abi.device_status() == 0


# ---------------------------------------------------------------- the step
class Server:
    """A few requests over one cache, through the calls in their order."""

    def __init__(self, requests, hq=8, hkv=2, d=64, page=16, width=24, pool=200, dtype=F16, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv, self.d, self.page, self.g, self.dtype = hq, hkv, d, page, g, dtype
        dev = "cuda"
        self.bt = torch.zeros(requests, width, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=dev)
        self.free = torch.randperm(pool, generator=g).int().to(dev)
        self.start = torch.zeros(1, dtype=torch.int32, device=dev)
        self.kc, self.vc = (torch.full((pool, page, hkv, d), float("nan"), dtype=dtype, device=dev) for _ in range(2))
        self.means = torch.zeros(pool, hkv, d, dtype=dtype, device=dev)
        self.rope = fa.rotary_table(width * page, d).cuda()
        self.w = (1 + 0.3 * _randn(g, d)).cuda()

    def x(self, total):
        return _randn(self.g, total, self.hq + 2 * self.hkv, self.d, dtype=self.dtype).cuda()

    def step(self, new, x, top=4):
        """Updates its own state in place, so that a captured step can be replayed."""
        s = fa.extend_block_table(self.bt, self.lens, new, self.free, self.start, page_size=self.page,
                                  total_q=x.shape[0])
        q = fa.paged_append(x[:, :self.hq], x[:, self.hq:-self.hkv], x[:, -self.hkv:], self.kc, self.vc,
                            s.slot_mapping, self.rope, s.positions, query_weight=self.w, key_weight=self.w)
        fa.update_page_means(self.kc, self.means, self.bt, s.cu_seqlens_q, s.seqlens_k)
        pages = fa.select_pages(q, self.means, self.bt, s.cu_seqlens_q, s.seqlens_k, page_size=self.page,
                                num_selected=top)
        o = fa.scaled_dot_product_attention_paged_sparse(q, self.kc, self.vc, self.bt, s.cu_seqlens_q, s.seqlens_k,
                                                         pages, enable_gqa=True)
        self.lens.copy_(s.seqlens_k)
        self.start.copy_(s.free_next)
        return q, pages, o, s


@pytest.mark.gpu
def test_serving_steps_against_dense_float64():
    """Three prompts and several decode steps, in padded batches; every row's
    pages and output against float64 over the plain history of its request."""
    sv = Server(3)
    history = [[[], []] for _ in range(3)]
    plans = [[40, 3, 0], [1, 1, 70], [1, 1, 1], [2, 30, 1], [1, 1, 1]]
    for plan in plans:
        x = sv.x(sum(plan) + 3)
        q, pages, o, s = sv.step(_i32(plan).cuda(), x)
        assert s.fits.all()
        lens = sv.lens.cpu().numpy()
        row = 0
        x64 = _f64(x)
        for r, n in enumerate(plan):
            pos = np.arange(lens[r] - n, lens[r])
            zk = orc.norm_rotary_reference(x64[row:row + n, sv.hq:-sv.hkv], _f64(sv.w), sv.rope.cpu().numpy(), pos,
                                           1e-6, False)["z"]
            zq = orc.norm_rotary_reference(x64[row:row + n, :sv.hq], _f64(sv.w), sv.rope.cpu().numpy(), pos, 1e-6,
                                           False)["z"]
            history[r][0].extend(zk)
            history[r][1].extend(x64[row:row + n, -sv.hkv:])
            k, v = (np.array(h).reshape(-1, sv.hkv, sv.d) for h in history[r])
            for i in range(n):
                own = pos[i] // 16
                for h in range(sv.hkv):
                    kept = pages[row + i, h].cpu().numpy()
                    kept = kept[kept >= 0]
                    assert len(kept) == min(4, own + 1) and 0 in kept and own in kept
                    rows = np.concatenate([np.arange(p * 16, min(p * 16 + 16, pos[i] + 1)) for p in kept])
                    qg = zq[i, h * 4:h * 4 + 4]
                    sc = qg @ k[rows, h].T * sv.d ** -0.5
                    w = np.exp(sc - sc.max(-1, keepdims=True))
                    want = (w / w.sum(-1, keepdims=True)) @ v[rows, h]
                    # the attention's bar of 2e-3, and queries and keys rounded to fp16 on the way
                    assert np.abs(_f64(o[row + i, h * 4:h * 4 + 4]) - want).max() <= 4e-3
            row += n
        assert (o[row:] == 0).all() and (s.slot_mapping[row:] == -1).all()
    assert _abi.device_status() == 0


@pytest.mark.gpu
def test_serving_step_captured_and_replayed():
    """A decode step captured once and replayed, the state advancing on the
    GPU, gives what eager steps give; two captured servers do not disturb each
    other."""
    eager, a, b = (Server(4, seed=9) for _ in range(3))
    prompt = _i32([50, 17, 200, 5]).cuda()
    x0 = eager.x(272)
    for sv in (eager, a, b):
        sv.step(prompt, x0)
    one = _i32([1, 1, 1, 1]).cuda()
    xs = [eager.x(4) for _ in range(20)]
    inputs, outs, graphs = [], [], []
    for sv in (a, b):
        xin = xs[0].clone()
        lens, start = sv.lens.clone(), sv.start.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sv.step(one, xin)  # warm-up, then the state as it was
        torch.cuda.current_stream().wait_stream(side)
        sv.lens.copy_(lens)
        sv.start.copy_(start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sv.step(one, xin)[2]
        inputs.append(xin)
        outs.append(out)
        graphs.append(graph)
    for x in xs:
        want = eager.step(one, x)[2]
        for i in range(2):
            inputs[i].copy_(x)
            graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    assert torch.equal(a.lens, eager.lens) and torch.equal(a.means, eager.means) and torch.equal(a.bt, eager.bt)
    assert _abi.device_status() == 0


@pytest.mark.gpu
def test_calls_on_two_streams_at_once_with_strided_queries_and_tables():
    """The same calls from two streams that overlap, with queries that are
    views of a projection (and one off the 16-byte boundary) and a table that
    is a view, give what they give alone."""
    cases = [Case([1, 2, 1], [900, 333, 64], 16, 8, 2, 64, BF16, s, pad=1) for s in (21, 22)]
    want, work = [], []
    for c in cases:
        q, kc, vc, table, cu, lens = c.cuda()
        proj = torch.zeros(q.shape[0], 12, 64, dtype=BF16, device="cuda")
        proj[:, 2:10] = q
        odd = torch.zeros(q.numel() + 1, dtype=BF16, device="cuda")
        odd[1:] = q.flatten()
        wide = torch.full((table.shape[0], table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
        wide[:, :-3] = table
        work.append((proj[:, 2:10], odd[1:].view(q.shape), kc, vc, wide[:, :-3], cu, lens))
        want.append(_select_and_attend(q, kc, vc, table, cu, lens))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for st, (view, odd, *rest) in zip(streams, work):
            with torch.cuda.stream(st):
                got.append([_select_and_attend(q, *rest) for q in (view, odd)])
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for one in g:
                assert all(torch.equal(a, b) for a, b in zip(one, w))
    assert _abi.device_status() == 0


def _select_and_attend(q, kc, vc, table, cu, lens):
    means = torch.zeros(kc.shape[0], *kc.shape[2:], dtype=kc.dtype, device=kc.device)
    full = torch.cat([cu[:1], lens.cumsum(0)]).int()
    fa.update_page_means(kc, means, table, full, lens)
    pages = fa.select_pages(q, means, table, cu, lens, page_size=kc.shape[1], num_selected=7)
    return pages, fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, lens, pages, enable_gqa=True)


@pytest.mark.gpu
def test_many_rows_a_sequence():
    """A prefill chunk through the decode calls: more rows than the GPU holds
    blocks, with lists of all their pages, against the paged call."""
    c = Case([700, 1, 300], [700, 1000, 333], 32, 8, 2, 64, F16, 31, junk=0.0)
    q, kc, vc, table, cu, lens = c.cuda()
    means = torch.zeros(kc.shape[0], 2, 64, dtype=F16, device="cuda")
    pages = fa.select_pages(q, means, table, cu, lens, page_size=32, num_selected=table.shape[1])
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, lens, pages, enable_gqa=True)
    want = fa.scaled_dot_product_attention_paged(q, kc, vc, table.clamp(min=0), cu, lens, 700, 1000, is_causal=True,
                                                 enable_gqa=True)
    assert float((got.float() - want.float()).abs().max()) <= 4e-3  # each within 2e-3 of float64


PACKED = ["fa_qk_norm_rotary", "fa_qk_norm_rotary_bwd", "fa_paged_append", "fa_extend_block_table",
          "fa_page_means", "fa_select_pages", "fa_fwd_paged_sparse"]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("name", PACKED)
def test_packed_entries_answer_as_the_entries_do(name, dtype):
    """Arguments that every entry refuses before any CUDA call: null pointers
    (after the head dim and sizes have passed), a head dim, an int of more
    than 32 bits."""
    dtype = None if name == "fa_extend_block_table" else dtype
    entry = _abi.entry(name, dtype)
    call, pack = _abi.packed_entry(name, dtype)
    kinds = _abi.SIGNATURES[entry.__name__][1]
    for ints in (64, 0, 48, 1 << 30):
        args = [ints if t is ctypes.c_int else 1e-6 if t is ctypes.c_float else 0 for t in kinds]
        alone = [None if t not in (ctypes.c_int, ctypes.c_float, ctypes.c_int64) else v for v, t in zip(args, kinds)]
        rc = entry(*alone)
        assert rc in (_abi.FA_ERR_BAD_SHAPE, _abi.FA_ERR_UNSUPPORTED_HEAD_DIM)
        assert call(pack(*args)) == rc
    wide = [(1 << 32) + 64 if t is ctypes.c_int else 1e-6 if t is ctypes.c_float else 0 for t in kinds]
    assert call(pack(*wide)) == _abi.FA_ERR_BAD_SHAPE
    assert call(None) == _abi.FA_ERR_BAD_SHAPE


def test_packed_entry_of_another_name():
    assert not _abi.lib().fa_packed_entry(b"fa_fwd") and not _abi.lib().fa_packed_entry(None)
    with pytest.raises(RuntimeError, match="packed"):
        _abi.packed_entry("fa_fwd", torch.float16)
    s = _abi.strides_of((1, 2, 3))
    assert s.at == ctypes.addressof(s) and list(s) == [1, 2, 3]


# ---------------------------------------------------------------- weights, lengths, refused requests
@pytest.mark.gpu
@pytest.mark.parametrize("group", [3, 4, 5])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
def test_sparse_attention_keeps_its_weights_in_more_bits_than_the_operands(dt, d, group):
    """Queries and keys of -1, 0 and 1: scores are exact in any order.  With A
    the attention of |v| and up to 64 keys, a weight is off by the scale's,
    the product's and the difference's roundings (3 x 2^-24 of at most 8, in
    base 2) and the exponential's 2^-22: 2^-20; once in the sum and once in
    the product, which adds 17 values a time at 2^-23 and joins 4 warps:
    below 2^-17 A in all.  To it come what is lost of a weight held as two
    numbers of the operand type, the first cut off and the second rounded:
    2^-10 2^-11 (fp16) or 2^-7 2^-8 (bf16), and the result's own rounding.
    Weights rounded once to the operand type would be off by 2^-11 or 2^-8."""
    rng = np.random.default_rng(d)
    lens = [2, 3, 5, 9, 16, 17, 33, 64]
    c = Case([1] * len(lens), lens, 16, 2 * group, 2, d, dt, d, junk=0.0)
    c.q[:] = torch.from_numpy(rng.integers(-1, 2, c.q.shape)).to(dt)
    c.kc[:] = torch.from_numpy(rng.integers(-1, 2, c.kc.shape)).to(dt)
    pages = np.tile(np.arange(4, dtype=np.int32), (len(lens), 2, 1))
    q, kc, vc, table, cu, ln = c.cuda()
    scale = 0.11 * (32 / d) ** 0.5
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, ln, _i32(pages).cuda(), scale=scale,
                                                       enable_gqa=True)
    o, a = orc.sparse_paged_reference(*c.refs(), pages, scale)
    split = 2.0 ** -21 if dt == F16 else 2.0 ** -15
    tol = (torch.finfo(dt).eps / 2 * np.abs(o) * 1.001 + (2.0 ** -17 + split) * a + (2.0 ** -25 if dt == F16 else 0.0))
    diff = np.abs(_f64(got) - o)
    assert (diff <= tol).all(), (float((diff - tol).max()), int((diff > tol).sum()))


@pytest.mark.gpu
def test_fp16_weights_far_below_the_largest_are_not_lost():
    """One key of every 16 has weight 1 and no value, the others 2^-19.84 each
    and large values.  2^-19.84 by itself lies between fp16's subnormal steps:
    rounded to one of them it would be off by half a percent."""
    n = 1001
    c = Case([1], [n], 16, 1, 1, 64, F16, 41, junk=0.0)
    c.q[:], c.kc[:], c.vc[:] = 0, 0, 0
    c.q[0, 0, 0] = 1.0
    j = np.arange(n)
    rows = torch.from_numpy(c.table[0, j // 16].astype(np.int64) * 16 + j % 16)
    c.kc.view(-1, 64)[rows, 0] = -13.75
    c.vc.view(-1, 64)[rows] = 1000.0
    c.kc.view(-1, 64)[rows[::16]] = 0.0
    c.vc.view(-1, 64)[rows[::16]] = 0.0
    pages = np.arange(63, dtype=np.int32)[None, None]
    q, kc, vc, table, cu, ln = c.cuda()
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, ln, _i32(pages).cuda(), scale=1.0)
    o, _ = orc.sparse_paged_reference(*c.refs(), pages, 1.0)
    # the result's rounding; the score in base 2 is off by 2 x 2^-24 of 20, the sums by 2^-23 of some hundred terms
    assert (np.abs(_f64(got) - o) <= (2.0 ** -11 + 2.0 ** -14) * o).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group", [3, 6])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("dt", [F16, BF16], ids=str)
def test_infinite_values_stay_infinite(dt, d, group):
    """Values of infinity under weights of 1, of few bits and of many; both
    signs in one column are no number.  The other columns are as without."""
    c = Case([1, 1], [40, 7], 16, group, 1, d, dt, d + 1, junk=0.0)
    c.q[:], c.kc[:] = 0, 0
    c.q[:, :, 0] = 1.0
    at = c.table[0, np.arange(40) // 16].astype(np.int64) * 16 + np.arange(40) % 16
    k, v = c.kc.view(-1, d), c.vc.view(-1, d)
    # weights (scale ln 2): keys 0 and 5 have 1, 9 has 1/2, 20 has 2^-3.25, 33 has 2^-14.5
    k[torch.from_numpy(at), 0] = -3.0
    for j, e in ((0, 0.0), (5, 0.0), (9, -1.0), (20, -3.25), (33, -14.5)):
        k[at[j], 0] = e
    pages = np.tile(np.arange(3, dtype=np.int32), (2, 1, 1))
    want, _ = orc.sparse_paged_reference(*c.refs(), pages, float(np.log(2.0)))
    inf = float("inf")
    for j, col, x in ((0, 1, inf), (9, 2, -inf), (20, 3, inf), (33, 4, inf), (5, 5, inf), (20, 5, -inf), (33, 6, -inf)):
        v[at[j], col] = x
    q, kc, vc, table, cu, lens = c.cuda()
    got = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, table, cu, lens, _i32(pages).cuda(),
                                                       scale=float(np.log(2.0)), enable_gqa=True)[0]
    for col, x in ((1, inf), (2, -inf), (3, inf), (4, inf), (6, -inf)):
        assert (got[:, col] == x).all(), col
    assert got[:, 5].isnan().all()
    u = torch.finfo(dt).eps / 2
    assert (np.abs(_f64(got)[:, 7:] - want[0][:, 7:]) <= u * np.abs(want[0][:, 7:]) * 1.001 + 2.0 ** -13).all()


@pytest.mark.gpu
def test_page_means_refuse_a_sequence_longer_than_its_table_row():
    """As the selection and the attention do: nothing of it is written, the
    device status is set, and the other sequences' means are made."""
    c = Case([40, 100], [200, 100], 16, 4, 2, 64, F16, 15)
    _, kc, _, table, _, _ = c.cuda()
    start = torch.full((kc.shape[0], 2, 64), 0.5, dtype=F16)
    width = table.shape[1]
    for nk in (width * 16 + 1, width * 16 + 39, 100_000, 2 ** 31 - 1):
        means = start.clone().cuda()
        fa.update_page_means(kc, means, table, _i32(c.cu).cuda(), _i32([nk, 100]).cuda())
        want = orc.page_means_reference(_f64(c.kc), _f64(start), c.table[1:], [0, 100], [100])
        assert torch.equal(means.cpu(), _rounded_mean(want, F16)), nk
        assert _abi.device_status(reset=True) & 0xff == _abi.FA_ERR_BAD_INDEX, nk
    # as long as its row, and one that brings no rows this step
    means = start.clone().cuda()
    fa.update_page_means(kc, means, table.clamp(min=0), _i32([0, 0, 100]).cuda(), _i32([100_000, 100]).cuda())
    assert _abi.device_status(reset=True) == 0


@pytest.mark.gpu
def test_a_token_without_a_slot_may_be_at_any_position():
    """A request that does not fit has slots of -1 and positions that may lie
    behind the angles' table: no error, and nothing is written for it.  A
    token with a slot and such a position is one."""
    g = torch.Generator().manual_seed(3)
    x = _randn(g, 6, 8, 64, dtype=F16).cuda()
    kc, vc = (torch.full((3, 16, 2, 64), float("nan"), dtype=F16, device="cuda") for _ in range(2))
    table = fa.rotary_table(8, 64).cuda()
    pos, slots = _i32([0, 8, -1, 2 ** 31 - 1, 7, 3]).cuda(), _i32([5, -1, -1, -1, -1, 20]).cuda()
    q = fa.paged_append(x[:, :4], x[:, 4:6], x[:, 6:], kc, vc, slots, table, pos)
    assert _abi.device_status(reset=True) == 0
    assert q[[0, 4, 5]].isfinite().all()
    assert torch.equal(vc.view(-1, 2, 64)[[5, 20]], x[[0, 5], 6:])
    left = torch.ones(48, dtype=torch.bool)
    left[[5, 20]] = False
    assert kc.view(-1, 2, 64)[left.cuda()].isnan().all() and vc.view(-1, 2, 64)[left.cuda()].isnan().all()
    slots[2] = 7
    fa.paged_append(x[:, :4], x[:, 4:6], x[:, 6:], kc, vc, slots, table, pos)
    assert _abi.device_status(reset=True) & 0xff == _abi.FA_ERR_BAD_INDEX


@pytest.mark.gpu
def test_a_step_with_requests_that_do_not_fit():
    """One request is too long for its row (its positions pass the angles'
    table), one finds no page.  With ``seqlens_attended`` for the calls behind
    the append their rows see no key and complete no page, nothing is an
    error, and the others get what they get when those two bring nothing."""
    def attend(sv, x, s, lens):
        q = fa.paged_append(x[:, :sv.hq], x[:, sv.hq:-sv.hkv], x[:, -sv.hkv:], sv.kc, sv.vc, s.slot_mapping, sv.rope,
                            s.positions, query_weight=sv.w, key_weight=sv.w)
        fa.update_page_means(sv.kc, sv.means, sv.bt, s.cu_seqlens_q, lens)
        pages = fa.select_pages(q, sv.means, sv.bt, s.cu_seqlens_q, lens, page_size=sv.page, num_selected=3)
        o = fa.scaled_dot_product_attention_paged_sparse(q, sv.kc, sv.vc, sv.bt, s.cu_seqlens_q, lens, pages,
                                                         enable_gqa=True)
        dense = fa.scaled_dot_product_attention_paged(q, sv.kc, sv.vc, sv.bt, s.cu_seqlens_q, lens, 1000, 24 * 16,
                                                      is_causal=True, enable_gqa=True)
        return pages, o, dense

    def served(new, rows):
        sv = Server(4, pool=12)
        for t in (sv.kc, sv.vc):  # the dense call wants finite rows behind a sequence's end
            t.zero_()
        x0 = sv.x(100)
        sv.step(_i32([40, 33, 20, 7]).cuda(), x0)  # 3 + 3 + 2 + 1 pages of 12
        before = sv.kc.clone(), sv.means.clone(), sv.bt.clone()
        x = _randn(torch.Generator().manual_seed(1), 512, sv.hq + 2 * sv.hkv, sv.d, dtype=sv.dtype).cuda()[rows]
        s = fa.extend_block_table(sv.bt, sv.lens, _i32(new).cuda(), sv.free, sv.start, page_size=sv.page,
                                  total_q=x.shape[0])
        return sv, before, x, s

    assert _abi.device_status(reset=True) == 0
    # request 1 has room in its row for 24 pages only, request 3 lacks pages; requests 0 and 2 need one page each
    first = [*range(9), *range(9, 409), *range(409, 422), *range(422, 512)]
    sv, before, x, s = served([9, 400, 13, 90], first)
    assert s.fits.tolist() == [True, False, True, False]
    assert s.seqlens_attended.tolist() == [49, 0, 33, 0] and s.seqlens_attended.dtype == torch.int32
    pages, o, dense = attend(sv, x, s, s.seqlens_attended)
    assert _abi.device_status(reset=True) == 0
    refused = [*range(9, 409), *range(422, 512)]
    assert (pages[refused] == -1).all() and (o[refused] == 0).all() and (dense[refused] == 0).all()
    kept = [*range(9), *range(409, 422)]
    sv2, _, x2, s2 = served([9, 0, 13, 0], kept)
    pages2, o2, dense2 = attend(sv2, x2, s2, s2.seqlens_attended)
    assert s2.fits.all() and s2.seqlens_attended.tolist() == s2.seqlens_k.tolist()[:1] + [33, 33, 7]
    assert torch.equal(pages[kept], pages2) and torch.equal(o[kept], o2) and torch.equal(sv.kc, sv2.kc)
    assert torch.equal(sv.means, sv2.means) and torch.equal(sv.bt, sv2.bt)
    assert float((dense[kept].float() - dense2.float()).abs().max()) <= 4e-3  # other tiles: each within 2e-3
    # the refused ones' history is as it was
    for r, n in ((1, 33), (3, 7)):
        for p in range(-(-n // 16)):
            page = int(sv.bt[r, p])
            assert page == int(before[2][r, p]) and torch.equal(sv.kc[page], before[0][page])
            assert torch.equal(sv.means[page], before[1][page])


@pytest.mark.gpu
def test_a_sequence_next_to_a_refused_one_is_the_reference():
    """Bad pages, lengths past the table and lengths below the rows' in one
    sequence: the other one's pages and output are float64's."""
    c = Case([1, 1], [200, 100], 16, 4, 2, 64, F16, 15)
    pages = _random_pages(c, 5, 1)
    o, a = orc.sparse_paged_reference(*c.refs(), pages, c.d ** -0.5)
    tol = (2.0 ** -11 * (a + np.abs(o)) * 1.01 + 2e-4 * a + 80 * 2.0 ** -25 * 5 + 2.0 ** -25)[1]
    q, kc, vc, table, cu, lens = c.cuda()
    means = torch.zeros(kc.shape[0], 2, 64, dtype=F16, device="cuda")
    fa.update_page_means(kc, means, table, _i32([0, 200, 300]).cuda(), lens)
    sel = orc.select_pages_reference(_f64(c.q), _f64(means), c.table, c.cu, c.lens, 16, 4, 1, 1)
    assert _abi.device_status(reset=True) == 0
    bad = [(torch.cat([torch.full_like(table[:1], b), table[1:]]), lens) for b in (-1, -2 ** 31, kc.shape[0], 2 ** 31 - 1)]
    bad += [(table, _i32([n, 100]).cuda()) for n in (100_000, 2 ** 31 - 1, -3, 0)]
    for t, ln in bad:
        out = fa.scaled_dot_product_attention_paged_sparse(q, kc, vc, t, cu, ln, _i32(pages).cuda(), enable_gqa=True)
        assert (out[0] == 0).all() and (np.abs(_f64(out[1]) - o[1]) <= tol).all()
        got = fa.select_pages(q, means, t, cu, ln, page_size=16, num_selected=4)
        assert np.array_equal(got[1].cpu().numpy(), sel[1])
        _abi.device_status(reset=True)
