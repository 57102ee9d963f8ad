"""What is measured of the operators around the paged K/V cache and the
query/key preparation: the cases, their inputs, the operators in plain torch
and the calls a user makes of them.

Five kinds of case:

* ``rotary``: ``qk_norm_rotary`` forward and backward, as a training step
  uses it between the projections and the attention;
* ``append``: ``paged_append``, the same preparation for serving, with keys
  and values written into the paged cache;
* ``tables``: ``extend_block_table``, the step's block table, slot map and
  offsets from request lengths;
* ``select``: ``update_page_means`` and ``select_pages``, the two calls of a
  step that choose the cache pages each new token attends to;
* ``attend``: ``scaled_dot_product_attention_paged_sparse`` over chosen pages.
"""

import math

import numpy as np
import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6
_BASE = 10000.0


def listed():
    """Sizes are those of this repository's own workloads (GQA 32/8 at D 128
    and N 8191, MHA 16 at D 64, decode of 16 x 8,192 and 2 x 65,536 cached
    tokens) and ragged neighbours of them."""
    return [
        # a long-context training step's queries and keys, GQA, weights kept in fp32
        dict(name="rotary gqa d128", kind="rotary", layout="dense", batch=2, tokens=8191, hq=32, hkv=8, d=128, rd=128,
             interleaved=False, norm=True, weights="fp32", dtype="bf16"),
        # MHA training at an odd length, interleaved pairs, weights in the operand type
        dict(name="rotary mha d64 odd", kind="rotary", layout="dense", batch=4, tokens=2049, hq=16, hkv=16, d=64,
             rd=64, interleaved=True, norm=True, weights="fp16", dtype="fp16"),
        # a small packed batch, half of each head rotated: latency counts
        dict(name="rotary packed small", kind="rotary", layout="packed", batch=3, tokens=301, hq=8, hkv=2, d=32,
             rd=16, interleaved=False, norm=True, weights="fp16", dtype="fp16"),
        # one decode step of 16 sequences: latency counts
        dict(name="append decode 16", kind="append", seqs=16, new=1, ctx=2048, page=64, hq=32, hkv=8, d=128, rd=128,
             interleaved=False, norm=True, weights="fp16", dtype="fp16", pad=0),
        # a prefill chunk of four long prompts in a padded batch
        dict(name="append prefill", kind="append", seqs=4, new=4093, ctx=4400, page=64, hq=32, hkv=8, d=128, rd=128,
             interleaved=False, norm=True, weights="bf16", dtype="bf16", pad=12),
        # a decode step's tables for 16 requests: latency counts
        dict(name="tables decode 16", kind="tables", seqs=16, new=1, ctx=8192, page=64, pool=4096, pad=0),
        # admission of many ragged prompts, in small pages, with a padded batch
        dict(name="tables prefill 256", kind="tables", seqs=256, new=2048, ctx=4096, page=16, pool=65536, pad=77),
        # a decode step of 16 sequences of 8,192 cached tokens, a quarter of the pages kept
        dict(name="select 16x8192", kind="select", seqs=16, nq=1, ctx=8192, page=64, hq=32, hkv=8, d=128, top=32,
             dtype="fp16"),
        # fewer and longer sequences in small pages, an eighth of the pages kept
        dict(name="select 8x32768", kind="select", seqs=8, nq=1, ctx=32768, page=16, hq=32, hkv=8, d=128, top=256,
             dtype="bf16"),
        # the attention of the first select case
        dict(name="attend 16x8192", kind="attend", seqs=16, nq=1, ctx=8192, page=64, hq=32, hkv=8, d=128, top=32,
             dtype="fp16"),
        # two long sequences in small pages: 16 (sequence, K/V head) units only
        dict(name="attend 2x65536", kind="attend", seqs=2, nq=1, ctx=65536, page=16, hq=32, hkv=8, d=128, top=512,
             dtype="bf16"),
        # a verification step of several drafted tokens a sequence, a group of 7 heads
        dict(name="attend verify g7 d64", kind="attend", seqs=31, nq=4, ctx=4099, page=32, hq=28, hkv=4, d=64, top=40,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "tables", "select", "attend"])
    d = rng.choice([32, 64, 128])
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 7, 8, 16])
    dt = rng.choice(["fp16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if kind == "rotary":
        heads = hkv * (group + 1)
        tokens = _log(rng, 1, min(8191, 2 * 8191 * 40 * 128 // (heads * d)))
        batch = _log(rng, 1, max(1, min(16, 2 * 8191 * 40 * 128 // (heads * d * tokens))))
        return dict(kind=kind, layout=rng.choice(["dense", "packed"]), batch=batch, tokens=tokens, hq=hkv * group,
                    hkv=hkv, d=d, rd=rng.choice([d, d // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.8, weights=rng.choice([dt, "fp32"]), dtype=dt)
    if kind == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 16384 // seqs))
        return dict(kind=kind, seqs=seqs, new=new, ctx=new + _log(rng, 1, max(2, 16384 // seqs)), page=page,
                    hq=hkv * group, hkv=hkv, d=d, rd=rng.choice([d, d // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.8, weights=rng.choice([dt, "fp32"]), dtype=dt, pad=rng.choice([0, 5]))
    if kind == "tables":
        seqs = _log(rng, 1, 512)
        new = _log(rng, 1, 2048)
        ctx = new + _log(rng, 1, 8192)
        return dict(kind=kind, seqs=seqs, new=new, ctx=ctx, page=page,
                    pool=_log(rng, 64, 2 + seqs * (ctx // page + 2)), pad=rng.choice([0, 31]))
    hq, nq = hkv * group, rng.choice([1, 1, 1, 2, 5])
    seqs = _log(rng, 1, 32)
    ctx = nq + _log(rng, 64, max(128, min(65536, 131072 * 8 * 128 // (seqs * hkv * d * 2))))
    pages = -(-ctx // page)
    top = max(2, _log(rng, 2, max(3, min(512, pages, 16 * 4096 * 8 * 128 // (seqs * nq * hkv * d * page)))))
    return dict(kind=kind, seqs=seqs, nq=nq, ctx=ctx, page=page, hq=hq, hkv=hkv, d=d, top=top, dtype=dt)


# ------------------------------------------------------------------ lengths
def _rs(c):
    return np.random.RandomState(c["ctx"] * 131 + c["seqs"])


def _lens(c):
    """Cached lengths, this step's tokens included, of a ragged batch: the
    first sequence ends a page, the last is the longest."""
    n = _rs(c).randint(max(c["nq"], c["ctx"] // 2), c["ctx"] + 1, c["seqs"])
    n[0] = max(c["nq"], n[0] // c["page"] * c["page"])
    n[-1] = c["ctx"]
    return n.astype(np.int64)


def _request_lens(c):
    """(cached, new) tokens of each request; a prefill step also carries
    requests with nothing new."""
    r = _rs(c)
    if c["new"] == 1:
        new = np.ones(c["seqs"], np.int64)
    else:
        new = r.randint(0, c["new"] + 1, c["seqs"]).astype(np.int64)
        new[-1] = c["new"]
    cached = r.randint(0, c["ctx"] - c["new"] + 1, c["seqs"]).astype(np.int64)
    return cached, new


def _cu(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int64)


def _i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).to(dev)


def _table(c, dev):
    """(max position, rd) fp32: cosines, then sines, of every position's
    angles, from 64-bit angles."""
    rd, n = c["rd"], c["tokens"] if c["kind"] == "rotary" else c["ctx"]
    freq = _BASE ** (-torch.arange(0, rd, 2, dtype=torch.float64, device=dev) / rd)
    ang = torch.arange(n, dtype=torch.float64, device=dev)[:, None] * freq
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "tables":
        return _prepare_tables(c, s, g, dev)
    dt = _DT[c["dtype"]]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    if c["kind"] in ("rotary", "append"):
        s["table"] = _table(c, dev)
        wt = _DT[c["weights"]]
        s["wq"], s["wk"] = ((1 + 0.3 * randn(d, dtype=torch.float32)).to(wt) if c["norm"] else None for _ in range(2))
    if c["kind"] == "rotary":
        b, n = c["batch"], c["tokens"]
        # the fused projection's output, heads behind each other in a token's row
        if c["layout"] == "dense":
            qkv = randn(b, n, hq + 2 * hkv, d)
            s["q"], s["k"] = qkv[:, :, :hq].transpose(1, 2), qkv[:, :, hq:hq + hkv].transpose(1, 2)
            s["pos"] = torch.arange(n, dtype=torch.int32, device=dev)
            s["gq"], s["gk"] = randn(b, hq, n, d), randn(b, hkv, n, d)
        else:
            lens = np.full(b, n // b, np.int64)
            lens[0] += n - lens.sum()
            qkv = randn(n, hq + 2 * hkv, d)
            s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
            s["pos"] = _i32(np.concatenate([np.arange(m) for m in lens]), dev)
            s["gq"], s["gk"] = randn(n, hq, d), randn(n, hkv, d)
        s["leaves"] = []
        for name in ("q", "k", "wq", "wk"):
            if s[name] is not None:
                s[name] = s[name].detach().requires_grad_()
                s["leaves"].append(s[name])
        return s
    if c["kind"] == "append":
        cached, new = _request_lens(c)
        total = int(new.sum()) + c["pad"]
        pages_of = -(-(cached + new) // c["page"])
        n_pages = int(pages_of.sum()) + 2
        perm = torch.randperm(n_pages, generator=g, device=dev)
        first = _cu(pages_of)
        pos = np.concatenate([np.arange(a, a + m) for a, m in zip(cached, new)] + [np.zeros(c["pad"], np.int64)])
        logical = np.concatenate([f + np.arange(a, a + m) // c["page"] for f, a, m in zip(first, cached, new)]
                                 + [np.zeros(c["pad"], np.int64)])
        slots = perm[torch.from_numpy(logical).to(dev)] * c["page"] + torch.from_numpy(pos % c["page"]).to(dev)
        slots[total - c["pad"]:] = -1
        s["slots"], s["pos"] = slots.int(), _i32(pos, dev)
        qkv = randn(total, hq + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["kc"], s["vc"] = (randn(n_pages, c["page"], hkv, d) for _ in range(2))
        return s
    # select, attend: a cache in shuffled pages, and this step's queries, last in their sequences
    lens = _lens(c)
    page, nq = c["page"], c["nq"]
    pages_of = -(-lens // page)
    width, n_pages = int(pages_of.max()), int(pages_of.sum()) + 1
    perm = torch.randperm(n_pages, generator=g, device=dev).int()
    at = torch.from_numpy(_cu(pages_of)[:-1, None] + np.arange(width)[None]).to(dev)
    used = torch.from_numpy(np.arange(width)[None] < pages_of[:, None]).to(dev)
    s["bt"] = torch.where(used, perm[at.clamp(max=n_pages - 1)], 0).int().contiguous()
    s["lens"] = _i32(lens, dev)
    s["cu"] = _i32(np.arange(c["seqs"] + 1) * nq, dev)
    s["q"] = randn(c["seqs"] * nq, hq, d)
    # keys of one page resemble each other, as neighbouring tokens' do
    s["kc"] = randn(n_pages, page, hkv, d).add_(randn(n_pages, 1, hkv, d))
    if c["kind"] == "select":
        s["means"] = _mean64(s["kc"])
        # the page each sequence's new tokens are in has no mean yet
        s["means"][s["bt"].long().gather(1, (s["lens"].long()[:, None] - nq) // page)] = 0
        return s
    s["vc"] = randn(n_pages, page, hkv, d)
    own_page = (s["lens"].long().repeat_interleave(nq) - nq
                + torch.arange(nq, device=dev).repeat(c["seqs"])) // page
    r = torch.rand(c["seqs"] * nq, hkv, width, generator=g, device=dev)
    p = torch.arange(width, device=dev)
    r = torch.where(p == own_page[:, None, None], 2.0, torch.where(p < own_page[:, None, None], r, -1.0))
    v, i = r.topk(min(c["top"], width), dim=-1)
    i = torch.where(v >= 0, i, width).sort(-1).values
    s["idx"] = torch.where(i < width, i, -1).int().contiguous()
    return s


def _prepare_tables(c, s, g, dev):
    cached, new = _request_lens(c)
    s["cached"], s["new"] = _i32(cached, dev), _i32(new, dev)
    have = -(-cached // c["page"])
    width = -(-c["ctx"] // c["page"])
    n_used = int(have.sum())
    perm = torch.randperm(n_used + c["pool"] + 3, generator=g, device=dev).int()
    at = torch.from_numpy(_cu(have)[:-1, None] + np.arange(width)[None]).to(dev)
    used = torch.from_numpy(np.arange(width)[None] < have[:, None]).to(dev)
    s["bt"] = torch.where(used, perm[at.clamp(max=perm.numel() - 1)], -1).int().contiguous()
    s["free"] = perm[n_used:].contiguous()
    s["start"] = torch.tensor([3], dtype=torch.int32, device=dev)
    s["total"] = int(new.sum()) + c["pad"]
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["kind"]](state)


def _run_own(s):
    import triton_flash_attention_b200 as fa

    c = s["case"]
    kind = c["kind"]
    if kind == "rotary":
        q, k = fa.qk_norm_rotary(s["q"], s["k"], s["table"], s["pos"], query_weight=s["wq"], key_weight=s["wk"],
                                 eps=_EPS, interleaved=c["interleaved"])
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), s["leaves"], (s["gq"], s["gk"]))]
    if kind == "append":
        q = fa.paged_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["table"], s["pos"],
                            query_weight=s["wq"], key_weight=s["wk"], eps=_EPS, interleaved=c["interleaved"])
        return [q[:q.shape[0] - c["pad"]], s["kc"], s["vc"]]
    if kind == "tables":
        r = fa.extend_block_table(s["bt"], s["cached"], s["new"], s["free"], s["start"], page_size=c["page"],
                                  total_q=s["total"])
        return [s["bt"], r.cu_seqlens_q, r.seqlens_k, r.positions, r.slot_mapping, r.fits, r.free_next]
    if kind == "select":
        fa.update_page_means(s["kc"], s["means"], s["bt"], s["cu"], s["lens"])
        idx = fa.select_pages(s["q"], s["means"], s["bt"], s["cu"], s["lens"], page_size=c["page"],
                              num_selected=c["top"], sink_pages=1, local_pages=1)
        return [s["means"], idx]
    return fa.scaled_dot_product_attention_paged_sparse(s["q"], s["kc"], s["vc"], s["bt"], s["cu"], s["lens"],
                                                        s["idx"], enable_gqa=True)


# ------------------------------------------------------------------ plain forms
def _rotate(y, table, pos, c, back=False):
    """Rotation of the first rd columns of y (..., d) by its row's angles;
    pos broadcasts to y's leading sizes.  ``back`` turns the other way."""
    rd = c["rd"]
    t = table[pos.long()].to(y.dtype)
    cos, sin = t[..., :rd // 2], t[..., rd // 2:]
    sin = -sin if back else sin
    x = y[..., :rd]
    if c["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        z = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:]
        z = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([z, y[..., rd:]], -1)


def _pos_of(s):
    """Positions against (batch, heads, tokens) or (total, heads)."""
    return s["pos"][:, None] if s["q"].ndim == 3 else s["pos"]


def _norm(x, w):
    if w is None:
        return x, None
    r = (x.square().mean(-1, keepdim=True) + _EPS).rsqrt()
    return x * r * w.to(x.dtype), r


def _plain_rotary(s):
    c, pos, t = s["case"], _pos_of(s), s["table"]

    def forward(x, w):
        return _rotate(_norm(x.float(), w)[0], t, pos, c).to(x.dtype)

    def backward(x, w, gz):
        gy = _rotate(gz.float(), t, pos, c, back=True)
        if w is None:
            return gy.to(x.dtype), None
        xf = x.float()
        _, r = _norm(xf, w)
        gw = (gy * xf * r).sum(tuple(range(x.ndim - 1)), dtype=torch.float64)
        gn = gy * w.float()
        return (r * (gn - xf * r * r * (gn * xf).mean(-1, keepdim=True))).to(x.dtype), gw.to(w.dtype)

    dq, dwq = backward(s["q"], s["wq"], s["gq"])
    dk, dwk = backward(s["k"], s["wk"], s["gk"])
    out = [forward(s["q"], s["wq"]), forward(s["k"], s["wk"]), dq, dk]
    return out if dwq is None else out + [dwq, dwk]


def _plain_append(s):
    c, pos, t = s["case"], _pos_of(s), s["table"]
    n = s["q"].shape[0] - c["pad"]
    q, k = (_rotate(_norm(x[:n].float(), w)[0], t, pos[:n], c).to(x.dtype)
            for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])))
    at = s["slots"][:n].long()
    s["kc"].view(-1, c["hkv"], c["d"])[at] = k
    s["vc"].view(-1, c["hkv"], c["d"])[at] = s["v"][:n]
    return [q, s["kc"], s["vc"]]


def _plain_tables(s):
    c, page, dev = s["case"], s["case"]["page"], s["bt"].device
    cached, new, bt = s["cached"].long(), s["new"].long(), s["bt"]
    width, total = bt.shape[1], s["total"]
    have, want = (cached + page - 1) // page, (cached + new + page - 1) // page
    ends = new.cumsum(0)
    placed = (want <= width) & (ends <= total)
    need = torch.where(placed, want - have, 0)
    upto = need.cumsum(0)
    start = s["start"].long()
    fits = placed & (upto <= s["free"].numel() - start)
    first = upto - need
    col = torch.arange(width, device=dev)
    fresh = fits[:, None] & (col >= have[:, None]) & (col < want[:, None])
    at = (start + first[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    bt.copy_(torch.where(fresh, s["free"][at], bt))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), ends]).clamp(max=total)
    row = torch.arange(total, device=dev)
    req = torch.searchsorted(ends, row, right=True)
    real = req < len(new)
    r = req.clamp(max=len(new) - 1)
    pos = torch.where(real, cached[r] + row - cu[r], 0)
    slot = bt[r, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    slot = torch.where(real & fits[r], slot, -1)
    used = torch.where(fits, upto, 0).max()
    return [bt, cu.int(), torch.where(fits, cached + new, cached).int(), pos.int(), slot.int(), fits,
            (start + used).int()]


def _mean64(pages):
    """Mean over the keys of whole pages, summed in 64 bits: the pages are
    ranked by it, so neither side may round it on the way."""
    return pages.double().mean(1).float().to(pages.dtype)


def _plain_select(s):
    c, page, dev = s["case"], s["case"]["page"], s["bt"].device
    hkv, nq, top = c["hkv"], c["nq"], c["top"]
    bt, lens = s["bt"].long(), s["lens"].long()
    width = bt.shape[1]
    # pages that the step's tokens completed: a step of nq tokens ends nq // page + 1 pages at most
    cand = (lens - nq)[:, None] // page + torch.arange(nq // page + 1, device=dev)
    done = cand < lens[:, None] // page
    phys = bt.gather(1, cand.clamp(max=width - 1))
    spare = s["means"].shape[0] - 1
    flat = torch.where(done, phys, phys.gather(1, torch.zeros_like(phys)).clamp(max=spare)).flatten()
    s["means"][flat] = torch.where(done.flatten()[:, None, None], _mean64(s["kc"][flat]), s["means"][flat])
    # scores in 64 bits: values next to the border decide which pages are kept
    q = s["q"].double().view(c["seqs"], nq, hkv, -1, c["d"])
    m = s["means"][bt].double()  # (seqs, width, hkv, d)
    score = torch.einsum("bqhgd,bphd->bqhgp", q, m).amax(3).float()
    own_page = ((lens - nq)[:, None] + torch.arange(nq, device=dev)) // page
    p = torch.arange(width, device=dev)
    o = own_page[:, :, None, None]
    forced = (p < 1) | (p > o - 1)
    score = torch.where(p > o, -math.inf, torch.where(forced, math.inf, score))
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    kept = torch.where(order <= o, order, width).sort(-1).values
    kept = torch.where(kept < width, kept, -1)
    pad = torch.full((*kept.shape[:-1], max(0, top - width)), -1, device=dev)
    return [s["means"], torch.cat([kept, pad], -1).view(c["seqs"] * nq, hkv, top).int()]


def _plain_attend(s):
    c, page, dev = s["case"], s["case"]["page"], s["bt"].device
    hkv, nq, d = c["hkv"], c["nq"], c["d"]
    t = c["seqs"] * nq
    idx = s["idx"].long()
    seq = torch.arange(t, device=dev) // nq
    last = s["lens"].long()[seq] - nq + torch.arange(t, device=dev) % nq
    phys = s["bt"].long()[seq[:, None, None], idx.clamp(min=0)]
    h = torch.arange(hkv, device=dev)[None, :, None]
    key = idx[..., None] * page + torch.arange(page, device=dev)
    seen = ((idx[..., None] >= 0) & (key <= last[:, None, None, None])).flatten(2)
    k = s["kc"].permute(0, 2, 1, 3)[phys, h].flatten(2, 3).float()
    v = s["vc"].permute(0, 2, 1, 3)[phys, h].flatten(2, 3).float()
    q = s["q"].float().view(t, hkv, -1, d)
    score = (q @ k.transpose(-1, -2)) * d ** -0.5
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    w = (score - score.amax(-1, keepdim=True)).exp()
    return ((w @ v) / w.sum(-1, keepdim=True)).view(t, -1, d).to(s["q"].dtype)


_PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "tables": _plain_tables, "select": _plain_select,
          "attend": _plain_attend}


# ------------------------------------------------------------------ 64 bits
def _turned(x, w, pos, c, sign):
    """Norm (with w) and rotation in 64 bits as one linear map a row, through
    complex numbers: pair (a, b) is a + ib, turned by the angle itself."""
    rd = c["rd"]
    x = x.double()
    if w is not None:
        x = w.double() * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt()
    f = torch.pow(torch.tensor(_BASE, dtype=torch.float64, device=x.device),
                  -2.0 * torch.arange(rd // 2, dtype=torch.float64, device=x.device) / rd)
    ang = sign * pos.double()[..., None] * f
    if c["interleaved"]:
        z = torch.view_as_complex(x[..., :rd].unflatten(-1, (rd // 2, 2)).contiguous())
    else:
        z = torch.complex(x[..., :rd // 2].contiguous(), x[..., rd // 2:rd].contiguous())
    z = z * torch.polar(torch.ones_like(ang), ang)
    parts = torch.view_as_real(z)
    turned = parts.flatten(-2) if c["interleaved"] else parts.transpose(-1, -2).flatten(-2)
    return torch.cat([turned, x[..., rd:]], -1)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    with torch.no_grad():
        if c["kind"] == "rotary":
            pos = _pos_of(s)
            out, grads, wgrads = [], [], []
            for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
                out.append(_turned(x, w, pos, c, 1.0))
                gy = _turned(g, None, pos, c, -1.0)
                if w is None:
                    grads.append(gy)
                    continue
                xd = x.double()
                rms = (xd.pow(2).sum(-1, keepdim=True) / c["d"] + _EPS).sqrt()
                unit = xd / rms
                wgrads.append(torch.einsum("...d,...d->d", gy, unit))
                gy = gy * w.double()
                grads.append((gy - unit * (gy * unit).sum(-1, keepdim=True) / c["d"]) / rms)
            return out + grads + wgrads
        if c["kind"] == "append":
            n = s["q"].shape[0] - c["pad"]
            pos, at = _pos_of(s)[:n], s["slots"][:n].long()
            kc, vc = s["kc"].double(), s["vc"].double()
            kc.view(-1, c["hkv"], c["d"]).index_copy_(0, at, _turned(s["k"][:n], s["wk"], pos, c, 1.0))
            vc.view(-1, c["hkv"], c["d"]).index_copy_(0, at, s["v"][:n].double())
            return [_turned(s["q"][:n], s["wq"], pos, c, 1.0), kc, vc]
        if c["kind"] == "select":
            means = s["means"].double()
            first, lens = (s["lens"].long() - c["nq"]) // c["page"], s["lens"].long()
            ended = torch.nonzero(lens // c["page"] > first).flatten()
            at = s["bt"][ended, first[ended]].long()
            means[at] = s["kc"][at].double().sum(1) / c["page"]
            return [means, None]
        if c["kind"] == "attend":
            return _exact_attend(c, s)
    return None


def _exact_attend(c, s):
    """Dense attention in 64 bits over each sequence's cache, with every page
    that is not listed hidden; one K/V head at a time."""
    page, nq, dev = c["page"], c["nq"], s["bt"].device
    lens = s["lens"].long()
    group = c["hq"] // c["hkv"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=dev)
    for b in range(c["seqs"]):
        n = int(lens[b])
        pages = s["bt"][b, :-(-n // page)].long()
        for h in range(c["hkv"]):
            k, v = (x[pages, :, h].reshape(-1, c["d"])[:n].double() for x in (s["kc"], s["vc"]))
            for i in range(nq):
                t = b * nq + i
                idx = s["idx"][t, h].long()
                keep = torch.zeros(len(pages), dtype=torch.bool, device=dev)
                keep[idx[idx >= 0]] = True
                keep = keep.repeat_interleave(page)[:n] & (torch.arange(n, device=dev) <= n - nq + i)
                q = s["q"][t, h * group:(h + 1) * group].double()
                a = (q @ k.T / math.sqrt(c["d"])).masked_fill(~keep, -math.inf).softmax(-1)
                out[t, h * group:(h + 1) * group] = a @ v
    return out


# ------------------------------------------------------------------ work
def work(case):
    c = case
    if c["kind"] == "rotary":
        rows = c["tokens"] * (c["batch"] if c["layout"] == "dense" else 1)
        elems = rows * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": 4 * 2 * elems + 4 * c["tokens"] * c["rd"], "flops": 22 * elems}
    if c["kind"] == "append":
        rows = int(_request_lens(c)[1].sum())
        elems = rows * c["d"]
        return {"bytes": 4 * elems * (c["hq"] + 2 * c["hkv"]) + 4 * rows * c["rd"],
                "flops": 8 * elems * (c["hq"] + c["hkv"])}
    if c["kind"] == "tables":
        cached, new = _request_lens(c)
        pages = -(-(cached + new) // c["page"]) - -(-cached // c["page"])
        rows = int(new.sum()) + c["pad"]
        return {"bytes": 8 * rows + 8 * int(pages.sum()) + 17 * c["seqs"], "flops": 4 * rows}
    lens, rows = _lens(c), c["seqs"] * c["nq"]
    pages = -(-lens // c["page"])
    if c["kind"] == "select":
        seen = int(pages.sum())
        ended = int((lens // c["page"] - (lens - c["nq"]) // c["page"]).sum())
        return {"bytes": 2 * c["hkv"] * c["d"] * (seen + ended * (c["page"] + 1)) + 2 * rows * c["hq"] * c["d"]
                + 4 * rows * c["hkv"] * c["top"], "flops": 2 * c["nq"] * seen * c["hq"] * c["d"]}
    kept = np.minimum(pages, c["top"])
    union = pages * (1 - (1 - kept / pages) ** c["nq"])  # pages that some token of the sequence reads
    return {"bytes": 4 * c["hkv"] * c["d"] * c["page"] * float(union.sum()) + 4 * rows * c["hq"] * c["d"],
            "flops": 4 * c["nq"] * float(kept.sum()) * c["page"] * c["hq"] * c["d"]}
