"""Norm and rotation of queries and keys (``qk_norm_rotary``) against float64.

Tolerances, from the arithmetic: with u half a step of the operand type
(2^-11 fp16, 2^-8 bf16) a result z is rounded once, u |z| (and 2^-25 for fp16
below its smallest normal number).  Before that, in fp32: the sum of D <= 128
squares in runs of 16 and a tree, its root and the products are within some
20 roundings of 2^-24 and the root's 2 of 2^-23, below 2^-19 of the rotation's
two terms |y_a| + |y_b| <= sum of both.  Gradients likewise, of the sums of
their terms' sizes; a weight's gradient sums its rows in chains of at most
some hundred here: 2^-16 of the sum of sizes.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import triton_flash_attention_b200 as fa
from oracle import fa2_oracle as orc
from triton_flash_attention_b200 import _abi

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _f64(t):
    return t.detach().double().cpu().numpy()


def _pair_size(y, rd, interleaved):
    """|y_a| + |y_b| at both columns of each pair, |y| behind them."""
    a = np.abs(y)
    s = a.copy()
    i, j = (slice(0, rd, 2), slice(1, rd, 2)) if interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    s[..., i] = s[..., j] = a[..., i] + a[..., j]
    return s


def _assert_close(got, want, slack, dtype, what):
    tol = _half_step(dtype) * np.abs(want) * (1 + 1e-3) + slack + (2.0 ** -25 if dtype == F16 else 1e-30)
    diff = np.abs(_f64(got) - want)
    assert (diff <= tol).all(), (what, float((diff - tol).max()), int((diff > tol).sum()))


def _check(x, w, table, pos, eps, interleaved, z, gz=None, dx=None, dw=None):
    """x, z, gz, dx: packed (tokens, heads, D) tensors; pos: numpy."""
    dt, rd = x.dtype, table.shape[1]
    ref = orc.norm_rotary_reference(_f64(x), None if w is None else _f64(w), table.cpu().numpy(), pos, eps,
                                    interleaved, None if gz is None else _f64(gz))
    x64 = _f64(x)
    r = 1.0 if w is None else 1 / np.sqrt((x64 ** 2).mean(-1, keepdims=True) + eps)
    y = x64 if w is None else x64 * r * _f64(w)
    _assert_close(z, ref["z"], 2.0 ** -19 * _pair_size(y, rd, interleaved), dt, "z")
    if gz is None:
        return
    dy = _pair_size(_f64(gz), rd, interleaved)
    if w is None:
        _assert_close(dx, ref["dx"], 2.0 ** -19 * dy, dt, "dx")
        return
    g = dy * np.abs(_f64(w))
    size = r * (g + np.abs(x64) * r * r * (g * np.abs(x64)).mean(-1, keepdims=True))
    _assert_close(dx, ref["dx"], 2.0 ** -18 * size, dt, "dx")
    if dw is not None:
        _assert_close(dw, ref["dw"], 2.0 ** -16 * (dy * np.abs(x64) * r).sum((0, 1)), dw.dtype, "dw")


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype)


def _packed(t):
    """(B, H, N, D) as (B * N, H, D)."""
    return t.transpose(1, 2).reshape(-1, t.shape[1], t.shape[3])


# ---------------------------------------------------------------- CPU
def test_oracle_gradient_is_the_formulas_difference_quotient():
    rng = np.random.default_rng(0)
    x, w, gz = rng.standard_normal((3, 2, 32)), rng.standard_normal(32), rng.standard_normal((3, 2, 32))
    table = fa.rotary_table(9, 16).numpy()
    pos = np.array([0, 5, 8])
    for inter in (False, True):
        def loss(x, w):
            return (orc.norm_rotary_reference(x, w, table, pos, 1e-6, inter)["z"] * gz).sum()

        ref = orc.norm_rotary_reference(x, w, table, pos, 1e-6, inter, gz)
        for _ in range(6):
            dx, dw = rng.standard_normal(x.shape), rng.standard_normal(w.shape)
            h = 1e-6
            diff = (loss(x + h * dx, w + h * dw) - loss(x - h * dx, w - h * dw)) / (2 * h)
            want = (ref["dx"] * dx).sum() + (ref["dw"] * dw).sum()
            # h^2 of the third derivative and 1e-16 / h of the loss, each some 1e-9
            assert abs(diff - want) < 1e-6 * (1 + abs(want))


def test_rotary_table():
    t = fa.rotary_table(100_000, 64, base=500_000.0)
    assert t.shape == (100_000, 64) and t.dtype == F32
    p = np.array([0, 1, 77_777, 99_999], np.float64)[:, None]
    ang = p * 500_000.0 ** (-np.arange(32) / 32)
    want = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    # the angle's own 64-bit rounding, 1e5 * 2^-52, and the result's rounding to fp32
    assert np.abs(t.numpy()[[0, 1, 77_777, 99_999]] - want).max() <= 2.0 ** -25 + 1e-10
    for bad in ((0, 16), (4, 0), (4, 24), (True, 16), (4.0, 16)):
        with pytest.raises(ValueError):
            fa.rotary_table(*bad)
    with pytest.raises(ValueError, match="base"):
        fa.rotary_table(4, 16, base=float("nan"))


def test_refusals_on_cpu():
    q, k = torch.randn(2, 4, 5, 32).half(), torch.randn(2, 2, 5, 32).half()
    t = fa.rotary_table(8, 32)
    with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
        fa.qk_norm_rotary(q, k, t)
    with pytest.raises(TypeError, match="query must be a torch.Tensor"):
        fa.qk_norm_rotary(q.numpy(), k, t)
    for bad, message in [
        ((q[0, 0], k, t), "must have shape"),
        ((q[0], k, t), "same layout"),
        ((q, k[:1], t), "batch and sequence"),
        ((q, k[:, :, :4], t), "batch and sequence"),
        ((q[:, :, :0], k, t), "greater than zero"),
        ((q, k.float(), t), "same dtype"),
        ((q[..., :16], k, t), "head dimensions must match"),
        ((q[0], k[0, :, :3].contiguous(), t), "number of rows"),
        ((q, k, t.double()), "float32"),
        ((q, k, t[0]), "float32"),
        ((q, k, fa.rotary_table(8, 48)), "rotary_dim"),
        ((q, k, t[:, :16]), "contiguous"),
        ((q, k, t[:, :24].contiguous()), "rotary_dim"),
        ((q, k, t, torch.arange(5)), "positions must be an int32"),
        ((q, k, t, torch.arange(4, dtype=torch.int32)), "positions must be an int32"),
        ((q[0], k[0, :1].expand(4, 5, 32), t), "need positions"),
    ]:
        with pytest.raises(ValueError, match=message):
            fa.qk_norm_rotary(*bad)
    w = torch.ones(32)
    for kw, message in [
        (dict(query_weight=w), "both query_weight and key_weight"),
        (dict(query_weight=w, key_weight=w[:16]), "head_dim weights"),
        (dict(query_weight=w, key_weight=w.half()), "same dtype"),
        (dict(query_weight=w.double(), key_weight=w.double()), "query's dtype or float32"),
        (dict(eps=-1.0), "eps"),
        (dict(eps=float("inf")), "eps"),
    ]:
        with pytest.raises(ValueError, match=message):
            fa.qk_norm_rotary(q, k, t, **kw)
    with pytest.raises(TypeError, match="interleaved"):
        fa.qk_norm_rotary(q, k, t, interleaved=1)


def test_abi_refuses_before_any_cuda_call():
    lib, p = _abi.lib(), 16
    s = _abi.strides_of((4096, 64, 64))
    odd = _abi.strides_of((4096, 63, 64))
    zero = _abi.strides_of((4096, 0, 64))

    def fwd(b=1, hq=4, hkv=2, n=8, d=64, rd=64, wq=p, wk=p, qs=s, qo=s, q=p, table=p, eps=1e-6, pos_sb=0):
        return lib.fa_qk_norm_rotary(q, p, p, p, table, p, wq, wk, b, hq, hkv, n, d, 8, rd, 0, 0, qs, s, qo, s,
                                     pos_sb, eps, None)

    assert fwd(d=48) == _abi.FA_ERR_UNSUPPORTED_HEAD_DIM
    for bad in (dict(b=0), dict(n=-1), dict(hq=0), dict(rd=0), dict(rd=24), dict(rd=128), dict(wk=None),
                dict(q=None), dict(table=None), dict(eps=float("nan")), dict(eps=-1.0), dict(pos_sb=-1),
                dict(b=1 << 20, n=1 << 20)):
        assert fwd(**bad) == _abi.FA_ERR_BAD_SHAPE, bad
    for bad in (dict(qs=odd), dict(qo=odd), dict(qo=zero), dict(q=18), dict(table=20)):
        assert fwd(**bad) == _abi.FA_ERR_MISALIGNED, bad
    # backward: weight gradients come in twos and want scratch and weights
    def bwd(dwq=p, dwk=p, part=p, wq=p, wk=p):
        return lib.fa_qk_norm_rotary_bwd(p, p, p, p, p, p, dwq, dwk, part, p, p, wq, wk, 1, 4, 2, 8, 48, 8, 32, 0, 0,
                                         s, s, s, s, s, s, 0, 1e-6, None)
    assert bwd() == _abi.FA_ERR_UNSUPPORTED_HEAD_DIM
    for bad in (dict(dwk=None), dict(part=None), dict(wq=None, wk=None)):
        assert bwd(**bad) == _abi.FA_ERR_BAD_SHAPE, bad


# ---------------------------------------------------------------- GPU
CASES = [
    # b, n, hq, hkv, d, rd, interleaved, norm, weights, dtype
    (1, 1, 1, 1, 32, 32, False, True, F16, F16),
    (2, 7, 4, 2, 64, 64, False, True, F32, F16),
    (3, 33, 5, 1, 128, 128, False, True, BF16, BF16),
    (1, 129, 8, 8, 128, 64, False, True, F32, BF16),
    (2, 65, 7, 7, 64, 32, True, True, F16, F16),
    (1, 50, 6, 3, 32, 16, True, False, None, BF16),
    (2, 31, 9, 3, 128, 96, True, True, BF16, BF16),
    (2, 31, 16, 1, 128, 48, False, False, None, F16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,hq,hkv,d,rd,interleaved,norm,wdt,dt", CASES)
@pytest.mark.parametrize("layout", ["dense", "projection", "packed"])
def test_forward_and_backward(b, n, hq, hkv, d, rd, interleaved, norm, wdt, dt, layout):
    g = torch.Generator().manual_seed(b * 1000 + n * 10 + d)
    table = fa.rotary_table(n + 40, rd)
    wq, wk = ((1 + 0.5 * _randn(g, d)).to(wdt) if norm else None for _ in range(2))
    x = _randn(g, b, n, hq + 2 * hkv, d, dtype=dt)
    q, k = x[:, :, :hq], x[:, :, hq:hq + hkv]
    gq, gk = _randn(g, b, hq, n, d, dtype=dt), _randn(g, b, hkv, n, d, dtype=dt)
    pos = torch.stack([torch.randperm(n + 40, generator=g)[:n] for _ in range(b)]).int()

    def cuda(t):
        return None if t is None else t.cuda()

    xc = x.cuda()
    if layout == "packed":
        xc = xc.view(b * n, hq + 2 * hkv, d)
        qc, kc, pc = xc[:, :hq], xc[:, hq:hq + hkv], pos.reshape(-1).cuda()
        gqc, gkc = _packed(gq).cuda(), _packed(gk).cuda()
    else:
        qc, kc = xc[:, :, :hq].transpose(1, 2), xc[:, :, hq:hq + hkv].transpose(1, 2)
        if layout == "dense":
            qc, kc = qc.contiguous(), kc.contiguous()
        pc, gqc, gkc = pos.cuda(), gq.cuda(), gk.cuda()
    leaves = [t.detach().requires_grad_() for t in (qc, kc)]
    weights = [cuda(w).requires_grad_() if norm else None for w in (wq, wk)]
    zq, zk = fa.qk_norm_rotary(*leaves, table.cuda(), pc, query_weight=weights[0], key_weight=weights[1], eps=1e-5,
                               interleaved=interleaved)
    grads = torch.autograd.grad((zq, zk), leaves + [w for w in weights if norm], (gqc, gkc))
    assert zq.is_contiguous() and zk.is_contiguous() and zq.dtype == dt
    as_packed = (lambda t: t) if layout == "packed" else _packed
    for i, (src, w, z, gz) in enumerate(((q, wq, zq, gq), (k, wk, zk, gk))):
        _check(src.reshape(b * n, -1, d), w, table, pos.reshape(-1).numpy(), 1e-5, interleaved, as_packed(z),
               _packed(gz), as_packed(grads[i]), grads[2 + i] if norm else None)
    assert _abi.device_status() == 0


@pytest.mark.gpu
def test_default_positions_shared_positions_and_broadcast_inputs():
    g = torch.Generator().manual_seed(5)
    b, n, hq, d = 3, 21, 4, 64
    table = fa.rotary_table(64, 64).cuda()
    q = _randn(g, b, hq, n, d, dtype=F16).cuda()
    k1 = _randn(g, 1, 1, n, d, dtype=F16).cuda().requires_grad_()
    k = k1.expand(b, 2, n, d)  # strides of zero
    w = torch.ones(d).cuda()
    ar = torch.arange(n, dtype=torch.int32).cuda()
    outs = [fa.qk_norm_rotary(q, k, table, p, query_weight=w, key_weight=w) for p in (None, ar, ar.expand(b, n))]
    for zq, zk in outs[1:]:
        assert torch.equal(zq, outs[0][0]) and torch.equal(zk, outs[0][1])
    gz = _randn(g, b, 2, n, d, dtype=F16).cuda()
    dk1, = torch.autograd.grad(outs[0][1], k1, gz)
    ref = orc.norm_rotary_reference(_f64(_packed(k)), np.ones(d), table.cpu().numpy(), np.tile(np.arange(n), b), 1e-6,
                                    False, _f64(_packed(gz)))
    want = ref["dx"].reshape(b, n, 2, d).sum((0, 2))
    # each of the 6 gradients is rounded once, and so is their sum
    tol = _half_step(F16) * 2 * np.abs(ref["dx"]).reshape(b, n, 2, d).sum((0, 2)) + 2.0 ** -16 * 6
    assert (np.abs(_f64(dk1)[0, 0] - want) <= tol).all()


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient():
    """The kernels' own forward, differenced in float64 along a direction:
    outputs are rounded to fp16 (2^-11 each), so the quotient with a step of
    2^-3 is compared within the root-mean-square of that noise."""
    g = torch.Generator().manual_seed(6)
    n, d = 64, 64
    table = fa.rotary_table(n, d).cuda()
    pos = torch.arange(n, dtype=torch.int32).cuda()
    q = _randn(g, n, 8, d, dtype=F16).cuda().requires_grad_()
    w = (1 + 0.3 * _randn(g, d)).cuda().requires_grad_()
    gz = _randn(g, n, 8, d, dtype=F16).cuda()
    v = _randn(g, n, 8, d, dtype=F16).cuda()

    def f(x, wt):
        return fa.qk_norm_rotary(x, x, table, pos, query_weight=wt, key_weight=wt)[0]

    dq, dw = torch.autograd.grad(f(q, w), (q, w), gz)
    h = 0.125
    with torch.no_grad():
        up, down = (f((q.double() + s * h * v.double()).half(), w).double() for s in (1, -1))
    quotient = float(((up - down) * gz.double()).sum() / (2 * h))
    want = float((dq.double() * v.double()).sum())
    # noise: 2^16 values, each off by 2^-11 of a value near 1 twice over 2 h, against g of size 1, in quadrature;
    # curvature: the norm's third derivative is of size 1 / D of the first a row, h^2 of it
    noise = 6 * 2.0 ** -11 * (n * 8 * d) ** 0.5 / (2 * h) * 2 ** 0.5
    curve = h * h * float((dq.double().abs() * v.double().abs()).sum()) * 4 / d
    assert abs(quotient - want) < noise + curve
    with torch.no_grad():
        up, down = (f(q, w + s * 0.25).double() for s in (1, -1))  # linear in w
    quotient = float(((up - down) * gz.double()).sum() / 0.5)
    noise = 6 * 2.0 ** -11 * (n * 8 * d) ** 0.5 / 0.5 * 2 ** 0.5
    assert abs(quotient - float(dw.double().sum())) < noise


@pytest.mark.gpu
def test_special_values_and_positions_out_of_range():
    table = fa.rotary_table(8, 32).cuda()
    q = torch.zeros(6, 2, 64, dtype=BF16).cuda()
    q[1] = float("inf")
    q[2] = float("nan")
    q[3] = 3e38
    q[4], q[5] = 1.0, 1.0
    w = torch.ones(64).cuda()
    pos = torch.tensor([0, 1, 2, 3, -1, 8], dtype=torch.int32).cuda()
    assert _abi.device_status(reset=True) == 0
    z, _ = fa.qk_norm_rotary(q, q, table, pos, query_weight=w, key_weight=w)
    assert (z[0] == 0).all()  # eps keeps a zero row finite
    assert z[2].isnan().all()
    assert z[4:, :, :32].isnan().all() and (z[4:, :, 32:] == 1).all()
    status = _abi.device_status(reset=True)
    assert status & 0xff == _abi.FA_ERR_BAD_INDEX and "out of range" in _abi.status_string(status)
    assert _abi.device_status() == 0


@pytest.mark.gpu
def test_repeats_bit_for_bit_on_another_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(7)
    n = 777
    table = fa.rotary_table(n, 128).cuda()
    pos = torch.arange(n, dtype=torch.int32).cuda()
    q, k = _randn(g, n, 8, 128, dtype=BF16).cuda(), _randn(g, n, 2, 128, dtype=BF16).cuda()
    gq, gk = _randn(g, n, 8, 128, dtype=BF16).cuda(), _randn(g, n, 2, 128, dtype=BF16).cuda()
    w = (1 + 0.3 * _randn(g, 128)).cuda()

    def step():
        z = fa.qk_norm_rotary_forward(q, k, table, pos, w, w, 1e-6, False)
        return z + fa.qk_norm_rotary_backward(q, k, gq, gk, table, pos, w, w, 1e-6, False)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    graph.replay()
    torch.cuda.synchronize()
    for other in (second, third):
        assert all(torch.equal(a, b) for a, b in zip(first, other))


@pytest.mark.gpu
def test_training_step_with_the_attention():
    """Projection, norm and rotation, attention and back, against float64
    autograd of the same formulas.  Bars are the dense attention's (O 2e-3,
    gradients 1e-2), the gradients scaled by their largest value."""
    from torch.nn.functional import scaled_dot_product_attention as sdpa

    g = torch.Generator().manual_seed(8)
    b, n, hq, hkv, d = 2, 193, 4, 2, 64
    x = _randn(g, b, n, hq + 2 * hkv, d, dtype=F16).cuda().requires_grad_()
    wq, wk = ((1 + 0.3 * _randn(g, d)).cuda().requires_grad_() for _ in range(2))
    do = _randn(g, b, hq, n, d, dtype=F16).cuda()
    table = fa.rotary_table(n, d).cuda()

    def split(t):
        return [p.transpose(1, 2) for p in t.split([hq, hkv, hkv], dim=2)]

    q, k, v = split(x)
    q, k = fa.qk_norm_rotary(q, k, table, query_weight=wq, key_weight=wk)
    o = fa.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
    got = torch.autograd.grad(o, (x, wq, wk), do)

    x64, wq64, wk64 = (t.detach().double().requires_grad_() for t in (x, wq, wk))
    cos, sin = table.double()[:, :d // 2], table.double()[:, d // 2:]

    def prep(t, w):
        y = t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, c = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * cos - c * sin, c * cos + a * sin], -1)

    q64, k64, v64 = split(x64)
    o64 = sdpa(prep(q64, wq64), prep(k64, wk64), v64, is_causal=True, enable_gqa=True)
    want = torch.autograd.grad(o64, (x64, wq64, wk64), do.double())
    assert float((o.double() - o64).abs().max()) <= 4e-3  # 2e-3, and q and k rounded on the way
    for a, r in zip(got, want):
        assert float((a.double() - r).abs().max()) <= 1e-2 * max(1.0, float(r.abs().max()))


@pytest.mark.gpu
def test_a_gradient_of_the_gradient_is_refused():
    q = torch.randn(4, 2, 32, device="cuda").half().requires_grad_()
    table, pos = fa.rotary_table(4, 32).cuda(), torch.arange(4, dtype=torch.int32).cuda()
    z, _ = fa.qk_norm_rotary(q, q, table, pos)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(z.float().sum(), q, create_graph=True)


@pytest.mark.gpu
def test_rows_that_cannot_be_read_in_place_are_copied():
    """Rows off the 16-byte boundary, odd strides and a transposed head
    dimension give what contiguous rows give, forward and backward."""
    g = torch.Generator().manual_seed(9)
    table, pos = fa.rotary_table(50, 64).cuda(), torch.arange(50, dtype=torch.int32).cuda()
    w = torch.rand(64, generator=g).cuda()
    base = _randn(g, 50, 4, 64, dtype=F16).cuda()
    wide = torch.zeros(50, 4, 67, dtype=F16, device="cuda")
    wide[:, :, 3:] = base
    shifted = torch.zeros(base.numel() + 1, dtype=F16, device="cuda")
    shifted[1:] = base.flatten()
    views = [wide[:, :, 3:], shifted[1:].view(50, 4, 64), base.transpose(1, 2).contiguous().transpose(1, 2)]
    gz = _randn(g, 50, 4, 64, dtype=F16).cuda()

    def step(x, gz):
        x = x.detach().requires_grad_()
        z = fa.qk_norm_rotary(x, x, table, pos, query_weight=w, key_weight=w)[0]
        return z.detach(), torch.autograd.grad(z, x, gz)[0]

    want = step(base, gz)
    for v in views:
        got = step(v, gz.transpose(1, 2).contiguous().transpose(1, 2))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    z = fa.qk_norm_rotary(base, base, table, pos)[0]
    assert torch.equal(z.expand(1, 50, 4, 64)[0], z)


@pytest.mark.gpu
def test_saved_tensors_may_come_back_laid_out_otherwise():
    """Queries and keys are views of a fused projection; hooks on the saved
    tensors give them back contiguous, off a 16-byte boundary, or by way of the
    host.  The gradients do not change."""
    g = torch.Generator().manual_seed(10)
    x = _randn(g, 2, 37, 8, 64, dtype=BF16).cuda().requires_grad_()
    w = (1 + 0.3 * _randn(g, 64)).cuda().requires_grad_()
    table = fa.rotary_table(37, 64).cuda()
    gq, gk = _randn(g, 2, 4, 37, 64, dtype=BF16).cuda(), _randn(g, 2, 2, 37, 64, dtype=BF16).cuda()

    def step():
        q, k = x[:, :, :4].transpose(1, 2), x[:, :, 4:6].transpose(1, 2)
        z = fa.qk_norm_rotary(q, k, table, query_weight=w, key_weight=w)
        return torch.autograd.grad(z, (x, w), (gq, gk))

    def contiguous(t):
        return t.detach().clone(memory_format=torch.contiguous_format)

    def shifted(t):
        if t.ndim < 4:
            return contiguous(t)
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        return room[1:].view(t.shape).copy_(t.detach())

    want = step()
    for hooks in (torch.autograd.graph.saved_tensors_hooks(contiguous, lambda t: t),
                  torch.autograd.graph.saved_tensors_hooks(shifted, lambda t: t),
                  torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True)):
        with hooks:
            got = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------- the ends of the range
def _edge_check(x, w, table, pos, eps, z, gz, dx, dw):
    """As ``_check`` for bf16 rows of any size: a result below 2^-126 is also
    off by half of bf16's smallest step, 2^-134, and of fp32's on the way."""
    x64, gz64, w64 = _f64(x), _f64(gz), _f64(w)
    rd = table.shape[1]
    ref = orc.norm_rotary_reference(x64, w64, table.cpu().numpy(), pos, eps, False, gz64)
    r = 1 / np.sqrt((x64 ** 2).mean(-1, keepdims=True) + eps)
    dy = _pair_size(gz64, rd, False)
    g = dy * np.abs(w64)
    size = r * (g + np.abs(x64) * r * r * (g * np.abs(x64)).mean(-1, keepdims=True))
    for what, got, want, slack in (("z", z, ref["z"], 2.0 ** -19 * _pair_size(x64 * r * w64, rd, False)),
                                   ("dx", dx, ref["dx"], 2.0 ** -18 * size)):
        tol = 2.0 ** -8 * np.abs(want) * 1.001 + slack + 2.0 ** -133
        diff = np.abs(_f64(got) - want)
        assert (diff <= tol).all(), (what, np.argwhere(~(diff <= tol))[:4].tolist(), int((~(diff <= tol)).sum()))
    _assert_close(dw, ref["dw"], 2.0 ** -16 * (dy * np.abs(x64) * r).sum((0, 1)), dw.dtype, "dw")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("eps,powers", [(1e-6, [0, 40, 49, 50, 51, 60, 63, 64, 65, 90, 110, 125]),
                                        (0.0, [0, -40, -49, -50, -51, -60, -64, -75, -90, -110, -120])])
def test_bf16_rows_whose_squares_leave_the_fp32_range(d, eps, powers):
    """Rows of size 2^p: from p = 64 on their squares pass the fp32 range, and
    without an eps below p = -64 they vanish in it.  The norm is the row's all
    the same, and so are the gradients."""
    g = torch.Generator().manual_seed(d)
    n, h = 3 * len(powers), 3
    x = _randn(g, n, h, d).clamp(-4, 4)
    x *= torch.tensor([2.0 ** p for p in powers], dtype=F32).repeat(3)[:, None, None]
    x[0, 1] *= 2.0 ** (20 if powers[1] > 0 else -20)  # rows of one token in and out of the range
    x[len(powers) - 1, 2] *= 2.0 ** (-80 if powers[1] > 0 else 80)
    x = x.to(BF16)
    x[-1, 0, 5:] = 0  # few values
    w = (1 + 0.3 * _randn(g, d)).cuda().requires_grad_()
    gz = _randn(g, n, h, d, dtype=BF16).cuda()
    table = fa.rotary_table(n, d).cuda()
    pos = torch.arange(n, dtype=torch.int32)
    xq = x.cuda().requires_grad_()
    z, _ = fa.qk_norm_rotary(xq, xq.detach(), table, pos.cuda(), query_weight=w, key_weight=w.detach(), eps=eps)
    dx, dw = torch.autograd.grad(z, (xq, w), gz)
    _edge_check(x, w, table, pos.numpy(), eps, z, gz, dx, dw)
    kc = torch.zeros(-(-n // 16), 16, h, d, dtype=BF16, device="cuda")
    q = fa.paged_append(xq.detach(), xq.detach(), xq.detach(), kc, kc.clone(), pos.cuda(), table, pos.cuda(),
                        query_weight=w.detach(), key_weight=w.detach(), eps=eps)
    assert torch.equal(q, z.detach()) and torch.equal(kc.view(-1, h, d)[:n], q)


@pytest.mark.gpu
def test_rows_with_infinities_zeros_and_the_largest_value():
    table = fa.rotary_table(4, 32).cuda()
    q = torch.zeros(4, 2, 64, dtype=BF16).cuda()
    q[0, 0] = 3e38
    q[0, 1] = torch.finfo(BF16).max
    q[1, :, 3] = float("inf")
    q[1, :, 40] = 5.0
    pos, w = torch.zeros(4, dtype=torch.int32).cuda(), torch.ones(64).cuda()
    z, _ = fa.qk_norm_rotary(q, q, table, pos, query_weight=w, key_weight=w)
    assert (z[0] == 1).all()
    # an infinity over an infinite norm, also in its pair's other column; everything else vanishes
    assert z[1, :, [3, 19]].isnan().all() and (z[1, :, 32:] == 0).all() and (z[1, :, [0, 15, 31]] == 0).all()
    assert (z[2:] == 0).all()
    z, _ = fa.qk_norm_rotary(q, q, table, pos, query_weight=w, key_weight=w, eps=0.0)
    assert (z[0] == 1).all() and z[2:].isnan().all()  # 0 / 0
    assert _abi.device_status() == 0


# ---------------------------------------------------------------- many tokens a warp
LONG = [
    # b, n, hq, hkv, d, rd, interleaved, norm, weights, dtype
    (3, 1367, 32, 8, 128, 128, False, True, F32, BF16),
    (3, 1367, 32, 8, 128, 64, False, False, None, F16),
    (3, 2221, 16, 16, 64, 64, True, True, F16, F16),
    (3, 2221, 16, 16, 64, 32, True, False, None, BF16),
    (5, 2665, 8, 8, 32, 32, False, True, BF16, BF16),
    (5, 2665, 8, 8, 32, 16, True, False, None, F16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("b,n,hq,hkv,d,rd,interleaved,norm,wdt,dt", LONG)
def test_ranges_of_many_tokens_that_cross_batches(b, n, hq, hkv, d, rd, interleaved, norm, wdt, dt):
    """A warp takes 10 to 18 tokens of its heads here (148 SMs), several turns
    of its ring, and ranges run over the ends of batches of odd length."""
    g = torch.Generator().manual_seed(n + d + rd)
    table = fa.rotary_table(n + 40, rd).cuda()
    weights = [(1 + 0.5 * _randn(g, d)).to(wdt).cuda().requires_grad_() if norm else None for _ in range(2)]
    x = _randn(g, b, n, hq + hkv, d, dtype=dt).cuda()
    q, k = (t.transpose(1, 2).detach().requires_grad_() for t in (x[:, :, :hq], x[:, :, hq:]))
    gz = [_randn(g, b, h, n, d, dtype=dt).cuda() for h in (hq, hkv)]
    pos = torch.stack([torch.randperm(n + 40, generator=g)[:n] for _ in range(b)]).int()
    z = fa.qk_norm_rotary(q, k, table, pos.cuda(), query_weight=weights[0], key_weight=weights[1], eps=1e-5,
                          interleaved=interleaved)
    grads = torch.autograd.grad(z, [q, k] + [w for w in weights if norm], gz)
    for i, src in enumerate((q, k)):
        _check(_packed(src.detach()), weights[i], table, pos.reshape(-1).numpy(), 1e-5, interleaved, _packed(z[i]),
               _packed(gz[i]), _packed(grads[i]), grads[2 + i] if norm else None)
    assert _abi.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("total,hq,hkv,d,dt", [(9174, 8, 2, 64, BF16), (9001, 3, 1, 128, F16), (15013, 4, 4, 32, F16)])
def test_append_of_many_tokens(total, hq, hkv, d, dt):
    """As above for the cache: 10 to 16 tokens a warp, some without a slot,
    against float64."""
    g = torch.Generator().manual_seed(total)
    page, n_pages = 16, total // 16 + 4
    x = _randn(g, total, hq + 2 * hkv, d, dtype=dt).cuda()
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    table = fa.rotary_table(total + 3, d).cuda()
    pos = torch.randperm(total + 3, generator=g)[:total].int()
    slots = torch.randperm(n_pages * page, generator=g)[:total].int()
    slots[torch.randperm(total, generator=g)[:total // 7]] = -1
    wq, wk = ((1 + 0.5 * _randn(g, d)).cuda() for _ in range(2))
    kc, vc = (torch.full((n_pages, page, hkv, d), float("nan"), dtype=dt, device="cuda") for _ in range(2))
    out = fa.paged_append(q, k, v, kc, vc, slots.cuda(), table, pos.cuda(), query_weight=wq, key_weight=wk)
    _check(q, wq, table, pos.numpy(), 1e-6, False, out)
    has = slots >= 0
    at = slots[has].long().cuda()
    _check(k[has.cuda()], wk, table, pos[has].numpy(), 1e-6, False, kc.view(-1, hkv, d)[at])
    assert torch.equal(vc.view(-1, hkv, d)[at], v[has.cuda()])
    rest = torch.ones(n_pages * page, dtype=torch.bool, device="cuda")
    rest[at] = False
    assert kc.view(-1, hkv, d)[rest].isnan().all() and vc.view(-1, hkv, d)[rest].isnan().all()
    assert _abi.device_status() == 0


# ---------------------------------------------------------------- the launches by themselves
def test_launches_refuse_what_they_would_misread():
    """The forward's and backward's launches check what ``qk_norm_rotary``
    does, and the gradients."""
    q, k = torch.randn(5, 4, 32).half(), torch.randn(5, 2, 32).half()
    t, p, w = fa.rotary_table(8, 32), torch.arange(5, dtype=torch.int32), torch.ones(32)
    fwd = [q, k, t, p, w, w, 1e-6, False]
    bwd = [q, k, q.clone(), k.clone(), t, p, w, w, 1e-6, False]
    for call, args, rest in ((fa.qk_norm_rotary_forward, fwd, 2), (fa.qk_norm_rotary_backward, bwd, 4)):
        with pytest.raises(RuntimeError, match="requires a CUDA tensor"):
            call(*args)
        for at, bad, message in [(rest + 1, p.long(), "int32"), (rest + 1, p[:4], "int32"), (rest, t[:, :16], "contiguous"),
                                 (rest + 2, w[:16], "head_dim weights"), (rest + 3, None, "both"),
                                 (rest + 4, -1.0, "eps"), (1, k[:4], None)]:
            with pytest.raises(ValueError, match=message):
                call(*[bad if j == at else x for j, x in enumerate(args)])
    for at, bad in ((2, q[:4]), (2, q.float()), (3, q)):
        with pytest.raises(ValueError, match="shape, dtype and device"):
            fa.qk_norm_rotary_backward(*[bad if j == at else x for j, x in enumerate(bwd)])
    with pytest.raises(TypeError, match="grad_q"):
        fa.qk_norm_rotary_backward(q, k, None, *bwd[3:])


@pytest.mark.gpu
def test_launches_take_positions_and_weights_of_any_stride():
    g = torch.Generator().manual_seed(11)
    q, k, gq, gk = (_randn(g, 40, h, 64, dtype=F16).cuda() for h in (4, 2, 4, 2))
    table, pos, w = fa.rotary_table(90, 64).cuda(), torch.arange(40, dtype=torch.int32).cuda() * 2, torch.rand(64).cuda()
    wide = torch.full((40, 3), 1 << 30, dtype=torch.int32, device="cuda")
    wide[:, 1] = pos
    ww = torch.full((64, 2), float("nan"), device="cuda")
    ww[:, 0] = w
    one = torch.full((1,), 7, dtype=torch.int32, device="cuda").expand(40)
    for p, v in ((pos, w), (wide[:, 1], ww[:, 0]), (one, w)):
        z = fa.qk_norm_rotary_forward(q, k, table, p, v, v, 1e-6, False)
        d = fa.qk_norm_rotary_backward(q, k, gq, gk, table, p, v, v, 1e-6, False)
        pc, vc = p.contiguous(), v.contiguous()
        want = (fa.qk_norm_rotary_forward(q, k, table, pc, vc, vc, 1e-6, False)
                + fa.qk_norm_rotary_backward(q, k, gq, gk, table, pc, vc, vc, 1e-6, False))
        assert all(torch.equal(a, b) for a, b in zip(z + d, want))
    assert _abi.device_status() == 0
