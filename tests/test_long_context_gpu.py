"""Rotary positions, query / key norms and windowed attention against plain implementations in 64 bits.

Tolerances are bounds per element, from the roundings a result goes through: U = half a step of the storage type (2^-8
bf16, 2^-24 fp32) for every value that is stored in it, E = 2^-24 for every fp32 operation, multiplied by the absolute
values that the rounded quantities meet on the way to the element."""
import decimal
import math
import threading

import pytest
import torch

from specialk_amd import _lib as L
from specialk_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
E = 2.0 ** -24
TINY = 1e-30


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rnd(shape, dtype, g, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def check(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    over = (got - want).abs() - bound.cpu()
    assert bool((over <= 0).all()), f"{what}: off by {(got - want).abs().max():.3g}, worst over its bound by {over.max():.3g}"


# ------------------------------------------------------------------------------ rotary and norm
def turn64(x, pos, f, rot, il, sign=1):
    """x (T, heads, d) with its first rot elements turned, in 64 bits; also |a| + |b| of every element's pair."""
    ang = sign * pos.double()[:, None] * torch.tensor(f.radians, dtype=torch.float64)[None]
    c, s = (torch.cos(ang) * f.amplitude)[:, None], (torch.sin(ang) * f.amplitude)[:, None]
    h = x[..., :rot]
    a, b = (h[..., 0::2], h[..., 1::2]) if il else (h[..., :rot // 2], h[..., rot // 2:])
    y0, y1 = a * c - b * s, b * c + a * s
    m = a.abs() + b.abs()
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if il else (lambda u, v: torch.cat((u, v), -1))
    return torch.cat((join(y0, y1), x[..., rot:]), -1), torch.cat((join(m, m) * f.amplitude, x[..., rot:].abs()), -1)


# cosine and sine: argument rounded twice (2 E x <= 2 E), a polynomial of six terms, two products, one sum
ROT_E = 12 * E


def rotary_case(T, H, G, d, rot, dtype, il, far, gen, **kw):
    f = ops.RotaryFrequencies(rot, device=DEV, **kw)
    pos = torch.randint(0, 300, (T,), generator=gen) + far
    q, k = rnd((T, H * d), dtype, gen, 1.5), rnd((T, G * d), dtype, gen, 1.5)
    return f, pos, q, k


SHAPES = [  # T, H, G, d, rot
    (1, 1, 1, 64, 64), (640, 8, 8, 64, 64), (37, 8, 2, 128, 64), (5, 3, 1, 80, 80), (19, 4, 4, 96, 48), (1030, 2, 1, 32, 32),
    (700, 4, 2, 64, 36), (33, 3, 1, 72, 40), (9, 2, 2, 96, 86), (50, 2, 1, 24, 6), (21, 1, 1, 248, 130), (300, 4, 1, 128, 2), (7, 5, 5, 37, 18), (3, 2, 2, 256, 256), (66, 16, 16, 16, 2), (2, 40, 8, 128, 128), (9, 1, 1, 3, 2), (8, 512, 512, 64, 30)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(shape, il, dtype):
    T, H, G, d, rot = shape
    g = torch.Generator().manual_seed(T * 7 + d)
    f, pos, q, k = rotary_case(T, H, G, d, rot, dtype, il, 0, g)
    dq, dk = rnd((T, H * d), dtype, g), rnd((T, G * d), dtype, g)
    qd, kd = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    oq, ok = ops.rotary(qd, kd, pos.to(DEV), f, H, G, interleaved=il)
    gq, gk = torch.autograd.grad((oq, ok), (qd, kd), (dq.to(DEV), dk.to(DEV)))
    for x, out, dy, dx in ((q, oq, dq, gq), (k, ok, dk, gk)):
        for src, got, sign, what in ((x, out, 1, "forward"), (dy, dx, -1, "gradient")):
            want, mag = turn64(src.double().view(T, -1, d), pos, f, rot, il, sign)
            check(got, want.view(T, -1), (unit(dtype) * want.abs() + ROT_E * mag).view(T, -1) + TINY, what)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
@pytest.mark.parametrize("far", [0, 100000, 1 << 31, -70000])
def test_rotary_far_positions(far, scaling):
    """Angles of far positions: exact but for the reference's own product pos * f, rounded to 2^-53 of the angle."""
    g = torch.Generator().manual_seed(3)
    f, pos, q, k = rotary_case(50, 2, 1, 64, 64, F32, False, far, g, scaling=scaling, factor=8.0, trained_len=4096)
    out, _ = ops.rotary(q.to(DEV), None, pos.to(DEV), f, 2, interleaved=False)
    want, mag = turn64(q.double().view(50, 2, 64), pos, f, 64, False)
    own = pos.abs().max().item() * 2.0 ** -52
    check(out, want.view(50, -1), (E * want.abs() + (ROT_E + own) * mag).view(50, -1), "far")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_reads_slices_and_odd_strides(dtype):
    """Slices of a fused projection (16-byte rows), the same one element off (scalar form), transposed rows: one result."""
    g = torch.Generator().manual_seed(8)
    T, H, d = 33, 4, 64
    f = ops.RotaryFrequencies(64, device=DEV)
    pos = torch.arange(T, device=DEV)
    x = rnd((T, H * d), dtype, g).to(DEV)
    want, _ = ops.rotary(x, None, pos, f, H)
    wide = torch.zeros((T, 3 * H * d + 8), dtype=dtype, device=DEV)
    for off in (0, 8, H * d, 1, 3):
        wide[:, off:off + H * d] = x
        got, _ = ops.rotary(wide[:, off:off + H * d], None, pos, f, H)
        assert torch.equal(got, want), off
    got, _ = ops.rotary(x.t().contiguous().t(), None, pos, f, H)
    assert torch.equal(got, want)
    part = ops.RotaryFrequencies(36, device=DEV)   # halves of a pair with different lanes, or element by element
    for il in (False, True):
        want36, _ = ops.rotary(x, None, pos, part, H, interleaved=il)
        for off in (8, 1):
            wide[:, off:off + H * d] = x
            got, _ = ops.rotary(wide[:, off:off + H * d], None, pos, part, H, interleaved=il)
            assert torch.equal(got, want36), (il, off)
    one, _ = ops.rotary(x[:1].expand(T, -1), None, pos, f, H)
    assert torch.equal(one, ops.rotary(x[:1].repeat(T, 1), None, pos, f, H)[0])


def norm64(x, gamma, eps, pos, f, rot, il):
    y = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gamma
    return (y, y.abs()) if f is None else turn64(y, pos, f, rot, il)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("shape", SHAPES[:-1] + [(6000, 8, 8, 64, 64), (25, 4, 2, 64, 0)])
def test_qk_norm_rotary(shape, il, dtype):
    T, H, G, d, rot = shape
    g = torch.Generator().manual_seed(T + d)
    f, pos, q, k = rotary_case(T, H, G, d, max(rot, 2), dtype, il, 5, g)
    if rot == 0:
        f = None
    eps = 1e-5
    gq, gk = 1 + 0.3 * torch.randn(d, generator=g), 1 + 0.3 * torch.randn(d, generator=g)
    dq, dk = rnd((T, H * d), dtype, g), rnd((T, G * d), dtype, g)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, gq, gk)]
    out = ops.qk_norm_rotary(*leaves, None if f is None else pos.to(DEV), f, H, G, eps=eps, interleaved=il)
    grads = torch.autograd.grad(out, leaves, (dq.to(DEV), dk.to(DEV)))
    # the mean of d squares, root, reciprocal, two products: relative to the normalised value
    rel = (d + 8) * E
    for x, gm, dy, y, dx, dg in ((q, gq, dq, out[0], grads[0], grads[2]), (k, gk, dk, out[1], grads[1], grads[3])):
        x64 = x.double().view(T, -1, d).requires_grad_()
        g64 = gm.double().requires_grad_()
        want, mag = norm64(x64, g64, eps, pos, f, rot, il)
        check(y, want.detach().view(T, -1), (unit(dtype) * want.abs() + (ROT_E + rel) * mag).detach().view(T, -1) + TINY, "forward")
        dx64, dg64 = torch.autograd.grad(want, (x64, g64), dy.double().view(T, -1, d))
        # by the formula: r = R^T dy, dx = rstd (r gamma - xhat mean(r gamma xhat))
        r, rmag = (dy.double().view(T, -1, d),) * 2 if f is None else turn64(dy.double().view(T, -1, d), pos, f, rot, il, -1)
        rmag = rmag.abs()
        xd = x.double().view(T, -1, d)
        rstd = 1 / (xd.pow(2).mean(-1, keepdim=True) + eps).sqrt()
        xhat = xd * rstd
        mean = (r * gm.double() * xhat).mean(-1, keepdim=True)
        formula = rstd * (r * gm.double() - xhat * mean)
        torch.testing.assert_close(dx64, formula, rtol=1e-9, atol=1e-9)
        mabs = (rmag * gm.double().abs() * xhat.abs()).mean(-1, keepdim=True)
        bound = unit(dtype) * formula.abs() + rstd * (rmag * gm.double().abs() + xhat.abs() * mabs) * (ROT_E + (2 * d + 16) * E)
        check(dx, dx64.view(T, -1), bound.view(T, -1) + TINY, "dx")
        # dgamma: terms r xhat, added by a thread over its rows, then lanes, waves and blocks: chains of 128 + T / 64 at most
        terms = (rmag * xhat.abs()).sum((0, 1))
        check(dg, dg64, terms * (ROT_E + rel + (128 + T / 64) * E) + TINY, "dgamma")


def test_qk_norm_rotary_gradient_by_differences():
    g = torch.Generator().manual_seed(1)
    T, H, d = 3, 2, 16
    f = ops.RotaryFrequencies(8, device=DEV)
    pos = torch.tensor([0, 4, 9], device=DEV)
    x, w = torch.randn((T, H * d), generator=g), torch.randn((T, H * d), generator=g).to(DEV)
    gm = (1 + 0.2 * torch.randn(d, generator=g)).to(DEV)

    def loss(t):
        return (ops.qk_norm_rotary(t, None, gm, None, pos, f, H)[0].double() * w.double()).sum()

    leaf = x.to(DEV).requires_grad_()
    (grad,) = torch.autograd.grad(loss(leaf), leaf)
    h = 2.0 ** -7
    for i, j in ((0, 0), (1, 5), (2, 20), (2, 31)):
        step = torch.zeros_like(x)
        step[i, j] = h
        diff = (loss((x + step).to(DEV)) - loss((x - step).to(DEV))) / (2 * h)
        # third derivatives of x / rms(x) are below 100 here: 100 h^2 / 6; and 64 outputs rounded to E over 2 h
        assert abs(diff.item() - grad[i, j].item()) <= 100 * h * h / 6 + 64 * 8 * E / (2 * h), (i, j)


def test_norm_row_of_zeros_and_large_values():
    f = ops.RotaryFrequencies(64, device=DEV)
    x = torch.zeros((3, 64), device=DEV)
    x[1] = 3e18      # squares near the largest fp32
    x[2, 5] = float("inf")
    out, _ = ops.qk_norm_rotary(x, None, torch.ones(64, device=DEV), None, torch.zeros(3, dtype=torch.int64, device=DEV), f, 1)
    assert torch.equal(out[0], torch.zeros(64, device=DEV))
    assert bool((out[1] - 1).abs().max() <= 80 * E)
    assert bool(torch.isnan(out[2, 5]))


def test_empty_rows():
    f = ops.RotaryFrequencies(64, device=DEV)
    x = torch.empty((0, 128), device=DEV, requires_grad=True)
    gm = torch.ones(64, device=DEV, requires_grad=True)
    out, _ = ops.qk_norm_rotary(x, None, gm, None, torch.empty(0, dtype=torch.int64, device=DEV), f, 2)
    dx, dg = torch.autograd.grad(out, (x, gm), torch.empty_like(out))
    assert out.shape == (0, 128) and dx.shape == (0, 128) and torch.equal(dg, torch.zeros(64, device=DEV))


# ------------------------------------------------------------------------------ windowed attention
def visible(n, m, window, sinks, causal, pad=None):
    p = torch.arange(n)[:, None] + m - n
    j = torch.arange(m)[None]
    v = ((p - j < window) | (j < sinks)) & ((j <= p) if causal else (j - p < window))
    return v if pad is None else v & ~pad.bool()[None]


def attention64(q, k, v, do, vis, scale, dtype):
    """One sequence and query head: (o, dq, dk, dv) in 64 bits and a bound on each (fp32 operations, values rounded to dtype).
    bf16 products take the probabilities and dS rounded to bf16; delta = rowsum(dO O) takes the rounded output."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    n, d = vis.sum(1).max().item(), q.shape[1]
    some = vis.any(1, keepdim=True)
    s = (q @ k.t() * scale).masked_fill(~vis, -math.inf)
    s = torch.where(some, s, torch.zeros_like(s))
    p = torch.softmax(s, 1) * vis
    o = p @ v
    dp = do @ v.t()
    delta = (do * o).sum(1, keepdim=True)
    ds = p * (dp - delta) * scale
    dq, dk, dv = ds @ k, ds.t() @ q, p.t() @ do
    ub = unit(dtype) if dtype == BF else 0.0                   # operands of the matrix products
    u = unit(dtype)
    smax = (q.abs() @ k.abs().t() * abs(scale) * vis).max()
    rel = (2 * (d + 6) * smax + 2 * n + 16) * E                # of a probability: score, exponential, row sum
    a = p @ v.abs()
    eo = u * o.abs() + a * (ub + rel)
    edelta = (do.abs() * eo).sum(1, keepdim=True) + (d + 2) * E * (do.abs() * o.abs()).sum(1, keepdim=True)
    edp = (d + 2) * E * (do.abs() @ v.abs().t())
    eds = ds.abs() * (ub + rel + 4 * E) + p * abs(scale) * (edelta + edp)
    acc = (max(vis.shape) + 8) * E
    return ((o, eo), (dq, u * dq.abs() + eds @ k.abs() + acc * ds.abs() @ k.abs()),
            (dk, u * dk.abs() + eds.t() @ q.abs() + acc * ds.abs().t() @ q.abs()),
            (dv, u * dv.abs() + (p * (ub + rel + acc)).t() @ do.abs()))


def run_window(lens_q, lens_k, H, G, d, window, sinks, causal, dtype, layout, seed=0, scale=None, pads=None):
    """All sequences against attention64; returns nothing, raises where an element leaves its bound."""
    g = torch.Generator().manual_seed(seed + d)
    B, Lq, Lk = len(lens_q), max(lens_q), max(lens_k)
    tq, tk = (sum(lens_q), sum(lens_k)) if layout == "packed" else (B * Lq, B * Lk)
    q, k, v, do = rnd((tq, H * d), dtype, g), rnd((tk, G * d), dtype, g), rnd((tk, G * d), dtype, g), rnd((tq, H * d), dtype, g)
    kw = {}
    if layout == "packed":
        kw = dict(q_off=torch.tensor([0] + lens_q).cumsum(0).int().to(DEV), k_off=torch.tensor([0] + lens_k).cumsum(0).int().to(DEV))
    elif pads is not None:
        kw = dict(key_pad=pads.to(DEV))
    qd, kd, vd = (t.to(DEV).requires_grad_() for t in (q, k, v))
    o = ops.window_attention(qd, kd, vd, B, Lq, Lk, H, G, window, sinks, causal, scale, **kw)
    grads = torch.autograd.grad(o, (qd, kd, vd), do.to(DEV))
    sc = d ** -0.5 if scale is None else scale
    want = [torch.zeros((t, w * d), dtype=torch.float64) for t, w in ((tq, H), (tq, H), (tk, G), (tk, G))]
    bound = [torch.zeros_like(t) + TINY for t in want]
    q0 = k0 = 0
    for b in range(B):
        n, m = (lens_q[b], lens_k[b]) if layout == "packed" else (Lq, Lk)
        vis = visible(n, m, window or 1 << 30, sinks, causal, None if pads is None else pads[b])
        for h in range(H if n and m else 0):
            hs, ks = slice(h * d, h * d + d), slice(h // (H // G) * d, h // (H // G) * d + d)
            kk = k[k0:k0 + m, ks]
            vv = v[k0:k0 + m, ks]
            res = attention64(q[q0:q0 + n, hs], kk, vv, do[q0:q0 + n, hs], vis, sc, dtype)
            for i, (rs, cs) in enumerate(((slice(q0, q0 + n), hs), (slice(q0, q0 + n), hs), (slice(k0, k0 + m), ks), (slice(k0, k0 + m), ks))):
                want[i][rs, cs] += res[i][0]
                bound[i][rs, cs] += res[i][1]
        q0, k0 = q0 + n, k0 + m
    for got, w, bd, what in zip((o,) + grads, want, bound, ("o", "dq", "dk", "dv")):
        check(got, w, bd, what)
    return o, grads


WINDOWS = [  # lens_q, lens_k, H, G, d, window, sinks, causal
    ([1], [1], 1, 1, 64, 1, 0, True),
    ([5], [5], 2, 2, 64, 2, 1, True),
    ([200], [200], 2, 1, 64, 33, 4, True),
    ([130], [130], 2, 2, 128, 64, 0, False),
    ([300], [300], 4, 1, 128, 40, 70, True),        # sinks over more than one tile
    ([257], [257], 2, 2, 32, 1000, 3, True),        # window beyond the text: plain causal
    ([190], [190], 1, 1, 80, 17, 2, False),
    ([64], [333], 2, 1, 64, 50, 5, True),           # queries at the end of a longer text
    ([150], [70], 2, 2, 64, 20, 2, True),           # more queries than keys: the first see nothing
    ([700], [700], 1, 1, 64, 20, 130, True),        # far queries in chunks, two sink tiles
    ([100], [100], 2, 2, 40, 10, 1, True),
    ([90], [90], 3, 3, 37, 12, 3, False),           # odd head size
    ([65, 1, 129], [65, 1, 129], 2, 1, 96, 30, 2, True)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", WINDOWS)
def test_window_attention(case, dtype):
    lens_q, lens_k, H, G, d, window, sinks, causal = case
    layout = "packed" if len(lens_q) > 1 else "dense"
    run_window(lens_q, lens_k, H, G, d, window, sinks, causal, dtype, layout)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
def test_window_packed_ragged(causal, dtype):
    """Sequences of no, one and many rows, queries and keys of different lengths."""
    run_window([0, 1, 70, 3, 128, 0, 65], [2, 1, 90, 0, 128, 0, 64], 2, 1, 64, 25, 3, causal, dtype, "packed")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128])
def test_window_key_padding(d, dtype):
    """Padding on the right, on the left, everywhere, in the middle: rows that are left with nothing give zeros."""
    B, n = 5, 150
    pads = torch.zeros((B, n), dtype=torch.uint8)
    pads[1, 90:] = 1
    pads[2, :100] = 1
    pads[3] = 1
    pads[4, 40:110:3] = 1
    o, grads = run_window([n] * B, [n] * B, 2, 2, d, 20, 2, True, dtype, "padded", pads=pads)
    assert not o.view(B, n, -1)[3].any() and not any(t.view(B, n, -1)[3].any() for t in grads)
    assert not o.view(B, n, -1)[2, :100].any()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_window_none_and_scale(dtype):
    run_window([140], [140], 2, 1, 64, None, 0, True, dtype, "dense", scale=0.3)
    run_window([140], [140], 2, 1, 64, None, 9, False, dtype, "dense")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 128, 80])
def test_masked_places_may_hold_anything(d, dtype):
    """Padded keys, keys that no query reaches and rows behind the last sequence hold NaN and infinities."""
    g = torch.Generator().manual_seed(5)
    B, n, H = 2, 200, 2
    q, k, v, do = (rnd((B * n, H * d), dtype, g).to(DEV) for _ in range(4))
    pads = torch.zeros((B, n), dtype=torch.uint8, device=DEV)
    pads[0, 120:] = 1
    pads[1, :33] = 1
    bad = pads.view(-1).bool()

    def run(k, v):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = ops.window_attention(*leaves, B, n, n, H, H, 40, 4, key_pad=pads)
        return (o,) + torch.autograd.grad(o, leaves, do)

    want = run(k.masked_fill(bad[:, None], 0.0), v.masked_fill(bad[:, None], 0.0))
    for fill in (float("nan"), float("inf"), torch.finfo(dtype).min):
        for a, b in zip(run(k.masked_fill(bad[:, None], fill), v.masked_fill(bad[:, None], fill)), want):
            assert torch.equal(a, b), fill
    # the last 20 queries of a text: keys before their windows are out of every query's reach
    lo = n - 20 - 39
    kk, vv = k[:n].clone(), v[:n].clone()
    base = ops.window_attention(q[:20], kk, vv, 1, 20, n, H, H, 40, 4)
    kk[4:lo], vv[4:lo] = float("nan"), float("-inf")
    assert torch.equal(ops.window_attention(q[:20], kk, vv, 1, 20, n, H, H, 40, 4), base)
    # packed rows before the first and behind the last sequence
    off = torch.tensor([3, 60, 111], dtype=torch.int32, device=DEV)
    kk, vv, qq, dd = (t[:n].clone() for t in (k, v, q, do))
    for t in (kk, vv, qq, dd):
        t[:3], t[111:] = float("nan"), float("inf")
    leaves = [t.requires_grad_() for t in (qq, kk, vv)]
    o = ops.window_attention(*leaves, 2, 60, 60, H, H, 40, 4, q_off=off, k_off=off)
    for t in (o,) + torch.autograd.grad(o, leaves, dd):
        assert bool(torch.isfinite(t).all()) and not t[:3].any() and not t[111:].any() and bool(t[3:111].any())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_window_strides_and_alignment(dtype):
    """Heads inside a fused projection, rows one element off, transposed storage: the result of contiguous rows."""
    g = torch.Generator().manual_seed(2)
    n, H, G, d = 150, 4, 2, 64
    q, k, v = rnd((n, H * d), dtype, g).to(DEV), rnd((n, G * d), dtype, g).to(DEV), rnd((n, G * d), dtype, g).to(DEV)
    do = rnd((n, H * d), dtype, g).to(DEV)

    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = ops.window_attention(*leaves, 1, n, n, H, G, 30, 2)
        return (o,) + torch.autograd.grad(o, leaves, do)

    want = run(q, k, v, do)
    for shift, extra in ((0, 9), (8, 9), (1, 9), (0, 16), (8, 16)):
        wide = torch.zeros((n, (H + 2 * G) * d + 16), dtype=dtype, device=DEV)
        cut = wide[:, shift:shift + (H + 2 * G) * d]
        cut[:, :H * d], cut[:, H * d:(H + G) * d], cut[:, (H + G) * d:] = q, k, v
        dw = torch.zeros((n, H * d + extra), dtype=dtype, device=DEV)
        dw[:, shift:shift + H * d] = do
        got = run(cut[:, :H * d], cut[:, H * d:(H + G) * d], cut[:, (H + G) * d:], dw[:, shift:shift + H * d])
        for a, b, name in zip(got, want, ("o", "dq", "dk", "dv")):
            # (rows of 16-byte pieces throughout: the same kernel)
            if dtype == F32 or (shift % 8 == 0 and (extra % 8 == 0 or name == "o")):
                assert torch.equal(a, b), (shift, extra, name)
            else:   # another kernel: same definition, both within the bounds that run_window checks
                torch.testing.assert_close(a.float(), b.float(), rtol=0.05, atol=0.05)
    for a, b in zip(run(q.t().contiguous().t(), k, v, do.t().contiguous().t()), want):
        assert torch.equal(a, b)
    # a gradient that autograd hands over expanded
    leaf = q.clone().requires_grad_()
    (dq,) = torch.autograd.grad(ops.window_attention(leaf, k, v, 1, n, n, H, G, 30, 2).sum(), leaf)
    assert torch.equal(dq, run(q, k, v, torch.ones_like(do))[1])


def test_window_gradient_by_differences():
    g = torch.Generator().manual_seed(4)
    n, H, G, d = 40, 2, 1, 16
    t = [torch.randn((n, w * d), generator=g) for w in (H, G, G)]
    w = torch.randn((n, H * d), generator=g).to(DEV).double()

    def loss(*x):
        return (ops.window_attention(*x, 1, n, n, H, G, 7, 2).double() * w).sum()

    leaves = [x.to(DEV).requires_grad_() for x in t]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    h = 2.0 ** -6
    for which in range(3):
        for i, j in ((0, 0), (1, 3), (17, 9), (39, 15)):
            step = torch.zeros_like(t[which])
            step[i, j] = h
            up = loss(*((x + step if a == which else x).to(DEV) for a, x in enumerate(t)))
            down = loss(*((x - step if a == which else x).to(DEV) for a, x in enumerate(t)))
            diff = ((up - down) / (2 * h)).item()
            # third derivatives along one entry of q or k: up to 80 outputs, each below 2; outputs rounded to 8 E of size 3
            assert abs(diff - grads[which][i, j].item()) <= 160 * h * h / 6 + n * H * d * 24 * E / (2 * h) / 10, (which, i, j)


def test_window_results_repeat_bit_for_bit():
    g = torch.Generator().manual_seed(6)
    n, H, G, d = 1500, 4, 1, 64
    q, k, v, do = (rnd((n, w * d), BF, g).to(DEV) for w in (H, G, G, H))
    first = None
    for _ in range(3):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = ops.window_attention(*leaves, 1, n, n, H, G, 100, 4)
        res = (o,) + torch.autograd.grad(o, leaves, do)
        first = first or res
        assert all(torch.equal(a, b) for a, b in zip(res, first))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", [  # few key heads: the dK / dV sums of a key tile come from several blocks
    ([400], [400], 8, 1, 64, 100, 3, True), ([700], [700], 4, 1, 128, 60, 140, True), ([520], [520], 2, 1, 64, None, 0, True),
    ([300], [410], 8, 2, 96, 200, 5, False), ([333], [333], 6, 1, 37, 150, 70, True), ([260], [130], 8, 1, 64, 90, 2, True)])
def test_window_keys_in_parts(case, dtype):
    lens_q, lens_k, H, G, d, window, sinks, causal = case
    run_window(lens_q, lens_k, H, G, d, window, sinks, causal, dtype, "dense", seed=3)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", [  # few queries before many keys: the keys of a query tile come to several blocks
    ([64], [4000], 2, 1, 64, None, 0, True), ([3], [3000], 4, 2, 128, 2500, 70, True), ([1], [2100], 1, 1, 37, None, 0, False),
    ([200], [1500], 2, 2, 96, 1200, 3, True), ([1500], [1500], 1, 1, 32, None, 0, True)])
def test_window_queries_in_cuts(case, dtype):
    lens_q, lens_k, H, G, d, window, sinks, causal = case
    run_window(lens_q, lens_k, H, G, d, window, sinks, causal, dtype, "dense", seed=6)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_window_queries_in_cuts_of_ragged_batches(dtype):
    run_window([5, 0, 40, 7], [2000, 900, 1300, 0], 2, 1, 64, 1900, 4, True, dtype, "packed", seed=7)
    pads = torch.zeros((3, 1800), dtype=torch.uint8)
    pads[0, 100:1700], pads[1, :1790], pads[2, :] = 1, 1, 1
    run_window([20] * 3, [1800] * 3, 2, 2, 80, None, 0, False, dtype, "padded", seed=8, pads=pads)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_window_keys_in_parts_of_ragged_batches(dtype):
    lens = [300, 1, 0, 170, 64]
    run_window(lens, lens, 8, 1, 64, 120, 4, True, dtype, "packed", seed=4)
    pads = torch.zeros((3, 290), dtype=torch.uint8)
    pads[0, 200:], pads[1, :40], pads[2, :] = 1, 1, 1
    run_window([290] * 3, [290] * 3, 8, 2, 80, 150, 2, True, dtype, "padded", seed=5, pads=pads)


# ------------------------------------------------------------------------------ one step over a cache
def slot_of(j, cap, sinks):
    return j if j < sinks else sinks + (j - sinks) % (cap - sinks)


def step_case(lens, H, G, d, cap, window, sinks, dtype, seed=0, fill=float("nan")):
    """Caches filled as a run would have left them (everything else `fill`), new rows, and the 64-bit result with bounds."""
    g = torch.Generator().manual_seed(seed + d)
    R = len(lens)
    q, kn, vn = rnd((R, H * d), dtype, g), rnd((R, G * d), dtype, g), rnd((R, G * d), dtype, g)
    kc = torch.full((R, cap, G * d), fill, dtype=dtype)
    vc = kc.clone()
    want, bound = torch.zeros((R, H * d), dtype=torch.float64), torch.full((R, H * d), TINY, dtype=torch.float64)
    for r, n in enumerate(lens):
        if n <= 0:
            continue
        pos = [j for j in range(n) if j >= n - window or j < sinks]
        k, v = rnd((len(pos), G * d), dtype, g), rnd((len(pos), G * d), dtype, g)
        k[-1], v[-1] = kn[r], vn[r]
        for i, j in enumerate(pos[:-1]):
            kc[r, slot_of(j, cap, sinks)], vc[r, slot_of(j, cap, sinks)] = k[i], v[i]
        for h in range(H):
            hs, ks = slice(h * d, h * d + d), slice(h // (H // G) * d, h // (H // G) * d + d)
            vis = torch.ones((1, len(pos)), dtype=torch.bool)
            (o, eo), *_ = attention64(q[r:r + 1, hs], k[:, ks], v[:, ks], q[r:r + 1, hs], vis, d ** -0.5, dtype)
            want[r, hs], bound[r, hs] = o[0], bound[r, hs] + eo[0]
    return q, kn, vn, kc, vc, want, bound


STEPS = [  # lens, H, G, d, cap, window, sinks
    ([1], 1, 1, 64, 8, 8, 0), ([5, 1, 0, 7, -3], 8, 8, 64, 16, 8, 2), ([100, 33], 8, 2, 128, 100, 64, 4),
    ([70, 69, 68, 300], 4, 1, 64, 68, 64, 4),            # rings, just full, one over, far over
    ([5000], 8, 8, 64, 5000, 4096, 1), ([4000, 9, 2500], 16, 2, 128, 1030, 1024, 6), ([50, 200], 3, 1, 80, 40, 33, 7),
    ([90], 2, 2, 37, 95, 40, 3), ([300, 20], 32, 1, 64, 200, 150, 0), ([1000] * 3, 6, 2, 96, 1000, 1000, 0),
    ([40000], 2, 1, 128, 600, 512, 60)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", STEPS)
def test_window_step(case, dtype):
    lens, H, G, d, cap, window, sinks = case
    q, kn, vn, kc, vc, want, bound = step_case(*case, dtype)
    kd, vd = kc.to(DEV), vc.to(DEV)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    o = ops.window_attention_step(q.to(DEV), kn.to(DEV), vn.to(DEV), kd, vd, n, H, G, window, sinks)
    check(o, want, bound, "o")
    for r, m in enumerate(lens):   # the new rows are in their slots, nothing else has changed
        if m > 0:
            kc[r, slot_of(m - 1, cap, sinks)], vc[r, slot_of(m - 1, cap, sinks)] = kn[r], vn[r]
    for got, ref in ((kd, kc), (vd, vc)):
        assert torch.equal(torch.nan_to_num(got.cpu(), 7.0), torch.nan_to_num(ref, 7.0))
        assert torch.equal(got.cpu().isnan(), ref.isnan())
    # with the rows in the caches already
    assert torch.equal(ops.window_attention_step(q.to(DEV), None, None, kd, vd, n, H, G, window, sinks), o)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_step_cache_layouts(dtype):
    """Keys and values side by side, position-major caches, rows one element off: the result of plain caches."""
    lens, H, G, d, cap, window, sinks = [100, 40, 260], 4, 2, 64, 104, 100, 4
    q, kn, vn, kc, vc, _, _ = step_case(lens, H, G, d, cap, window, sinks, dtype, fill=0.0)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    args = (q.to(DEV), kn.to(DEV), vn.to(DEV))
    k0, v0 = kc.to(DEV), vc.to(DEV)
    want = ops.window_attention_step(*args, k0, v0, n, H, G, window, sinks)
    both = torch.stack((kc, vc), 2).to(DEV)
    major = [t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1) for t in (kc, vc)]
    odd = torch.zeros((2, 3, cap, G * d + 1), dtype=dtype, device=DEV)
    odd[0, ..., 1:], odd[1, ..., 1:] = kc.to(DEV), vc.to(DEV)
    for k, v in ((both[:, :, 0], both[:, :, 1]), major, (odd[0, ..., 1:], odd[1, ..., 1:])):
        got = ops.window_attention_step(*args, k, v, n, H, G, window, sinks)
        torch.testing.assert_close(got.float(), want.float(), rtol=2.0 ** -6 if dtype == BF else 1e-5,
                                   atol=2.0 ** -6 if dtype == BF else 1e-5)
        assert torch.equal(k, k0) and torch.equal(v, v0)
    wide = torch.zeros((3, 2 * G * d), dtype=dtype, device=DEV)
    wide[:, :G * d], wide[:, G * d:] = args[1], args[2]
    got = ops.window_attention_step(args[0], wide[:, :G * d], wide[:, G * d:], k0, v0, n, H, G, window, sinks)
    assert torch.equal(got, want)


def test_step_offsets_beyond_32_bits():
    """A cache of more than 2^32 elements: the last sequence's rows lie behind the 32-bit range."""
    R, cap, G, d = 3, 1 << 21, 12, 128     # 3 x 3.2 G elements of bf16, keys only once
    free, _ = torch.cuda.mem_get_info()
    if free < 48 << 30:
        pytest.skip("needs 48 GiB of free memory")
    g = torch.Generator().manual_seed(9)
    cache = torch.zeros((R, cap, G * d), dtype=BF, device=DEV)
    n = torch.tensor([cap, 1, cap - 5], dtype=torch.int32, device=DEV)
    rowk = rnd((300, G * d), BF, g).to(DEV)
    cache[2, cap - 5 - 300:cap - 5] = rowk
    cache[0, cap - 300:] = rowk
    q = rnd((1, G * d), BF, g).to(DEV).expand(R, -1).contiguous()
    o = ops.window_attention_step(q, None, None, cache, cache, n, G, G, 300, 0)
    small = torch.zeros((1, 300, G * d), dtype=BF, device=DEV)
    small[0] = rowk
    want = ops.window_attention_step(q[:1], None, None, small, small, torch.tensor([300], dtype=torch.int32, device=DEV), G, G, 300, 0)
    torch.testing.assert_close(o[2:].float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    torch.testing.assert_close(o[:1].float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -6)


# ------------------------------------------------------------------------------ used together
def block(x, pos, w, f, H, G, d, gq, gk, **kw):
    """norm + rotation + windowed attention of the fused projection rows x (T, (H + 2 G) d)."""
    q, k, v = x[:, :H * d], x[:, H * d:(H + G) * d], x[:, (H + G) * d:]
    q, k = ops.qk_norm_rotary(q, k, gq, gk, pos, f, H, G)
    return q, k, v, ops.window_attention(q, k, v, n_head=H, n_kv_head=G, window=w, **kw)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_training_and_generation_agree(dtype):
    """A text attended as a whole, and the same text token by token over a ring cache of sinks + window slots."""
    g = torch.Generator().manual_seed(12)
    n, H, G, d, window, sinks = 180, 4, 2, 64, 48, 4
    f = ops.RotaryFrequencies(64, device=DEV, scaling="yarn", factor=4.0, trained_len=64)
    x = rnd((n, (H + 2 * G) * d), dtype, g).to(DEV)
    gq, gk = (1 + 0.1 * torch.randn(d, generator=g)).to(DEV), (1 + 0.1 * torch.randn(d, generator=g)).to(DEV)
    pos = torch.arange(n, device=DEV)
    _, _, v, whole = block(x, pos, window, f, H, G, d, gq, gk, B=1, Lq=n, Lk=n, sinks=sinks)
    cap = window + sinks
    kc = torch.full((1, cap, G * d), float("nan"), dtype=dtype, device=DEV)
    vc = kc.clone()
    for t in range(n):
        q1, k1 = ops.qk_norm_rotary(x[t:t + 1, :H * d], x[t:t + 1, H * d:(H + G) * d], gq, gk, pos[t:t + 1], f, H, G)
        o = ops.window_attention_step(q1, k1, v[t:t + 1].contiguous(), kc, vc, torch.tensor([t + 1], dtype=torch.int32, device=DEV), H, G,
                                      window, sinks)
        # same inputs bit for bit; both within the bounds of test_window_attention of one exact value
        torch.testing.assert_close(o[0].float(), whole[t].float(), rtol=3 * unit(dtype) + 1e-5, atol=4 * unit(dtype) * 3 + 1e-5)


@pytest.mark.parametrize("dtype", [F32, BF])
def test_block_gradients(dtype):
    """Gradients through norm, rotation and attention against the tape in 64 bits."""
    g = torch.Generator().manual_seed(13)
    n, H, G, d, window, sinks = 140, 4, 2, 64, 30, 3
    f = ops.RotaryFrequencies(32, device=DEV)
    x, do = rnd((n, (H + 2 * G) * d), dtype, g), rnd((n, H * d), dtype, g)
    gq, gk = 1 + 0.1 * torch.randn(d, generator=g), 1 + 0.1 * torch.randn(d, generator=g)
    pos = torch.arange(n) + 1000
    leaves = [t.to(DEV).requires_grad_() for t in (x, gq, gk)]
    *_, o = block(leaves[0], pos.to(DEV), window, f, H, G, d, leaves[1], leaves[2], B=1, Lq=n, Lk=n, sinks=sinks)
    got = (o,) + torch.autograd.grad(o, leaves, do.to(DEV))
    x64, q64, k64 = (t.double().requires_grad_() for t in (x, gq, gk))
    y = x64.view(n, -1, d)
    q, _ = norm64(y[:, :H], q64, 1e-6, pos, f, 32, False)
    k, _ = norm64(y[:, H:H + G], k64, 1e-6, pos, f, 32, False)
    v = y[:, H + G:]
    s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(H // G, 1)) * d ** -0.5
    p = torch.softmax(s.masked_fill(~visible(n, n, window, sinks, True), -math.inf), -1)
    want = torch.einsum("hij,jhd->ihd", p, v.repeat_interleave(H // G, 1)).reshape(n, -1)
    ref = (want.detach(),) + torch.autograd.grad(want, (x64, q64, k64), do.double())
    for a, b, name in zip(got, ref, ("o", "dx", "dgamma_q", "dgamma_k")):
        # bf16: six roundings (q, k, P, o, dS, dq or dk) of 2^-8 on sums whose terms cancel to about a quarter of their size
        tol = (6 * 4 * unit(BF) if dtype == BF else 2e-5) * b.abs().max().item()
        assert (a.double().cpu() - b).abs().max().item() <= tol, name


# ------------------------------------------------------------------------------ streams, graphs
def test_other_stream_and_captured_graph():
    """Forward, backward and a step captured once and replayed on new inputs, between eager calls on another stream."""
    g = torch.Generator().manual_seed(14)
    n, H, G, d, window, sinks, cap = 300, 4, 2, 64, 50, 4, 5000
    f = ops.RotaryFrequencies(64, device=DEV)
    pos = torch.arange(n, device=DEV)
    x = rnd((n, (H + 2 * G) * d), BF, g).to(DEV)
    do = rnd((n, H * d), BF, g).to(DEV)
    gq, gk = torch.ones(d, device=DEV), torch.ones(d, device=DEV)
    kc, vc = rnd((1, cap, G * d), BF, g).to(DEV), rnd((1, cap, G * d), BF, g).to(DEV)
    length = torch.tensor([4500], dtype=torch.int32, device=DEV)

    def work():
        leaf = x.detach().requires_grad_()
        a, b = gq.detach().requires_grad_(), gk.detach().requires_grad_()
        q, k, v, o = block(leaf, pos, window, f, H, G, d, a, b, B=1, Lq=n, Lk=n, sinks=sinks)
        grads = torch.autograd.grad(o, (leaf, a, b), do)
        with torch.no_grad():
            one = ops.window_attention_step(q[:1], k[:1], v[:1].contiguous(), kc, vc, length, H, G, 4096, sinks)
        return (o.detach(), one) + grads

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = work()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(warm, work()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in range(3):
        gen = torch.Generator().manual_seed(100 + seed)
        x.copy_(rnd(x.shape, BF, gen))
        length.fill_(4500 + 7 * seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = work()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_two_graphs_share_a_pool():
    """Two graphs whose workspaces are the same memory, replayed in turn on new inputs: nothing is carried between calls."""
    g = torch.Generator().manual_seed(15)
    H, G, d, sinks, cap = 4, 2, 64, 3, 5000
    do = rnd((400, H * d), BF, g).to(DEV)
    x = rnd((400, (H + 2 * G) * d), BF, g).to(DEV)
    kc, vc = rnd((1, cap, G * d), BF, g).to(DEV), rnd((1, cap, G * d), BF, g).to(DEV)
    length = torch.tensor([4500], dtype=torch.int32, device=DEV)

    def work(n, window):
        leaf = x[:n].detach().requires_grad_()
        q, k, v = leaf[:, :H * d], leaf[:, H * d:(H + G) * d], leaf[:, (H + G) * d:]
        o = ops.window_attention(q, k, v, 1, n, n, H, G, window, sinks)
        grad, = torch.autograd.grad(o, leaf, do[:n])
        return o.detach(), grad, ops.window_attention_step(x[:1, :H * d], None, None, kc, vc, length, H, G, 100 * window, sinks)

    cases, graphs = ((400, 30), (150, 40)), []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in cases:
            work(*c)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    pool = torch.cuda.graph_pool_handle()
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = work(*c)
        graphs.append((graph, out))
    for seed in range(3):
        x.copy_(rnd(x.shape, BF, torch.Generator().manual_seed(200 + seed)))
        for (graph, out), c in zip(graphs, cases):
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            want = work(*c)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (seed, c)


# ------------------------------------------------------------------------------ odd calls
def test_no_second_derivative():
    f = ops.RotaryFrequencies(8, device=DEV)
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    gamma = torch.ones(16, device=DEV)
    pos = torch.arange(6, device=DEV)
    for y in (ops.rotary(x, None, pos, f, 2)[0], ops.qk_norm_rotary(x, None, gamma, None, pos, f, 2)[0],
              ops.window_attention(x, x, x, 1, 6, 6, 2)):
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_masks_may_not_change_before_the_backward_pass():
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    pad = torch.zeros((1, 6), dtype=torch.uint8, device=DEV)
    off = torch.tensor([0, 6], dtype=torch.int32, device=DEV)
    for y, t in ((ops.window_attention(x, x, x, 1, 6, 6, 2, key_pad=pad), pad),
                 (ops.window_attention(x, x, x, 1, 6, 6, 2, q_off=off, k_off=off.clone()), off)):
        t.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 37])
def test_window_lengths_given_as_any_upper_bound(d, dtype):
    """Packed rows: longest lengths far beyond the rows (and 32 bits) change nothing."""
    g = torch.Generator().manual_seed(16)
    q, k, v, do = (rnd((90, 2 * d), dtype, g).to(DEV) for _ in range(4))
    off = torch.tensor([0, 70, 70, 85], dtype=torch.int32, device=DEV)
    res = []
    for L in (70, 1 << 33):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        o = ops.window_attention(*leaves, 3, L, L, 2, None, 20, 2, q_off=off, k_off=off)
        res.append((o,) + torch.autograd.grad(o, leaves, do))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 37])
def test_nan_query_stays_in_its_row(d, dtype):
    """A query with a NaN gives a row of NaN, and every other row what it gives without it."""
    g = torch.Generator().manual_seed(17)
    n, H = 200, 2
    q, k, v = (rnd((n, H * d), dtype, g).to(DEV) for _ in range(3))
    want = ops.window_attention(q, k, v, 1, n, n, H, None, 40, 2)
    bad = q.clone()
    bad[77, d + 3] = float("nan")
    got = ops.window_attention(bad, k, v, 1, n, n, H, None, 40, 2)
    assert got[77, d:].isnan().all()
    got[77, d:] = want[77, d:]
    assert torch.equal(got, want)
    big = q.clone()   # nor do large scores change what other rows get, to the last bit
    big[77] *= 300
    got = ops.window_attention(big, k, v, 1, n, n, H, None, 40, 2)
    got[77] = want[77]
    assert torch.equal(got, want)
    # one step, one split and several, with positions in one split only and in all
    for cap, lens in ((64, [1, 60, 64]), (6000, [1, 50, 5000])):
        kc, vc = rnd((3, cap, H * d), dtype, g).to(DEV), rnd((3, cap, H * d), dtype, g).to(DEV)
        for r in range(3):
            length = torch.tensor(lens, dtype=torch.int32, device=DEV)
            want = ops.window_attention_step(q[:3], None, None, kc, vc, length, H)
            bad = q[:3].clone()
            bad[r, 5] = float("nan")
            got = ops.window_attention_step(bad, None, None, kc, vc, length, H)
            assert got[r, :d].isnan().all(), (cap, r)
            got[r, :d] = want[r, :d]
            assert torch.equal(got, want), (cap, r)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 37])
def test_query_gradient_depends_on_its_own_row(d, dtype):
    """Other queries and output gradients change nothing in a row of dQ, to the last bit."""
    g = torch.Generator().manual_seed(19)
    n, H = 150, 2
    q, k, v, do = (rnd((n, H * d), dtype, g).to(DEV) for _ in range(4))

    def dq(q, do):
        leaf = q.clone().requires_grad_()
        return torch.autograd.grad(ops.window_attention(leaf, k, v, 1, n, n, H, None, 60, 1), leaf, do)[0]

    want = dq(q, do)
    q2, do2 = q.clone(), do.clone()
    q2[40:44] *= 100
    do2[3] = 1000
    got = dq(q2, do2)
    for r in (3, 40, 41, 42, 43):
        got[r] = want[r]
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [0.0, 1e-35, -0.2])
def test_window_scales(scale):
    """A scale of nothing and next to it (every visible key counts alike), and a negative one."""
    run_window([90], [90], 2, 1, 64, 20, 2, True, BF, "dense", scale=scale)


def test_step_scale_of_nothing():
    g = torch.Generator().manual_seed(18)
    kc, vc = rnd((1, 600, 64), BF, g).to(DEV), rnd((1, 600, 64), BF, g).to(DEV)
    length = torch.tensor([600], dtype=torch.int32, device=DEV)
    for scale in (0.0, 1e-35):
        o = ops.window_attention_step(kc[0, :1] * 3, None, None, kc, vc, length, 1, scale=scale)
        want = vc[0].double().mean(0)
        # the mean of 600 values in fp32 (n E of their mean size), rounded once
        bound = want.abs() * unit(BF) + 700 * E * vc[0].double().abs().mean(0)
        check(o[0], want, bound, scale)


# ------------------------------------------------------------------------------ infinities at visible positions of a cache
def step_without(dead, n, d, dtype, shift=0, H=2):
    """A cache of n positions, those in `dead` with scores of -inf: the result is that of the others, within its bound."""
    g = torch.Generator().manual_seed(n + d)
    q = rnd((1, H * d), dtype, g).abs() + 0.1
    kc, vc = rnd((1, n, H * d), dtype, g), rnd((1, n, H * d), dtype, g)
    for h in range(H):
        kc[0, dead, h * d] = -math.inf
    alive = torch.ones(n, dtype=torch.bool)
    alive[dead] = False
    want, bound = torch.zeros((1, H * d), dtype=torch.float64), torch.full((1, H * d), TINY, dtype=torch.float64)
    for h in range(H):
        s = slice(h * d, h * d + d)
        vis = torch.ones((1, int(alive.sum())), dtype=torch.bool)
        (o, eo), *_ = attention64(q[:, s], kc[0, alive][:, s], vc[0, alive][:, s], q[:, s], vis, d ** -0.5, dtype)
        want[:, s], bound[:, s] = o, bound[:, s] + eo
    wide = torch.zeros((2, 1, n, H * d + shift), dtype=dtype, device=DEV)
    k, v = wide[0, ..., shift:], wide[1, ..., shift:]
    k.copy_(kc), v.copy_(vc)
    o = ops.window_attention_step(q.to(DEV), None, None, k, v, torch.tensor([n], dtype=torch.int32, device=DEV), H)
    check(o, want, bound, (n, d, shift))


# one position alone in a wave's first pass; a wave's whole first pass; all passes of a wave, of a split; all but one position
DEAD = [(65, [64]), (200, list(range(64))), (200, list(range(64, 128))), (700, list(range(256))), (6000, list(range(100, 4000))),
        (300, list(range(299)))]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d,shift", [(37, 0), (64, 1)])
@pytest.mark.parametrize("n,dead", DEAD)
def test_step_scores_of_minus_infinity_on_odd_rows(n, dead, d, shift, dtype):
    step_without(dead, n, d, dtype, shift)


def test_step_without_any_finite_score_gives_zeros():
    """As a row of window_attention whose scores are all -inf, on odd rows and on whole 16-byte pieces."""
    for d in (37, 64):
        for n in (65, 6000):
            k = torch.full((1, n, d), -math.inf, dtype=BF, device=DEV)
            v = torch.ones((1, n, d), dtype=BF, device=DEV)
            q = torch.ones((1, d), dtype=BF, device=DEV)
            o = ops.window_attention_step(q, None, None, k, v, torch.tensor([n], dtype=torch.int32, device=DEV), 1)
            assert not o.any(), (d, n)
            assert torch.equal(o, ops.window_attention(q, k[0], v[0], 1, 1, n, 1)), (d, n)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [8, 64, 72, 80, 96, 128])
@pytest.mark.parametrize("n,dead", DEAD)
def test_step_scores_of_minus_infinity(n, dead, d, dtype):
    """Head sizes below the width they are computed at: the infinity is the head's first element."""
    step_without(dead, n, d, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [37, 64, 80])
@pytest.mark.parametrize("n,at", [(1, 0), (5, 0), (33, 32), (129, 128), (40, 32), (40, 35), (6000, 5999)])
def test_step_infinite_value(n, at, d, dtype):
    """An infinity in a visible value is one in its column of the output, and nothing but that."""
    g = torch.Generator().manual_seed(n)
    q, kc, vc = rnd((1, d), dtype, g).to(DEV), rnd((1, n, d), dtype, g).to(DEV), rnd((1, n, d), dtype, g).to(DEV)
    length = torch.tensor([n], dtype=torch.int32, device=DEV)
    want = ops.window_attention_step(q, None, None, kc, vc, length, 1)
    vc[0, at, 3] = math.inf
    got = ops.window_attention_step(q, None, None, kc, vc, length, 1)
    want[0, 3] = math.inf
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------ one row, whose stride says nothing
def one_row(x):
    """The same (1, w) row with a row stride of 1, which torch calls contiguous."""
    return x.view(-1, 1).t()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_row_of_any_stride(dtype):
    g = torch.Generator().manual_seed(20)
    H, d = 2, 64
    f = ops.RotaryFrequencies(64, device=DEV)
    pos = torch.tensor([7], device=DEV)
    x, y, z, do = (rnd((1, H * d), dtype, g).to(DEV) for _ in range(4))
    gamma = torch.ones(d, device=DEV)
    calls = (lambda a, b, c: ops.rotary(a, b, pos, f, H)[0], lambda a, b, c: ops.qk_norm_rotary(a, b, gamma, gamma, pos, f, H)[0],
             lambda a, b, c: ops.window_attention(a, b, c, 1, 1, 1, H))
    for call in calls:
        leaves = [t.clone().requires_grad_() for t in (x, y, z)]
        want = call(*leaves)
        (dx,) = torch.autograd.grad(want, leaves[0], do)
        odd = [one_row(t).requires_grad_() for t in (x, y, z)]
        assert odd[0].stride() == (1, 1)
        got = call(*odd)
        assert torch.equal(got, want)
        assert torch.equal(torch.autograd.grad(got, odd[0], do)[0], dx)
        got = call(*leaves)   # gradients as autograd hands them over: strides (1, 1) and (0, 1)
        assert torch.equal(torch.autograd.grad(got.t().contiguous(), leaves[0], do.t())[0], dx)
        got = call(*leaves)
        assert torch.equal(torch.autograd.grad(got.sum(0), leaves[0], do[0])[0], dx)
    kc, vc = rnd((1, 9, H * d), dtype, g).to(DEV), rnd((1, 9, H * d), dtype, g).to(DEV)
    length = torch.tensor([9], dtype=torch.int32, device=DEV)
    want = ops.window_attention_step(x, y, z, kc, vc, length, H)
    assert torch.equal(ops.window_attention_step(one_row(x), one_row(y), one_row(z), kc, vc, length, H), want)
    # caches of one position: its stride says nothing either
    k1, v1 = kc[:, :1].clone(), vc[:, :1].clone()
    length.fill_(1)
    want = ops.window_attention_step(x, y, z, k1, v1, length, H)
    k2, v2 = (t.reshape(1, -1, 1).transpose(1, 2) for t in (torch.zeros_like(k1), torch.zeros_like(v1)))
    assert k2.shape == k1.shape and k2.stride(1) < H * d
    assert torch.equal(ops.window_attention_step(x, y, z, k2, v2, length, H), want)
    assert torch.equal(k2, k1) and torch.equal(v2, v1)


# ------------------------------------------------------------------------------ many first keys
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n,m,sinks", [(200, 200, 200), (200, 200, 1000), (150, 90, 90), (70, 260, 260)])
def test_window_all_keys_are_sinks(n, m, sinks, causal, dtype):
    """Every key stays visible: windows no longer matter to the past."""
    run_window([n], [m], 2, 1, 64, 5, sinks, causal, dtype, "dense", seed=9)


def many_sinks(B, n, H, G, d, window, sinks, dtype, packed, causal=True):
    """A few rows of every gradient in 64 bits, all of the others through the same call on fewer heads at a time."""
    g = torch.Generator().manual_seed(22)
    T = B * n
    q, k, v, do = rnd((T, H * d), dtype, g), rnd((T, G * d), dtype, g), rnd((T, G * d), dtype, g), rnd((T, H * d), dtype, g)
    off = torch.arange(0, T + 1, n, dtype=torch.int32, device=DEV) if packed else None
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o = ops.window_attention(*leaves, B, n, n, H, G, window, sinks, causal, q_off=off, k_off=off)
    grads = torch.autograd.grad(o, leaves, do.to(DEV))
    for b, h in ((0, 0), (B - 1, H - 1)):
        kh, rs = h // (H // G), slice(b * n, b * n + n)
        vis = visible(n, n, window, sinks, causal)
        want = [torch.zeros((n, d), dtype=torch.float64) for _ in range(4)]
        bound = [torch.full((n, d), TINY, dtype=torch.float64) for _ in range(4)]
        for hh in range(kh * (H // G), (kh + 1) * (H // G)):
            hs, ks = slice(hh * d, hh * d + d), slice(kh * d, kh * d + d)
            res = attention64(q[rs, hs], k[rs, ks], v[rs, ks], do[rs, hs], vis, d ** -0.5, dtype)
            for i in range(4):
                if i >= 2 or hh == h:
                    want[i] += res[i][0]
                    bound[i] += res[i][1]
        for i, (got, x) in enumerate(zip((o,) + grads, (h, h, kh, kh))):
            check(got[rs, x * d:x * d + d], want[i], bound[i], ("o", "dq", "dk", "dv")[i])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("case", [  # B, n, H, G, d, window, sinks: longer chunks, fewer of them, and none
    (4, 1400, 16, 16, 128, 20, 700), (6, 1100, 16, 16, 64, 9, 1000), (24, 700, 16, 16, 128, 33, 650), (12, 1000, 32, 16, 96, 33, 777)])
def test_window_many_sinks(case, dtype):
    many_sinks(*case, dtype, packed=False)


def test_window_many_sinks_packed_both_ways():
    many_sinks(12, 1000, 16, 16, 128, 33, 990, BF, packed=True, causal=False)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows", [70, 3000])
def test_window_queries_in_cuts_inside_a_larger_tensor(rows, dtype):
    """Few packed queries before many keys, further rows around them: the result of the queries alone, zeros elsewhere."""
    g = torch.Generator().manual_seed(23)
    H, d, n, m = 2, 64, 40, 3000
    q, do = (rnd((rows, H * d), dtype, g).to(DEV) for _ in range(2))
    k, v = (rnd((m, H * d), dtype, g).to(DEV) for _ in range(2))
    first = rows - n - 9
    q_off, k_off = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([first, first + n], [0, m]))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ops.window_attention(*leaves, 1, n, m, H, q_off=q_off, k_off=k_off)
    got = (o,) + torch.autograd.grad(o, leaves, do)
    few = slice(first, first + n)
    alone = [q[few].clone().requires_grad_(), k.clone().requires_grad_(), v.clone().requires_grad_()]
    o = ops.window_attention(*alone, 1, n, m, H)
    want = (o,) + torch.autograd.grad(o, alone, do[few])
    for a, b, name in zip(got, want, ("o", "dq", "dk", "dv")):
        if name in ("o", "dq"):
            assert not a[:first].any() and not a[first + n:].any()
            a = a[few]
        # (cut or not: the same sums in another order; bf16 results are within a step of each other, as each is within
        # test_window_queries_in_cuts' bounds of one exact value)
        torch.testing.assert_close(a.float(), b.float(), rtol=2 * unit(dtype) + 1e-5, atol=(unit(dtype) + 1e-6) * b.abs().max().item())


# ------------------------------------------------------------------------------ batches of nothing
@pytest.mark.parametrize("dtype", [BF, F32])
def test_packed_rows_without_sequences(dtype):
    """No sequence at all, or none with queries, or none with keys, before tensors that hold rows: zeros."""
    g = torch.Generator().manual_seed(21)
    H, d, n, m = 2, 64, 6, 5000
    off = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    for q_off, k_off, Lq, Lk in ((off(0), off(0), n, m), (off(0, 0), off(0, m), 0, m), (off(0, n), off(0, 0), n, 0), (off(2, 2), off(9, 9), 0, 0)):
        for n_kv, sinks in ((H, 0), (1, 300)):
            q, do = rnd((n, H * d), dtype, g).to(DEV).requires_grad_(), rnd((n, H * d), dtype, g).to(DEV)
            k, v = (rnd((m, n_kv * d), dtype, g).to(DEV).requires_grad_() for _ in range(2))
            o = ops.window_attention(q, k, v, q_off.numel() - 1, Lq, Lk, H, n_kv, 4000, sinks, q_off=q_off, k_off=k_off)
            for t in (o,) + torch.autograd.grad(o, (q, k, v), do):
                assert not t.any(), (Lq, Lk, n_kv)
    q, do = rnd((4000, H * d), dtype, g).to(DEV).requires_grad_(), rnd((4000, H * d), dtype, g).to(DEV)
    k, v = (rnd((3, d), dtype, g).to(DEV).requires_grad_() for _ in range(2))
    o = ops.window_attention(q, k, v, 1, 4000, 0, H, 1, q_off=off(0, 4000), k_off=off(0, 0))
    for t in (o,) + torch.autograd.grad(o, (q, k, v), do):
        assert not t.any()


# ------------------------------------------------------------------------------ gradients of rows that see few keys
def few_keys64(q, k, v, do, vis, scale, operands):
    """dq, dk of one sequence and head with bounds that hold delta = sum_j P_j dP_j to fp32: no rounding of the output in them.
    operands: what a value of dS loses as an operand of the last product (0: fp32 arithmetic)."""
    q, k, v, do = (t.double() for t in (q, k, v, do))
    n, d, u = vis.sum(1).max().item(), q.shape[1], unit(BF)
    p = torch.softmax((q @ k.t() * scale).masked_fill(~vis, -math.inf), 1) * vis
    dp = do @ v.t()
    ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
    smax = (q.abs() @ k.abs().t() * abs(scale) * vis).max()
    rel = (2 * (d + 6) * smax + 2 * n + 16) * E          # of a probability, as in attention64
    edp = (d + 2) * E * (do.abs() @ v.abs().t())
    edelta = (p * (dp.abs() * (rel + (n + 2) * E) + edp)).sum(1, keepdim=True)
    # of a probability times a difference: its own error, that of the difference, and one step of its operands' sizes
    eds = ds.abs() * (operands + rel + 4 * E) + p * abs(scale) * (edelta + edp + E * (dp.abs() + (p * dp).sum(1, keepdim=True).abs()))
    acc = (max(vis.shape) + 8) * E
    return ((ds @ k, u * (ds @ k).abs() + eds @ k.abs() + acc * ds.abs() @ k.abs()),
            (ds.t() @ q, u * (ds.t() @ q).abs() + eds.t() @ q.abs() + acc * ds.abs().t() @ q.abs()))


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 0), (1, 1), (5, 2), (8, 24)])
@pytest.mark.parametrize("d,shift", [(64, 0), (128, 0), (37, 0), (64, 1), (100, 0)])
def test_gradients_of_rows_with_few_keys(d, shift, window, sinks):
    """bf16 rows of at most 32 visible keys, on whole 16-byte pieces and on odd rows."""
    g = torch.Generator().manual_seed(24)
    n, H, G = 170, 2, 1
    x = torch.zeros((n, (H + 2 * G) * d + shift), dtype=BF)
    x[:, shift:] = rnd((n, (H + 2 * G) * d), BF, g)
    do = rnd((n, H * d), BF, g)
    cut = lambda t: (t[:, shift:shift + H * d], t[:, shift + H * d:shift + (H + G) * d], t[:, shift + (H + G) * d:])
    leaves = [t.detach().requires_grad_() for t in cut(x.to(DEV))]
    o = ops.window_attention(*leaves, 1, n, n, H, G, window, sinks)
    dq, dk, _ = torch.autograd.grad(o, leaves, do.to(DEV))
    q, k, v = cut(x)
    vis = visible(n, n, window, sinks, True)
    want, bound = torch.zeros((n, d), dtype=torch.float64), torch.full((n, d), TINY, dtype=torch.float64)
    for h in range(H):
        s = slice(h * d, h * d + d)
        a, b = few_keys64(q[:, s], k, v, do[:, s], vis, d ** -0.5, unit(BF) if d % 8 == 0 and shift % 8 == 0 else 0.0)
        check(dq[:, s], a[0], a[1] + TINY, ("dq", h))
        want, bound = want + b[0], bound + b[1]
    check(dk, want, bound, "dk")


# ------------------------------------------------------------------------------ very far positions
@pytest.mark.parametrize("il", [False, True])
@pytest.mark.parametrize("far", [1 << 32, -(1 << 45), (1 << 53) + 1, 1 << 56])
def test_rotary_very_far_positions(far, il):
    """Angles from the formula in 60 digits: off by at most half a unit of 2^-64 turns a position."""
    g = torch.Generator().manual_seed(25)
    T, H, d, rot = 20, 2, 64, 48
    pos = torch.randint(0, 300, (T,), generator=g) + far
    x = rnd((T, H * d), F32, g)
    f = ops.RotaryFrequencies(rot, device=DEV)
    out, _ = ops.rotary(x.to(DEV), None, pos.to(DEV), f, H, interleaved=il)
    with decimal.localcontext(decimal.Context(prec=60)):
        turn = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494")
        ln = decimal.Decimal(10000).ln()
        per = [(-ln * 2 * i / rot).exp() / turn for i in range(rot // 2)]
        ang = torch.tensor([[float(p * t % 1) * 2 * math.pi for t in per] for p in pos.tolist()], dtype=torch.float64)[:, None]
    h = x.double().view(T, H, d)
    a, b = (h[..., 0:rot:2], h[..., 1:rot:2]) if il else (h[..., :rot // 2], h[..., rot // 2:rot])
    y = (a * torch.cos(ang) - b * torch.sin(ang), b * torch.cos(ang) + a * torch.sin(ang))
    m = a.abs() + b.abs()
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if il else (lambda u, v: torch.cat((u, v), -1))
    want = torch.cat((join(*y), h[..., rot:]), -1)
    mag = torch.cat((join(m, m), h[..., rot:].abs()), -1)
    off = pos.abs().max().item() * 2.0 ** -65 * 2 * math.pi + 2.0 ** -50   # (and this reference's own angles)
    check(out, want.view(T, -1), (E * want.abs() + (ROT_E + off) * mag).view(T, -1), "far")


def test_frequencies_may_change_after_the_forward_pass():
    """The gradient is that of the frequencies the forward pass used, or an error where those are gone."""
    g = torch.Generator().manual_seed(26)
    q = rnd((6, 32), F32, g).to(DEV).requires_grad_()
    gamma, pos, w = torch.ones(16, device=DEV), torch.arange(6, device=DEV), rnd((6, 32), F32, g).to(DEV)
    calls = (lambda f: ops.rotary(q, None, pos, f, 2)[0], lambda f: ops.qk_norm_rotary(q, None, gamma, None, pos, f, 2)[0])
    make = lambda: ops.RotaryFrequencies(16, device=DEV, scaling="yarn", factor=4.0, trained_len=64)
    other = ops.RotaryFrequencies(16, device=DEV, base=77.0)
    for call in calls:
        want, = torch.autograd.grad(call(make()), q, w)
        f = make()
        y = call(f)
        f.turns, f.amplitude, f.rot_dim = other.turns, 9.0, 8
        assert torch.equal(torch.autograd.grad(y, q, w)[0], want)
        f = make()
        y = call(f)
        f.turns.copy_(other.turns)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, q, w)


@pytest.mark.parametrize("live", [range(0, 9), range(1990, 2000), range(3, 1990, 150), [700], [], range(1200, 1240)])
@pytest.mark.parametrize("d", [64, 128, 37])
def test_gradients_where_padding_leaves_few_keys(d, live):
    """Few queries before keys that are nearly all padding: the keys are cut, and rows of few keys keep their delta."""
    g = torch.Generator().manual_seed(27)
    n, m, H = 40, 2000, 1
    q, do, k, v = (rnd((r, d), BF, g) for r in (n, n, m, m))
    pads = torch.ones((1, m), dtype=torch.uint8)
    pads[0, list(live)] = 0
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    o = ops.window_attention(*leaves, 1, n, m, H, causal=False, key_pad=pads.to(DEV))
    dq, dk, _ = torch.autograd.grad(o, leaves, do.to(DEV))
    if len(live) == 0:
        assert not dq.any() and not dk.any()
        return
    keep = list(live)
    vis = torch.ones((n, len(keep)), dtype=torch.bool)
    if len(keep) <= 32:
        a, b = few_keys64(q, k[keep], v[keep], do, vis, d ** -0.5, unit(BF) if d % 8 == 0 else 0.0)
    else:
        _, a, b, _ = attention64(q, k[keep], v[keep], do, vis, d ** -0.5, BF)
    check(dq, a[0], a[1] + TINY, "dq")
    check(dk[keep], b[0], b[1] + TINY, "dk")
    assert not dk[pads[0].bool().to(DEV)].any()


# ------------------------------------------------------------------------------ calls side by side
def test_threads_and_streams_side_by_side():
    """Four threads, each on a stream of its own, run the operators on their own tensors at once: each gets what it gets alone."""
    H, G, d, sinks, cap = 4, 2, 64, 3, 5000
    f = ops.RotaryFrequencies(64, device=DEV)

    def case(seed):
        g = torch.Generator().manual_seed(seed)
        n, window, dtype = 150 + 40 * seed, 30 + seed, (BF, F32)[seed % 2]
        x, do = rnd((n, (H + 2 * G) * d), dtype, g).to(DEV), rnd((n, H * d), dtype, g).to(DEV)
        gq, gk = (1 + 0.1 * torch.randn(d, generator=g)).to(DEV), torch.ones(d, device=DEV)
        kc, vc = rnd((1, cap, G * d), dtype, g).to(DEV), rnd((1, cap, G * d), dtype, g).to(DEV)
        length, pos = torch.tensor([4500 + seed], dtype=torch.int32, device=DEV), torch.arange(n, device=DEV)

        def work():
            leaf = x.detach().requires_grad_()
            q, k, v, o = block(leaf, pos, window, f, H, G, d, gq, gk, B=1, Lq=n, Lk=n, sinks=sinks)
            few = ops.window_attention(q[-5:], k.repeat(20, 1), v.repeat(20, 1), 1, 5, 20 * n, H, G)   # keys cut over blocks
            grad, = torch.autograd.grad((o, few), leaf, (do, do[-5:]))
            with torch.no_grad():
                return o.detach(), few.detach(), grad, ops.window_attention_step(q[:1], k[:1], v[:1], kc, vc, length, H, G, 4096, sinks)

        return work

    works = [case(s) for s in range(4)]
    want = [w() for w in works]
    torch.cuda.synchronize()
    wrong = []

    def thread(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = works[i]()
                stream.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("d", [64, 80, 128, 37])
def test_window_scores_of_minus_infinity(d, dtype):
    """Keys whose score is -inf to every query count for nothing, whole tiles of them and single ones."""
    g = torch.Generator().manual_seed(28)
    n, m = 90, 400
    q, k, v = rnd((n, d), dtype, g).abs() + 0.1, rnd((m, d), dtype, g), rnd((m, d), dtype, g)
    alive = torch.ones(m, dtype=torch.bool)
    alive[list(range(64, 200)) + list(range(201, 399, 2)) + [0, 399]] = False
    k[~alive, 0] = -math.inf
    o = ops.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), 1, n, m, 1, causal=False)
    vis = torch.ones((n, int(alive.sum())), dtype=torch.bool)
    (want, bound), *_ = attention64(q, k[alive], v[alive], q, vis, d ** -0.5, dtype)
    check(o, want, bound + TINY, "o")


@pytest.mark.parametrize("n,window,sinks,causal", [(150, 30, 2, True), (260, 70, 0, False), (64, None, 0, True)])
@pytest.mark.parametrize("shift", [1, 3, 4])
def test_window_bf16_rows_off_their_pieces(shift, n, window, sinks, causal):
    """bf16 heads of 64 in rows that are not 16-byte aligned: the bounds of test_window_attention."""
    g = torch.Generator().manual_seed(29)
    H, G, d = 4, 2, 64
    x = torch.zeros((n, (H + 2 * G) * d + shift), dtype=BF)
    x[:, shift:] = rnd((n, (H + 2 * G) * d), BF, g)
    do = torch.zeros((n, H * d + shift), dtype=BF)
    do[:, shift:] = rnd((n, H * d), BF, g)
    cut = lambda t: (t[:, shift:shift + H * d], t[:, shift + H * d:shift + (H + G) * d], t[:, shift + (H + G) * d:])
    leaves = [t.detach().requires_grad_() for t in cut(x.to(DEV))]
    o = ops.window_attention(*leaves, 1, n, n, H, G, window, sinks, causal)
    got = (o,) + torch.autograd.grad(o, leaves, do.to(DEV)[:, shift:])
    q, k, v = cut(x)
    want = [torch.zeros((n, w * d), dtype=torch.float64) for w in (H, H, G, G)]
    bound = [torch.full_like(t, TINY) for t in want]
    for h in range(H):
        hs, ks = slice(h * d, h * d + d), slice(h // 2 * d, h // 2 * d + d)
        res = attention64(q[:, hs], k[:, ks], v[:, ks], do[:, shift:][:, hs], visible(n, n, window or 1 << 30, sinks, causal), d ** -0.5, BF)
        for i, cs in enumerate((hs, hs, ks, ks)):
            want[i][:, cs] += res[i][0]
            bound[i][:, cs] += res[i][1]
    for a, w, b, name in zip(got, want, bound, ("o", "dq", "dk", "dv")):
        check(a, w, b, name)


@pytest.mark.parametrize("dtype,n,sinks", [(BF, 5000, 3300), (F32, 4500, 4100)])
def test_window_many_sinks_under_few_key_heads(dtype, n, sinks):
    """Key tiles in parts and bounded chunks of far queries at once."""
    H, G, d, window = 4, 1, 128, 20
    g = torch.Generator().manual_seed(30)
    q, do = (rnd((n, H * d), dtype, g).to(DEV) for _ in range(2))
    k, v = (rnd((n, d), dtype, g).to(DEV) for _ in range(2))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o = ops.window_attention(*leaves, 1, n, n, H, G, window, sinks)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    vis = visible(n, n, window, sinks, True).to(DEV)
    sums = [torch.zeros((n, d), dtype=torch.float64, device=DEV) for _ in range(4)]
    for h in range(H):
        s = slice(h * d, h * d + d)
        res = attention64(q[:, s], k, v, do[:, s], vis, d ** -0.5, dtype)
        check(o[:, s], *res[0], ("o", h))
        check(dq[:, s], *res[1], ("dq", h))
        for i, x in enumerate(res[2] + res[3]):
            sums[i] += x
    check(dk, sums[0], sums[1], "dk")
    check(dv, sums[2], sums[3], "dv")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("B,Lq,Lk", [(0, 5, 5), (3, 0, 5), (3, 5, 0), (3, 0, 0), (0, 0, 0)])
def test_padded_batches_of_nothing(B, Lq, Lk, dtype):
    q, do = torch.ones((B * Lq, 128), dtype=dtype, device=DEV).requires_grad_(), torch.ones((B * Lq, 128), dtype=dtype, device=DEV)
    k, v = (torch.ones((B * Lk, 64), dtype=dtype, device=DEV).requires_grad_() for _ in range(2))
    pad = torch.zeros((B, Lk), dtype=torch.bool, device=DEV)
    o = ops.window_attention(q, k, v, B, Lq, Lk, 2, 1, 3, 2, key_pad=pad)
    assert o.shape == (B * Lq, 128)
    for t in (o,) + torch.autograd.grad(o, (q, k, v), do):
        assert not t.any()
