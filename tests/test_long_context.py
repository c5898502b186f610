"""Refusals of the rotary / query-key norm / windowed-attention operators, on the CPU, and what their frequency tables
hold."""
import decimal
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from specialk_amd import _lib as L
from specialk_amd import ops


def rows(n, w, dtype=torch.float32):
    return torch.zeros((n, w), dtype=dtype)


def freqs(rot=16, **kw):
    return ops.RotaryFrequencies(rot, device="cpu", **kw)


# ------------------------------------------------------------------------------ frequencies
def test_turns_are_the_frequencies_as_fractions_of_a_turn():
    f = freqs(64)
    for i, w in enumerate(f.turns.tolist()):
        assert 0 <= w < 1 << 62
        # a double holds the frequency to 2^-53; the word adds at most half a unit of 2^-64 turns
        want = 10000.0 ** (-2.0 * i / 64) / (2 * math.pi)
        assert abs(w / 2.0 ** 64 - want) <= want * 2.0 ** -50 + 2.0 ** -65


def formula(rot, base, scaling, factor, trained_len):
    """Turns per position of every pair, to 70 digits, from the formulas: logarithms and exponentials instead of powers."""
    with decimal.localcontext(decimal.Context(prec=70)):
        D = decimal.Decimal
        arctan = lambda n: sum(D((-1) ** k) / ((2 * k + 1) * D(n) ** (2 * k + 1)) for k in range(60))
        turn = 8 * (4 * arctan(5) - arctan(239))                     # 2 pi by Machin
        ln = D(base).ln()
        if scaling == "ntk":
            ln += D(factor).ln() * rot / (rot - 2)
        out = []
        for i in range(rot // 2):
            f = (-ln * 2 * i / rot).exp() / turn
            r = trained_len * f                                      # turns within the trained length
            if scaling == "linear" or (scaling == "yarn" and r <= 1):
                f /= D(factor)
            elif scaling == "yarn" and r < 32:                       # between: (r - 1) of 31 parts kept
                f *= ((r - 1) + (32 - r) / D(factor)) / 31
            out.append(f)
        return out


@pytest.mark.parametrize("rot,base", [(4, 10000.0), (64, 10000.0), (36, 500000.0), (128, 1e6)])
@pytest.mark.parametrize("scaling,factor,trained_len", [(None, 1.0, 0), ("linear", 3.7, 0), ("ntk", 8.0, 0), ("yarn", 32.0, 4096),
                                                        ("yarn", 1.5, 131072)])
def test_every_turn_is_its_formula_to_half_a_unit(rot, base, scaling, factor, trained_len):
    f = freqs(rot, base=base, scaling=scaling, factor=factor, trained_len=trained_len)
    want = formula(rot, base, scaling, factor, trained_len)
    assert len(f.turns) == len(want) == rot // 2
    for got, w in zip(f.turns.tolist(), want):
        # rounded once: half a unit of 2^-64, and what 60 digits leave out
        assert abs(got % (1 << 64) - w * (1 << 64)) <= decimal.Decimal("0.5000001")
    assert f.radians == pytest.approx([float(w) * 2 * math.pi for w in want], rel=1e-14)


def test_frequencies_made_in_inference_mode_serve_training():
    with torch.inference_mode():
        f = freqs(8)
    assert not f.turns.is_inference()


def test_frequencies_of_other_number_types():
    want = freqs(64, scaling="yarn", factor=4.0, trained_len=2048, base=10000.0).turns
    for num in (int, np.float32, np.float64, np.int64):
        assert torch.equal(freqs(np.int64(64), scaling="yarn", factor=num(4), trained_len=num(2048), base=num(10000)).turns, want)
    with pytest.raises(ValueError, match="2\\^64"):
        freqs(8, base=1e-300)


@pytest.mark.parametrize("scaling", ["linear", "ntk", "yarn"])
def test_scaling_keeps_and_stretches_the_right_ends(scaling):
    plain, f = freqs(128), freqs(128, scaling=scaling, factor=16.0, trained_len=4096)
    ratio = [a / b for a, b in zip(plain.radians, f.radians)]
    assert ratio[0] == pytest.approx(16.0 if scaling == "linear" else 1.0)
    assert ratio[-1] == pytest.approx(16.0)
    assert all(x <= y * (1 + 1e-12) for x, y in zip(ratio, ratio[1:]))
    assert f.amplitude == pytest.approx(0.1 * math.log(16.0) + 1.0 if scaling == "yarn" else 1.0)


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=-2), dict(rot_dim=8, base=0.0), dict(rot_dim=8, factor=-1.0),
                                dict(rot_dim=8, base=float("nan")), dict(rot_dim=8, scaling="other"),
                                dict(rot_dim=2, scaling="ntk", factor=2.0), dict(rot_dim=8, scaling="yarn", factor=2.0),
                                dict(rot_dim=8, scaling="yarn", factor=0.5, trained_len=64)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        ops.RotaryFrequencies(device="cpu", **kw)


# ------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("x", [torch.arange(8.0).view(8, 1).t(), torch.arange(8.0).expand(1, 8), torch.ones(()).expand(1, 8),
                               torch.zeros(16)[::2].view(1, 8), torch.empty(8, 0).t(), torch.arange(8.0).view(1, 8),
                               torch.zeros(3, 8)[1:2], torch.zeros(8, 3).t(), torch.ones(8).expand(3, 8), torch.zeros(3, 20)[:, 3:11]])
def test_rows_have_a_stride_of_their_length_at_least(x):
    """What torch calls contiguous may have any stride along a dimension of one."""
    y = ops._rows(x, 8, "x")
    assert torch.equal(x, y) and y.stride(1) == 1 and y.stride(0) >= 8
    if x.stride(0) >= 8 and x.stride(1) == 1:
        assert y is x


# ------------------------------------------------------------------------------ rotary, norm
def rotary_args(**kw):
    a = dict(q=rows(5, 64), k=rows(5, 32), pos=torch.arange(5), freqs=freqs(), n_head=4, n_kv_head=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [dict(q=rows(5, 63)), dict(q=rows(5, 64).view(5, 4, 16)), dict(k=rows(4, 32)), dict(k=rows(5, 64)),
                                dict(k=rows(5, 32, torch.bfloat16)), dict(pos=torch.arange(4)),
                                dict(pos=torch.arange(5, dtype=torch.int32)), dict(pos=None), dict(freqs=None),
                                dict(freqs=freqs(18)), dict(n_head=3, n_kv_head=2), dict(n_head=0),
                                dict(q=rows(5, 4 * 258), k=None, freqs=freqs(2))])
def test_rotary_refusals(kw):
    with pytest.raises(ValueError):
        ops.rotary(**rotary_args(**kw))


def test_rotary_types_and_devices():
    with pytest.raises(TypeError):
        ops.rotary(**rotary_args(q=rows(5, 64, torch.float16), k=rows(5, 32, torch.float16)))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.rotary(**rotary_args())


@pytest.mark.parametrize("kw", [dict(gamma_q=torch.ones(8)), dict(gamma_k=torch.ones(16, dtype=torch.bfloat16)),
                                dict(gamma_k=None), dict(k=None), dict(eps=-1.0), dict(eps=float("nan")),
                                dict(gamma_q=torch.ones(32)[::2])])
def test_norm_refusals(kw):
    a = rotary_args(gamma_q=torch.ones(16), gamma_k=torch.ones(16))
    a.update(kw)
    with pytest.raises(ValueError):
        ops.qk_norm_rotary(**a)


# ------------------------------------------------------------------------------ windowed attention
def window_args(**kw):
    a = dict(q=rows(12, 64), k=rows(12, 32), v=rows(12, 32), B=2, Lq=6, Lk=6, n_head=4, n_kv_head=2, window=3, sinks=1)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(q=rows(12, 62)), dict(v=rows(11, 32)), dict(v=rows(12, 64)), dict(k=rows(12, 32, torch.bfloat16)), dict(B=3),
    dict(Lk=5), dict(n_head=4, n_kv_head=3), dict(window=0), dict(window=-4), dict(sinks=-1), dict(B=-1),
    dict(q_off=torch.zeros(3, dtype=torch.int32)), dict(k_off=torch.zeros(3, dtype=torch.int32)),
    dict(q_off=torch.zeros(2, dtype=torch.int32), k_off=torch.zeros(3, dtype=torch.int32)),
    dict(q_off=torch.zeros(3, dtype=torch.int64), k_off=torch.zeros(3, dtype=torch.int64)),
    dict(q_off=torch.zeros(3, dtype=torch.int32), k_off=torch.zeros(3, dtype=torch.int32),
         key_pad=torch.zeros((2, 6), dtype=torch.uint8)),
    dict(key_pad=torch.zeros((2, 5), dtype=torch.uint8)), dict(key_pad=torch.zeros((2, 6), dtype=torch.int32)),
    dict(q=rows(12, 4 * 130), k=rows(12, 2 * 130), v=rows(12, 2 * 130))])
def test_window_refusals(kw):
    with pytest.raises(ValueError):
        ops.window_attention(**window_args(**kw))


def test_window_types_and_devices():
    h = torch.float16
    with pytest.raises(TypeError):
        ops.window_attention(**window_args(q=rows(12, 64, h), k=rows(12, 32, h), v=rows(12, 32, h)))
    with pytest.raises(RuntimeError, match="GPU"):
        ops.window_attention(**window_args())


# ------------------------------------------------------------------------------ one step over a cache
def step_args(**kw):
    a = dict(q=rows(2, 64), k_new=rows(2, 32), v_new=rows(2, 32), k_cache=torch.zeros(2, 10, 32), v_cache=torch.zeros(2, 10, 32),
             kv_len=torch.ones(2, dtype=torch.int32), n_head=4, n_kv_head=2, window=8, sinks=2)
    a.update(kw)
    return a


@pytest.mark.parametrize("kw", [
    dict(window=9), dict(window=0), dict(sinks=3), dict(sinks=-1), dict(sinks=10, window=None), dict(k_new=None),
    dict(v_new=None), dict(k_new=rows(3, 32)), dict(k_new=rows(2, 16)), dict(k_new=rows(2, 32, torch.bfloat16)),
    dict(k_cache=torch.zeros(3, 10, 32)), dict(v_cache=torch.zeros(2, 11, 32)), dict(k_cache=torch.zeros(2, 32)),
    dict(k_cache=torch.zeros(2, 10, 32, dtype=torch.bfloat16)), dict(kv_len=torch.ones(2, dtype=torch.int64)),
    dict(kv_len=torch.ones(3, dtype=torch.int32)), dict(n_head=3), dict(q=rows(2, 63)),
    dict(k_cache=torch.zeros(1, 10, 32).expand(2, 10, 32)),               # rows that share memory
    dict(v_cache=torch.zeros(2, 1, 32).expand(2, 10, 32)),
    dict(k_cache=torch.zeros(2, 10, 64)[:, :, ::2])])
def test_step_refusals(kw):
    with pytest.raises(ValueError):
        ops.window_attention_step(**step_args(**kw))


def test_step_has_no_gradient():
    with pytest.raises(RuntimeError, match="gradient"):
        ops.window_attention_step(**step_args(q=rows(2, 64).requires_grad_()))
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        ops.window_attention_step(**step_args(q=rows(2, 64).requires_grad_()))


# ------------------------------------------------------------------------------ forward mode
@pytest.mark.parametrize("leaf", [False, True])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(grad, leaf):
    """A dual tensor in any place: an error, not a result without a tangent."""
    gammas = dict(gamma_q=torch.ones(16), gamma_k=torch.ones(16))
    calls = ((ops.rotary, rotary_args(), "qk"), (ops.qk_norm_rotary, rotary_args(**gammas), ("q", "k", "gamma_q", "gamma_k")),
             (ops.window_attention, window_args(), "qkv"),
             (ops.window_attention_step, step_args(), ("q", "k_new", "v_new", "k_cache", "v_cache")))
    for fn, args, names in calls:
        if leaf and fn is ops.window_attention_step:
            continue
        for name in names:
            with torch.set_grad_enabled(grad), forward_ad.dual_level():
                x = args[name].clone().requires_grad_(leaf)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    fn(**{**args, name: forward_ad.make_dual(x, torch.ones_like(x))})
                with pytest.raises(RuntimeError, match="GPU"):   # (a level alone changes nothing)
                    fn(**args)


# ------------------------------------------------------------------------------ the C entry points
def test_entry_points_refuse_before_any_launch():
    """Wrong shapes and missing buffers come back as codes with a message (nothing here reaches a GPU)."""
    lib = L.load()
    p = 1 << 20   # stands for a pointer: every call below fails before one is used

    def rot(T=4, H=2, G=1, d=16, rot=8, ldq=32, ldk=16, gq=None, gk=None, inverse=0, dtype=0, q=p, pos=p):
        return lib.skhip_qk_rotary(q, p, p, p, pos, p, 1.0, gq, gk, 0.0, T, H, G, d, rot, ldq, ldk, 32, 16, 0, inverse, dtype, None)

    for kw in (dict(d=257, ldq=1000, ldk=1000), dict(rot=7), dict(rot=18), dict(ldq=31), dict(ldk=15), dict(gq=p),
               dict(gq=p, gk=p, inverse=1), dict(dtype=2), dict(q=None), dict(pos=None), dict(H=0), dict(T=-1)):
        assert rot(**kw) == -1, kw
        assert b"skhip_qk_rotary" in lib.skhip_last_error()
    assert rot(T=0) == 0

    def bwd_norm(ws=None, n=0):
        return lib.skhip_qk_norm_rotary_bwd(p, p, p, p, p, p, p, p, p, p, 1.0, p, p, 0.0, 4, 2, 1, 16, 8, 32, 16, 32, 16, 32, 16, 0,
                                            ws, n, 0, None)

    assert bwd_norm() == -3 and bwd_norm(p, 31) == -3

    def fwd(H=4, G=2, d=16, window=3, sinks=1, ldq=64, ldk=32, B=2, Lq=6, Tq=12, qo=None, ko=None, pad=None, lse=p):
        return lib.skhip_window_attn_fwd(p, p, p, p, lse, pad, qo, ko, B, H, G, Tq, 12, Lq, 6, d, ldq, ldk, 32, 64, 0.25, window,
                                         sinks, 1, None, 0, 0, None)

    for kw in (dict(G=3), dict(d=129, ldq=1000, ldk=1000), dict(window=0), dict(sinks=-1), dict(ldq=63), dict(ldk=31), dict(Tq=11),
               dict(qo=p), dict(qo=p, ko=p, pad=p), dict(lse=None), dict(B=65535, Lq=0, Tq=0),
               dict(qo=p, ko=p, B=65000, Lq=1 << 20)):
        assert fwd(**kw) == -1, kw
        assert b"skhip_window_attn_fwd" in lib.skhip_last_error()

    def step(cap=10, window=8, sinks=2, d=16, kn=p, vn=p, length=p, H=4, pos=32, ws=None, R=2):
        return lib.skhip_window_attn_step(p, kn, vn, p, p, p, length, R, H, 2, d, cap, 64, 32, 64, 320, pos, 320, 32, 0.25, window,
                                          sinks, ws, 0, 0, None)

    for kw in (dict(window=9), dict(sinks=10), dict(kn=None), dict(length=None), dict(H=3), dict(pos=31), dict(d=0), dict(R=65536)):
        assert step(**kw) == -1, kw
    assert step(cap=100000, window=90000) == -3   # several splits, no workspace


def test_workspace_sizes():
    lib = L.load()
    base = 2 * 4 * 12
    # no sinks, or a window that reaches the first key from everywhere: the rows' deltas alone
    assert lib.skhip_window_attn_bwd_ws_floats(2, 4, 2, 12, 6, 6, 16, 3, 0, 1) == base
    assert lib.skhip_window_attn_bwd_ws_floats(2, 4, 2, 12, 6, 6, 16, 100, 2, 1) == base
    assert lib.skhip_window_attn_bwd_ws_floats(2, 4, 2, 12, 6, 6, 16, 3, 2, 1) > base
    # forward: only where few rows see many keys, and then refused without it
    assert lib.skhip_window_attn_fwd_ws_floats(2, 4, 2, 12, 6, 6, 16, 3, 0, 1) == 0
    assert lib.skhip_window_attn_fwd_ws_floats(64, 8, 8, 64 * 2048, 2048, 2048, 64, 2048, 0, 1) == 0
    p = 1 << 20   # stands for a pointer
    need = lib.skhip_window_attn_fwd_ws_floats(1, 2, 2, 3, 3, 8192, 16, 8192, 0, 1)
    assert need > 0
    for ws, n, code in ((None, 0, -3), (p, 1, -3), (p + 4, need, -1)):
        assert lib.skhip_window_attn_fwd(p, p, p, p, p, None, None, None, 1, 2, 2, 3, 8192, 3, 8192, 16, 32, 32, 32, 32, 0.25, 8192,
                                         0, 1, ws, n, 0, None) == code
    assert lib.skhip_window_attn_step_ws_floats(65535, 8, 8, 64, 4096, 4096, 0) == 0
    assert lib.skhip_window_attn_step_ws_floats(1, 8, 8, 64, 4096, 4096, 0) > 0


def test_backward_workspace_of_many_sinks():
    """The sums of the first keys' far queries stay within 2 ^ 24 floats or 4 blocks a CU, however many first keys there are."""
    lib = L.load()
    for B, H, G, n, d, window, sinks in ((1, 8, 8, 32768, 128, 64, 4096), (1, 8, 8, 32768, 128, 1, 32768), (4, 8, 8, 8192, 64, 64, 8191),
                                         (4, 8, 8, 8192, 64, 64, 4096), (1, 32, 8, 32768, 128, 256, 4096),
                                         (1, 8, 8, 32768, 128, 64, 16384), (64, 8, 8, 4096, 64, 100, 500), (1, 1, 1, 1 << 20, 64, 10, 5000)):
        got = lib.skhip_window_attn_bwd_ws_floats(B, H, G, B * n, n, n, d, window, sinks, 1)
        rest = lib.skhip_window_attn_bwd_ws_floats(B, H, G, B * n, n, n, d, window, 0, 1)
        # 256 CUs: 4 * 256 blocks and as many tiles' own windows, each of 128 rows of dK and dV
        assert got - rest <= max(1 << 24, 2 * 4 * 256 * 2 * 128 * d), (got, rest)


def test_workspace_of_few_queries_in_a_large_packed_tensor():
    """Rows outside every sequence are only zeroed: their partial results are not multiplied by the cuts."""
    lib = L.load()
    few = lib.skhip_window_attn_fwd_ws_floats(1, 8, 8, 64, 64, 32768, 128, 32768, 0, 1)
    assert few > 0
    for Tq in (1 << 16, 1 << 20):
        assert lib.skhip_window_attn_fwd_ws_floats(1, 8, 8, Tq, 64, 32768, 128, 32768, 0, 1) <= few * 2, Tq
        back = lib.skhip_window_attn_bwd_ws_floats(1, 8, 8, Tq, 64, 32768, 128, 32768, 0, 1)
        assert back - 2 * 8 * Tq <= 2 * lib.skhip_window_attn_bwd_ws_floats(1, 8, 8, 64, 64, 32768, 128, 32768, 0, 1), Tq


def test_workspace_sizes_of_refused_calls():
    """0, as for every size that a call refuses, not what is left of an overflow."""
    lib, M = L.load(), (1 << 31) - 1
    for q in (lib.skhip_window_attn_fwd_ws_floats, lib.skhip_window_attn_bwd_ws_floats):
        for Lq, Lk, d, H, G in ((M, M, 64, 8, 8), (100, M, 64, 8, 8), ((1 << 29) + 1, 5, 64, 8, 8), (100, 100, 129, 8, 8), (100, 100, 64, 8, 3)):
            for window, sinks in ((M, 0), (M, 3), (60, M), (60, 5)):
                assert q(1, H, G, 100, Lq, Lk, d, window, sinks, 1) == 0, (Lq, Lk, d, H, G, window, sinks)
