"""Workloads of the rotary, query / key norm and windowed-attention operators, with the operators' plain forms.

`listed()` names the workloads, `draw(rng)` makes further ones of the same ranges, `prepare` makes a workload's inputs on
the GPU and `run` makes one pass: through elementary torch operations in 32 bits (own = False) or through the
framework's operators (own = True).  `exact` gives a pass's results from the operators' definitions in 64 bits and
`work` the bytes and operations a pass cannot do without.

Notation: T token rows, n_head query heads sharing n_kv key / value heads of d elements; position p of a query sees key j
when p - j < window or j < sinks, and j <= p (causal) resp. j - p < window (both directions), unless key j is padding.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------ the workloads
def listed():
    return [
        # one new token for each of 640 beam rows (128 sentences x beam 5), base model heads
        dict(name="rotary_step_640", op="rotary", T=640, n_head=8, n_kv=8, d=64, rot=64, interleaved=False, scaling="none",
             factor=1.0, trained_len=0, first_pos=0, last_pos=150, dtype="bf16", backward=False),
        # a long document far behind the trained length: half of each head rotated, neighbouring pairs, shared key heads
        dict(name="rotary_long_fp32", op="rotary", T=16381, n_head=16, n_kv=4, d=128, rot=64, interleaved=True,
             scaling="yarn", factor=32.0, trained_len=4096, first_pos=98304, last_pos=114684, dtype="fp32", backward=True),
        # the same decoding step with normalised heads
        dict(name="qknorm_step_640", op="qk_norm", T=640, n_head=8, n_kv=8, d=64, rot=64, interleaved=False, scaling="none",
             factor=1.0, trained_len=0, first_pos=0, last_pos=150, dtype="bf16", backward=False),
        # the packed target tokens of one training step of the base model (640 sentences), forward and backward
        dict(name="qknorm_train_25487", op="qk_norm", T=25487, n_head=8, n_kv=8, d=64, rot=64, interleaved=False,
             scaling="none", factor=1.0, trained_len=0, first_pos=0, last_pos=99, dtype="bf16", backward=True),
        # long-context training rows with wide heads and shared keys, forward and backward
        dict(name="qknorm_train_65536", op="qk_norm", T=65536, n_head=32, n_kv=8, d=128, rot=128, interleaved=False,
             scaling="ntk", factor=8.0, trained_len=8192, first_pos=0, last_pos=65535, dtype="bf16", backward=True),
        # encoder side of a training step: packed sentences of a ragged batch, window in both directions
        dict(name="window_encoder_ragged", op="window", layout="packed", B=256, min_len=3, max_len=400, lens_seed=5,
             n_head=8, n_kv=8, d=64, window=64, sinks=0, causal=False, dtype="bf16", backward=True),
        # decoder side on long documents, padded batch, forward and backward
        dict(name="window_train_4x8000", op="window", layout="padded", B=4, min_len=5000, max_len=8000, lens_seed=7,
             n_head=8, n_kv=8, d=64, window=1024, sinks=4, causal=True, dtype="bf16", backward=True),
        # reading in one long document before generation: wide heads, shared keys, odd length, forward only
        dict(name="window_prefill_32771", op="window", layout="dense", B=1, min_len=32771, max_len=32771, lens_seed=0,
             n_head=32, n_kv=8, d=128, window=4096, sinks=4, causal=True, dtype="bf16", backward=False),
        # the 32-bit mode that parity runs use
        dict(name="window_train_fp32", op="window", layout="packed", B=16, min_len=100, max_len=1000, lens_seed=3,
             n_head=8, n_kv=8, d=64, window=256, sinks=2, causal=True, dtype="fp32", backward=True),
        # one sentence with five beams: the smallest decoding step
        dict(name="step_beam5", op="step", R=5, n_head=8, n_kv=8, d=64, cap=101, min_len=40, max_len=100, lens_seed=1,
             window=64, sinks=4, dtype="bf16"),
        # two long documents, wide window, cache that holds everything
        dict(name="step_long_2", op="step", R=2, n_head=32, n_kv=4, d=128, cap=40000, min_len=30000, max_len=39999,
             lens_seed=2, window=16384, sinks=4, dtype="bf16"),
        # a large serving batch over ring caches of just sinks + window slots, some sequences shorter than that
        dict(name="step_serving_256", op="step", R=256, n_head=32, n_kv=8, d=128, cap=2052, min_len=700, max_len=9000,
             lens_seed=4, window=2048, sinks=4, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "window", "window", "step", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    d = rng.choice([32, 64, 64, 80, 96, 128])
    n_kv = rng.choice([1, 2, 4, 8])
    n_head = n_kv * rng.choice([1, 1, 2, 4])
    if op in ("rotary", "qk_norm"):
        rot = rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)])
        scaling = rng.choice(["none", "linear", "ntk", "yarn"]) if rot > 2 else "none"
        first = rng.choice([0, 1, _log_int(rng, 1, 1000000)])
        most = 80000000 * (2 if dtype == "bf16" else 1) // ((n_head + n_kv) * d)
        return dict(op=op, T=_log_int(rng, 1, min(65536, most)), n_head=n_head, n_kv=n_kv, d=d, rot=rot,
                    interleaved=rng.random() < 0.5, scaling=scaling, factor=rng.uniform(2.0, 32.0), trained_len=4096,
                    first_pos=first, last_pos=first + _log_int(rng, 1, 65536), dtype=dtype, backward=rng.random() < 0.7)
    if op == "window":
        longest = _log_int(rng, 16, 8192)
        B = rng.randint(1, max(1, min(64, 16384 // longest)))
        layout = rng.choice(["packed", "padded", "dense"])
        return dict(op=op, layout=layout, B=B, min_len=longest if layout == "dense" else rng.randint(1, longest),
                    max_len=longest, lens_seed=rng.randrange(1 << 30), n_head=n_head, n_kv=n_kv, d=d,
                    window=_log_int(rng, 1, 2048), sinks=rng.choice([0, 1, 4, rng.randint(5, 160)]),
                    causal=rng.random() < 0.7, dtype=dtype, backward=rng.random() < 0.6)
    window, sinks = _log_int(rng, 16, 8192), rng.choice([0, 1, 4, rng.randint(5, 64)])
    longest = _log_int(rng, 16, 32768)
    # a ring of the visible slots, or a cache with room for every position
    cap = window + sinks if rng.random() < 0.5 else max(window + sinks, longest + rng.randint(0, 50))
    return dict(op=op, R=rng.randint(1, max(1, min(256, 65536 // cap))), n_head=n_head, n_kv=n_kv, d=d, cap=cap,
                min_len=rng.randint(1, longest), max_len=longest, lens_seed=rng.randrange(1 << 30), window=window,
                sinks=sinks, dtype=dtype)


def _lens(case):
    """The sequences' lengths: the longest one is among them."""
    rng = random.Random(case["lens_seed"])
    n = case["R"] if case["op"] == "step" else case["B"]
    lens = [rng.randint(case["min_len"], case["max_len"]) for _ in range(n)]
    lens[rng.randrange(n)] = case["max_len"]
    return lens


# ------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dt)

    d, H, G = case["d"], case["n_head"], case["n_kv"]
    s = {"case": case}
    if case["op"] in ("rotary", "qk_norm"):
        T = case["T"]
        s["q"], s["k"] = rand(T, H * d, scale=1.5), rand(T, G * d, scale=1.5)
        s["pos"] = torch.randint(case["first_pos"], case["last_pos"] + 1, (T,), generator=gen, device=dev)
        leaves = [s["q"], s["k"]]
        if case["op"] == "qk_norm":
            s["gq"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=dev)
            s["gk"] = 1.0 + 0.2 * torch.randn(d, generator=gen, device=dev)
            leaves += [s["gq"], s["gk"]]
        if case["backward"]:
            s["dq"], s["dk"] = rand(T, H * d), rand(T, G * d)
            for t in leaves:
                t.requires_grad_(True)
        if own:
            from specialk_amd import ops
            s["freqs"] = ops.RotaryFrequencies(case["rot"], base=10000.0, scaling=None if case["scaling"] == "none" else
                                               case["scaling"], factor=case["factor"], trained_len=case["trained_len"],
                                               device=dev)
        return s
    lens = _lens(case)
    if case["op"] == "window":
        B, L = case["B"], case["max_len"]
        packed = case["layout"] == "packed"
        T = sum(lens) if packed else B * L
        s["q"], s["k"], s["v"] = rand(T, H * d), rand(T, G * d), rand(T, G * d)
        s["lens"], s["off"], s["key_pad"] = lens, None, None
        if packed:
            s["off"] = torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)
        elif case["layout"] == "padded":
            n = torch.tensor(lens, device=dev)
            s["key_pad"] = (torch.arange(L, device=dev)[None] >= n[:, None]).to(torch.uint8)
        if case["backward"]:
            s["do"] = rand(T, H * d)
            for t in (s["q"], s["k"], s["v"]):
                t.requires_grad_(True)
        return s
    R, cap = case["R"], case["cap"]
    s["q"], s["k_new"], s["v_new"] = rand(R, H * d), rand(R, G * d), rand(R, G * d)
    s["k_cache"], s["v_cache"] = rand(R, cap, G * d), rand(R, cap, G * d)
    s["kv_len"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["lens"] = lens
    return s


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "qk_norm": _own_qk_norm, "window": _own_window, "step": _own_step}[op](state)
    with torch.no_grad():
        return {"rotary": _plain_rotary, "qk_norm": _plain_rotary, "window": _plain_window, "step": _plain_step}[op](state)


def _own_rotary(s):
    from specialk_amd import ops
    c = s["case"]
    q, k = ops.rotary(s["q"], s["k"], s["pos"], s["freqs"], c["n_head"], c["n_kv"], interleaved=c["interleaved"])
    if not c["backward"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))


def _own_qk_norm(s):
    from specialk_amd import ops
    c = s["case"]
    q, k = ops.qk_norm_rotary(s["q"], s["k"], s["gq"], s["gk"], s["pos"], s["freqs"], c["n_head"], c["n_kv"], eps=1e-6,
                              interleaved=c["interleaved"])
    if not c["backward"]:
        return q, k
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (s["q"], s["k"], s["gq"], s["gk"]), (s["dq"], s["dk"]))


def _own_window(s):
    from specialk_amd import ops
    c = s["case"]
    L = c["max_len"]
    o = ops.window_attention(s["q"], s["k"], s["v"], c["B"], L, L, c["n_head"], c["n_kv"], c["window"], sinks=c["sinks"],
                             causal=c["causal"], key_pad=s["key_pad"], q_off=s["off"], k_off=s["off"])
    if not c["backward"]:
        return o
    return (o.detach(),) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


def _own_step(s):
    from specialk_amd import ops
    c = s["case"]
    o = ops.window_attention_step(s["q"], s["k_new"], s["v_new"], s["k_cache"], s["v_cache"], s["kv_len"], c["n_head"],
                                  c["n_kv"], c["window"], sinks=c["sinks"])
    return o, s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------------ plain forms
def _frequencies(c, dev):
    """(radians per position of each pair in 64 bits, factor on the rotated pair)."""
    rot, base = c["rot"], 10000.0
    if c["scaling"] == "ntk":
        base = base * c["factor"] ** (rot / (rot - 2))
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=dev) / rot)
    amp = 1.0
    if c["scaling"] == "linear":
        f = f / c["factor"]
    elif c["scaling"] == "yarn":
        turns = c["trained_len"] * f / (2 * math.pi)
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f = f / c["factor"] * (1.0 - keep) + f * keep
        amp = 0.1 * math.log(c["factor"]) + 1.0
    return f, amp


def _rotate(x, cos, sin, interleaved):
    """x (T, heads, rot) rotated by the angles whose cosines and sines are (T, 1, rot / 2)."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_rotary(s):
    c = s["case"]
    T, d, rot, norm = c["T"], c["d"], c["rot"], c["op"] == "qk_norm"
    f, amp = _frequencies(c, s["pos"].device)
    angle = s["pos"].to(torch.float64)[:, None] * f[None]
    cos, sin = (torch.cos(angle) * amp).float()[:, None], (torch.sin(angle) * amp).float()[:, None]
    outs, grads, gammas = [], [], []
    for x, dy, g in ((s["q"], s.get("dq"), s.get("gq")), (s["k"], s.get("dk"), s.get("gk"))):
        x32 = x.view(T, -1, d).float()
        y = x32
        if norm:
            rstd = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + 1e-6)
            xhat = x32 * rstd
            y = xhat * g
        outs.append(torch.cat((_rotate(y[..., :rot], cos, sin, c["interleaved"]), y[..., rot:]), -1).view(T, -1).to(x.dtype))
        if not c["backward"]:
            continue
        dy = dy.view(T, -1, d).float()
        dy = torch.cat((_rotate(dy[..., :rot], cos, -sin, c["interleaved"]), dy[..., rot:]), -1)
        if norm:
            gammas.append((dy * xhat).double().sum((0, 1)).float())
            dy = dy * g
            dy = rstd * (dy - xhat * (dy * xhat).mean(-1, keepdim=True))
        grads.append(dy.reshape(T, -1).to(x.dtype))
    return tuple(outs + grads + gammas)


def _visible(p, j, c):
    """(queries, keys) truth values for query positions p and key positions j."""
    p, j = p[:, None], j[None, :]
    return ((p - j < c["window"]) | (j < c["sinks"])) & ((j <= p) if c["causal"] else (j - p < c["window"]))


def _plain_window(s):
    c = s["case"]
    B, L, H, G, d = c["B"], c["max_len"], c["n_head"], c["n_kv"], c["d"]
    q, k, v = s["q"], s["k"], s["v"]
    dev, scale, back = q.device, 1.0 / math.sqrt(d), c["backward"]
    rows = None
    n = torch.tensor(s["lens"], device=dev)
    inside = torch.arange(L, device=dev)[None] < n[:, None]
    if c["layout"] == "packed":
        rows = inside.flatten().nonzero().flatten()

    def heads(x, m):     # (B, m, L, d) in 32 bits
        x = x.float()
        if rows is not None:
            x = torch.zeros((B * L, m * d), device=dev).index_copy_(0, rows, x)
        return x.view(B, L, m, d).transpose(1, 2).contiguous()

    def tokens(x, dt):
        x = x.transpose(1, 2).reshape(B * L, -1)
        return (x if rows is None else x[rows]).to(dt)

    q32, k32, v32 = heads(q, H), heads(k, G), heads(v, G)
    key_ok = inside if c["layout"] != "dense" else torch.ones_like(inside)
    o = torch.empty_like(q32)
    if back:
        do = heads(s["do"], H)
        dq, dk, dv = torch.empty_like(q32), torch.zeros_like(k32), torch.zeros_like(v32)
    step = max(64, min(1024, (1 << 28) // max(1, B * H * min(L, c["window"] + 1024))))
    for i0 in range(0, L, step):
        i1 = min(L, i0 + step)
        lo = max(0, i0 - c["window"] + 1)
        hi = min(L, i1 if c["causal"] else i1 + c["window"] - 1)
        j = torch.arange(lo, hi, device=dev)
        if c["sinks"] and lo > 0:
            j = torch.cat((torch.arange(0, min(c["sinks"], lo), device=dev), j))
        m = _visible(torch.arange(i0, i1, device=dev), j, c)[None] & key_ok[:, None, j]      # (B, queries, keys)
        m = m[:, None, None]
        kj, vj = k32[:, :, j], v32[:, :, j]
        qi = q32[:, :, i0:i1].reshape(B, G, H // G, i1 - i0, d)
        sc = (torch.matmul(qi, kj.transpose(-1, -2).contiguous()[:, :, None]) * scale).masked_fill(~m, float("-inf"))
        top = sc.amax(-1, keepdim=True)
        e = torch.exp(sc - torch.where(top == float("-inf"), torch.zeros_like(top), top))
        total = e.sum(-1, keepdim=True)
        prob = e / torch.where(total == 0, torch.ones_like(total), total)
        o[:, :, i0:i1] = torch.matmul(prob, vj[:, :, None]).reshape(B, H, i1 - i0, d)
        if back:
            doi = do[:, :, i0:i1].reshape(B, G, H // G, i1 - i0, d)
            dp = torch.matmul(doi, vj.transpose(-1, -2).contiguous()[:, :, None])
            ds = prob * (dp - (prob * dp).sum(-1, keepdim=True)) * scale
            dq[:, :, i0:i1] = torch.matmul(ds, kj[:, :, None]).reshape(B, H, i1 - i0, d)
            dk.index_add_(2, j, torch.matmul(ds.transpose(-1, -2).contiguous(), qi).sum(2))
            dv.index_add_(2, j, torch.matmul(prob.transpose(-1, -2).contiguous(), doi).sum(2))
    if not back:
        return tokens(o, q.dtype)
    return tokens(o, q.dtype), tokens(dq, q.dtype), tokens(dk, q.dtype), tokens(dv, q.dtype)


def _plain_step(s):
    c = s["case"]
    R, H, G, d, cap, sinks = c["R"], c["n_head"], c["n_kv"], c["d"], c["cap"], c["sinks"]
    n = s["kv_len"].long()
    dev = n.device
    row = torch.arange(R, device=dev)
    last = n - 1
    slot = torch.where(last < sinks, last, sinks + (last - sinks) % (cap - sinks))
    s["k_cache"][row, slot] = s["k_new"]
    s["v_cache"][row, slot] = s["v_new"]
    # position that each slot holds: the newest one that falls on it
    e = torch.arange(cap, device=dev)[None]
    j = torch.where(e < sinks, e, last[:, None] - (last[:, None] - e) % (cap - sinks))
    ok = (j <= last[:, None]) & ((j < sinks) | ((j >= sinks) & (last[:, None] - j < c["window"])))
    ok &= (e < sinks) | (j >= sinks)
    outs = []
    per = max(1, (1 << 28) // (cap * G * d))
    for r0 in range(0, R, per):
        r1 = min(R, r0 + per)
        k = s["k_cache"][r0:r1].float().view(r1 - r0, cap, G, d).transpose(1, 2).contiguous()
        v = s["v_cache"][r0:r1].float().view(r1 - r0, cap, G, d).transpose(1, 2).contiguous()
        q = s["q"][r0:r1].float().view(r1 - r0, G, H // G, d)
        sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(d)
        sc = sc.masked_fill(~ok[r0:r1, None, None], float("-inf"))
        ex = torch.exp(sc - sc.amax(-1, keepdim=True))
        outs.append((torch.matmul(ex, v) / ex.sum(-1, keepdim=True)).reshape(r1 - r0, H * d))
    return torch.cat(outs).to(s["q"].dtype), s["k_cache"], s["v_cache"]


# ------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "qk_norm": _exact_rotary, "window": _exact_window, "step": _exact_step}[case["op"]](s)


def _exact_rotary(s):
    """Pairs as complex numbers turned by exp(i angle); the gradients from the tape."""
    c = s["case"]
    T, d, rot = c["T"], c["d"], c["rot"]
    pos = s["pos"].double().cpu()
    half = rot // 2
    angle = torch.empty((T, half), dtype=torch.float64)
    amp = 1.0 + 0.1 * math.log(c["factor"]) if c["scaling"] == "yarn" else 1.0
    for i in range(half):
        f = 10000.0 ** (-2.0 * i / rot)
        if c["scaling"] == "ntk":
            f = (10000.0 * c["factor"] ** (rot / (rot - 2.0))) ** (-2.0 * i / rot)
        elif c["scaling"] == "linear":
            f = f / c["factor"]
        elif c["scaling"] == "yarn":
            r = c["trained_len"] * f / (2.0 * math.pi)
            g = min(1.0, max(0.0, (r - 1.0) / 31.0))
            f = (1.0 - g) * f / c["factor"] + g * f
        angle[:, i] = pos * f
    turn = torch.polar(torch.full_like(angle, amp), angle).to(s["q"].device)[:, None]
    outs, leaves = [], []
    for x, g in ((s["q"], s.get("gq")), (s["k"], s.get("gk"))):
        x = x.detach().double().requires_grad_(c["backward"])
        y = x.view(T, -1, d)
        if g is not None:
            g = g.detach().double().requires_grad_(c["backward"])
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * g
        head, tail = y.split((rot, d - rot), -1)
        if c["interleaved"]:
            z = torch.view_as_complex(head.reshape(T, -1, half, 2).contiguous()) * turn
            head = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()) * turn
            head = torch.cat((z.real, z.imag), -1)
        outs.append(torch.cat((head, tail), -1).reshape(T, -1))
        leaves.append((x, g))
    if not c["backward"]:
        return tuple(outs)
    wrt = [x for x, _ in leaves] + [g for _, g in leaves if g is not None]
    grads = torch.autograd.grad(outs, wrt, (s["dq"].double(), s["dk"].double()))
    return tuple(o.detach() for o in outs) + grads


def _exact_window(s):
    """Sequence by sequence, a block of queries against every key, gradients from the tape."""
    c = s["case"]
    B, L, H, G, d = c["B"], c["max_len"], c["n_head"], c["n_kv"], c["d"]
    out = [torch.zeros_like(s["q"], dtype=torch.float64, requires_grad=False)]
    if c["backward"]:
        out += [torch.zeros_like(s[x], dtype=torch.float64, requires_grad=False) for x in ("q", "k", "v")]
    dev, first = s["q"].device, 0
    for b in range(B):
        n = s["lens"][b] if c["layout"] == "packed" else L
        alive = s["lens"][b] if c["layout"] == "padded" else n
        sl = slice(first, first + n)
        first += n
        q, k, v = (s[x].detach()[sl].double().view(n, -1, d).permute(1, 0, 2).contiguous().requires_grad_(c["backward"])
                   for x in ("q", "k", "v"))
        size = max(1, min(n, (1 << 28) // (H * n)))
        key = torch.arange(n, device=dev)
        for a in range(0, n, size):
            z = min(n, a + size)
            query = torch.arange(a, z, device=dev)
            dist = query.view(-1, 1) - key.view(1, -1)
            see = dist.abs() < c["window"]
            see |= (key < c["sinks"]).view(1, -1) & (dist > -c["window"])
            if c["causal"]:
                see &= dist >= 0
            see &= (key < alive).view(1, -1)
            some = see.any(1).view(1, -1, 1)
            lg = torch.matmul(q[:, a:z], k.repeat_interleave(H // G, 0).transpose(1, 2).contiguous()) * d ** -0.5
            lg = torch.where(see[None] | ~some, lg, torch.full_like(lg, -math.inf))
            o = torch.matmul(torch.softmax(lg, -1) * some, v.repeat_interleave(H // G, 0))
            rows = slice(sl.start + a, sl.start + z)
            out[0][rows] = o.detach().permute(1, 0, 2).reshape(z - a, H * d)
            if c["backward"]:
                do = s["do"][rows].double().view(z - a, H, d).permute(1, 0, 2)
                for t, g in zip(out[1:], torch.autograd.grad(o, (q, k, v), do)):
                    t[sl] += g.permute(1, 0, 2).reshape(n, -1)
    return out[0] if len(out) == 1 else tuple(out)


def _exact_step(s):
    """Row by row over the list of visible positions."""
    c = s["case"]
    H, G, d, sinks, ring = c["n_head"], c["n_kv"], c["d"], c["sinks"], c["cap"] - c["sinks"]
    kc, vc = s["k_cache"].clone(), s["v_cache"].clone()
    out = []
    for r, n in enumerate(s["lens"]):
        slots = [j if j < sinks else sinks + (j - sinks) % ring
                 for j in list(range(min(sinks, n))) + list(range(max(sinks, n - c["window"]), n))]
        kc[r, slots[-1]], vc[r, slots[-1]] = s["k_new"][r], s["v_new"][r]
        at = torch.tensor(slots, device=kc.device)
        k, v = kc[r, at].double().view(-1, G, d), vc[r, at].double().view(-1, G, d)
        q = s["q"][r].double().view(G, H // G, d)
        w = torch.stack([torch.softmax(torch.mv(k[:, h // (H // G)].contiguous(), q.view(H, d)[h]) / d ** 0.5, 0)
                         for h in range(H)])
        o = [torch.mv(v[:, h // (H // G)].t().contiguous(), w[h]) for h in range(H)]
        out.append(torch.cat(o))
    return torch.stack(out), kc.double(), vc.double()


# ------------------------------------------------------------------------------------------------------ work
def _pairs(n, alive, c):
    """Visible (query, key) pairs of a sequence of n queries and keys, the first `alive` keys of which are no padding."""
    p = torch.arange(n, dtype=torch.int64)
    hi = torch.clamp(p + 1 if c["causal"] else p + c["window"], max=alive)
    lo = torch.clamp(p - c["window"] + 1, min=0)
    near = torch.clamp(hi - lo, min=0)
    far = torch.minimum(torch.clamp(lo, max=c["sinks"]), hi.clamp(min=0)).clamp(min=0)
    return int((near + far).sum())


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    H, G, d = case["n_head"], case["n_kv"], case["d"]
    if case["op"] in ("rotary", "qk_norm"):
        T, rot, norm = case["T"], case["rot"], case["op"] == "qk_norm"
        n = T * (H + G) * d
        per = 3 * rot + (4 * d if norm else 0)          # a head forward: a pair costs 6, the norm 4 an element
        if not case["backward"]:
            return {"bytes": 2 * n * size + 8 * T, "flops": T * (H + G) * per}
        back = 3 * rot + (10 * d if norm else 0)
        # forward: x -> y; backward: dy (and x, for the norm's) -> dx
        moved = 2 * n + 2 * n
        return {"bytes": moved * size + 8 * T, "flops": T * (H + G) * (per + back)}
    lens = _lens(case)
    if case["op"] == "window":
        L, B = case["max_len"], case["B"]
        if case["layout"] == "packed":
            T, pairs = sum(lens), sum(_pairs(n, n, case) for n in lens)
        else:
            T = B * L
            pairs = sum(_pairs(L, n if case["layout"] == "padded" else L, case) for n in lens)
        q, kv = T * H * d, T * G * d
        if not case["backward"]:
            return {"bytes": (2 * q + 2 * kv) * size, "flops": 4 * d * H * pairs}
        # forward q, k, v -> o; backward those and do -> dq, dk, dv: 2 + 5 products over the visible pairs
        return {"bytes": (2 * q + 2 * kv + 2 * q + 2 * kv) * size, "flops": (4 + 10) * d * H * pairs}
    seen = sum(min(n, case["window"]) + min(case["sinks"], max(0, n - case["window"])) for n in lens)
    R = case["R"]
    # the visible keys and values but the new ones, which come from their own rows and go into the cache
    return {"bytes": (2 * seen * G * d + 2 * R * G * d + 2 * R * H * d) * size, "flops": 4 * d * H * seen}
