"""Measured cases of the block operators (video_diffusion_amd/block_hip.py): attention over time with a decay per head
(whole sequences and single tokens), the norms before and after a block with its gate and residual scale, activation
checkpoints in 8 bits.

`run` computes a case in plain torch operations, or, with `own` set, through the library's calls on the same inputs.
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the temporal layer of the finest level in training: 16 frames at 64 x 64 sites, 8 heads of 32 features
        {"name": "decay frames train", "op": "decay", "b": 4, "s": 4096, "n": 16, "h": 8, "d": 32, "dt": "bf16", "train": True,
         "state": False, "ragged": False},
        # a long clip flattened to one token axis, in training
        {"name": "decay long train", "op": "decay", "b": 2, "s": 1, "n": 8192, "h": 8, "d": 64, "dt": "bf16", "train": True,
         "state": False, "ragged": False},
        # one long prompt: the outputs and the state that single tokens go on from
        {"name": "decay prompt", "op": "decay", "b": 1, "s": 1, "n": 16384, "h": 8, "d": 128, "dt": "f16", "train": False,
         "state": True, "ragged": False},
        # truncated training through time: a padded batch that starts from given states and hands its states on
        {"name": "decay ragged train", "op": "decay", "b": 6, "s": 1, "n": 701, "h": 4, "d": 64, "dt": "bf16", "train": True,
         "state": True, "ragged": True},
        # a small latent clip at sampling time: 10 frames at 4 x 4 sites
        {"name": "decay small", "op": "decay", "b": 1, "s": 16, "n": 10, "h": 8, "d": 32, "dt": "bf16", "train": False,
         "state": False, "ragged": False},
        # one more token of one stream
        {"name": "step single", "op": "step", "b": 1, "h": 8, "d": 64, "dt": "bf16"},
        # one more frame at every site of two 64 x 64 streams
        {"name": "step frame", "op": "step", "b": 8192, "h": 8, "d": 32, "dt": "f16"},
        # between two blocks of the coarsest level, one clip of 10 frames at 4 x 4
        {"name": "norm small", "op": "norm", "b": 1, "r": 160, "c": 512, "dt": "bf16", "kind": "rms", "train": False,
         "alpha": 1.0},
        # between two blocks in training, 16 frames at 64 x 64 of 4 clips
        {"name": "norm train", "op": "norm", "b": 4, "r": 65536, "c": 256, "dt": "bf16", "kind": "layer", "train": True,
         "alpha": 1.0},
        # wide float32 rows of an odd count in training, with a scaled residual
        {"name": "norm wide f32", "op": "norm", "b": 3, "r": 1237, "c": 2048, "dt": "f32", "kind": "rms", "train": True,
         "alpha": 0.70710678},
        # activations put away in 8 bits and taken out again
        {"name": "rows8 keep", "op": "keep", "r": 262144, "c": 256, "dt": "bf16"},
        # a projection to q, k and v: its input kept in 8 bits, its weight gradient from there
        {"name": "rows8 linear", "op": "linear", "r": 131072, "c": 512, "o": 1536, "dt": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["op"], [0.0, 0.0])
        m[0], m[1] = max(m[0], w["bytes"]), max(m[1], w["flops"])
    while True:
        op = rng.choice(["decay", "decay", "step", "norm", "norm", "keep", "linear"])
        if op == "decay":
            c = {"op": op, "b": _log(rng, 1, 16), "s": rng.choice([1, _log(rng, 1, 4096)]), "n": _log(rng, 1, 16384),
                 "h": rng.randint(1, 12), "d": rng.choice([32, 64, 128]), "dt": rng.choice(["bf16", "f16"]),
                 "train": rng.random() < 0.6, "state": rng.random() < 0.5, "ragged": rng.random() < 0.4}
        elif op == "step":
            c = {"op": op, "b": _log(rng, 1, 8192), "h": rng.randint(1, 12), "d": rng.choice([32, 64, 128]),
                 "dt": rng.choice(["bf16", "f16"])}
        elif op == "norm":
            c = {"op": op, "b": rng.randint(1, 8), "r": _log(rng, 1, 65536), "c": _log(rng, 8, 4096),
                 "dt": rng.choice(["bf16", "f16", "f32"]), "kind": rng.choice(["rms", "layer"]),
                 "train": rng.random() < 0.6, "alpha": rng.choice([1.0, 0.70710678])}
        elif op == "keep":
            c = {"op": op, "r": _log(rng, 1, 262144), "c": 8 * _log(rng, 1, 256), "dt": rng.choice(["bf16", "f16", "f32"])}
        else:
            c = {"op": op, "r": _log(rng, 16, 131072), "c": 8 * _log(rng, 2, 160), "o": 8 * _log(rng, 2, 200),
                 "dt": rng.choice(["bf16", "f32"])}
        w = work(c)
        if w["bytes"] <= most[op][0] and w["flops"] <= most[op][1]:
            return c


def work(case):
    op = case["op"]
    if op == "decay":
        seqs, e = case["b"] * case["s"], _BYTES[case["dt"]]
        rows = seqs * case["n"] * case["h"]
        d, state = case["d"], 4 * seqs * case["h"] * case["d"] ** 2
        # per token and head: the scan's outer product and product with the state, or the pairs where the sequence is short
        fl = rows * d * 4 * min(d, (case["n"] + 1) / 2)
        if not case["train"]:
            return {"bytes": 4 * rows * d * e + (2 * state if case["state"] else 0), "flops": fl}
        # forward q k v -> o; backward q k v do -> dq dk dv; the states and their gradients in and out
        return {"bytes": 11 * rows * d * e + (4 * state if case["state"] else 0), "flops": 3.5 * fl}
    if op == "step":
        rows = case["b"] * case["h"]
        return {"bytes": rows * (8 * case["d"] ** 2 + 4 * case["d"] * _BYTES[case["dt"]]), "flops": 5 * rows * case["d"] ** 2}
    if op == "norm":
        n = case["b"] * case["r"] * case["c"]
        return {"bytes": n * _BYTES[case["dt"]] * (10 if case["train"] else 4), "flops": n * (50 if case["train"] else 20)}
    n, e = case["r"] * case["c"], _BYTES[case["dt"]]
    kept = case["r"] * (case["c"] + -(-case["c"] // 32))
    if op == "keep":
        return {"bytes": 2 * n * e + 2 * kept, "flops": 6 * n}
    return {"bytes": n * e + 2 * kept + 2 * case["r"] * case["o"] + 4 * case["c"] * case["o"],
            "flops": 2 * n * case["o"]}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, dt = case["op"], _DT[case["dt"]]

    def rand(*shape, dtype=dt, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).to(dtype)

    st = {"case": case}
    if op in ("decay", "step"):
        h, d = case["h"], case["d"]
        # memories from 8 to 512 tokens, one length per head
        st["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(3, 9, h, device=DEV)))
    if op == "decay":
        b, s, n = case["b"], case["s"], case["n"]
        # the rows of a qkv projection: (sample, time, site) rows, so a site's tokens lie s rows apart
        qkv = rand(b, n, s, 3, h, d)
        st["q"], st["k"], st["v"] = (t.permute(0, 2, 1, 3, 4) for t in qkv.unbind(3))
        st["state"] = rand(b, s, h, d, d, dtype=torch.float32) if case["state"] else None
        st["lengths"] = None
        if case["ragged"]:
            ln = torch.randint(0, n + 1, (b, s), generator=g, device=DEV, dtype=torch.int32)
            ln.view(-1)[0] = n
            st["lengths"] = ln
        if case["train"]:
            st["do"] = rand(b, n, s, h, d).permute(0, 2, 1, 3, 4)
            st["dstate"] = rand(b, s, h, d, d, dtype=torch.float32) if case["state"] else None
    elif op == "step":
        b = case["b"]
        qkv = rand(b, 3, h, d)
        st["q"], st["k"], st["v"] = qkv.unbind(1)
        st["state"] = rand(b, h, d, d, dtype=torch.float32)
    elif op == "norm":
        b, r, c = case["b"], case["r"], case["c"]
        st["x"], st["h"] = rand(b, r, c, std=1.5), rand(b, r, c, std=0.7)
        f32 = torch.float32
        st["post_weight"], st["weight"] = 1 + rand(c, dtype=f32, std=0.2), 1 + rand(c, dtype=f32, std=0.2)
        # per sample, from the embedding of its time step
        st["gate"], st["scale"], st["shift"] = (rand(b, c, dtype=f32, std=0.5) for _ in range(3))
        if case["train"]:
            st["dout"], st["dy"] = rand(b, r, c), rand(b, r, c)
    else:
        r, c = case["r"], case["c"]
        # activations: channels of different spreads
        st["x"] = (rand(r, c, dtype=torch.float32) * torch.exp(rand(c, dtype=torch.float32))).to(dt)
        if op == "linear":
            st["dy"] = rand(r, case["o"], dtype=torch.bfloat16, std=0.1)
    return st


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    from video_diffusion_amd import block_hip as B
    case = st["case"]
    op = case["op"]
    if op == "decay":
        kw = dict(lengths=st["lengths"], return_state=case["state"])
        if not case["train"]:
            with torch.no_grad():
                return B.decay_attention(st["q"], st["k"], st["v"], st["log_decay"], initial_state=st["state"], **kw)
        ins = [t.detach().requires_grad_() for t in (st["q"], st["k"], st["v"])]
        if case["state"]:
            s0 = st["state"].detach().requires_grad_()
            o, s = B.decay_attention(*ins, st["log_decay"], initial_state=s0, **kw)
            return (o.detach(), s.detach(), *torch.autograd.grad((o, s), (*ins, s0), (st["do"], st["dstate"])))
        o = B.decay_attention(*ins, st["log_decay"], **kw)
        return (o.detach(), *torch.autograd.grad(o, ins, st["do"]))
    if op == "step":
        return B.decay_attention_step(st["q"], st["k"], st["v"], st["log_decay"], st["state"]), st["state"]
    if op == "norm":
        kw = dict(alpha=case["alpha"], kind=case["kind"], post_kind=case["kind"])
        names = ("x", "h", "post_weight", "gate", "weight", "scale", "shift")
        if not case["train"]:
            with torch.no_grad():
                return B.norm_between(*(st[k] for k in names), **kw)
        ins = [st[k].detach().requires_grad_() for k in names]
        out, y = B.norm_between(*ins, **kw)
        return (out.detach(), y.detach(), *torch.autograd.grad((out, y), ins, (st["dout"], st["dy"])))
    kept = B.pack_rows8(st["x"])
    if op == "keep":
        return kept.unpack()
    return B.rows8_wgrad(kept, st["dy"])


def _run_plain(st):
    case = st["case"]
    op = case["op"]
    if op == "decay":
        if not case["train"]:
            with torch.no_grad():
                o, s = _decay(st["q"], st["k"], st["v"], st["log_decay"], st["state"], st["lengths"])
            return (o, s) if case["state"] else o
        ins = [t.detach().requires_grad_() for t in (st["q"], st["k"], st["v"])]
        if case["state"]:
            s0 = st["state"].detach().requires_grad_()
            o, s = _decay(*ins, st["log_decay"], s0, st["lengths"])
            return (o.detach(), s.detach(), *torch.autograd.grad((o, s), (*ins, s0), (st["do"], st["dstate"])))
        o, _ = _decay(*ins, st["log_decay"], None, st["lengths"])
        return (o.detach(), *torch.autograd.grad(o, ins, st["do"]))
    if op == "step":
        q, k, v = (st[x].float() for x in ("q", "k", "v"))
        s = st["state"]
        s.mul_(st["log_decay"].exp().view(1, -1, 1, 1)).add_(k[..., :, None] * v[..., None, :])
        o = (q[..., None, :] @ s)[..., 0, :] * q.shape[-1] ** -0.5
        return o.to(st["q"].dtype), s
    if op == "norm":
        return _norm(st, case)
    kept = _rows8(st["x"])
    if op == "keep":
        return kept.to(st["x"].dtype)
    return st["dy"].float().t() @ kept


def _decay(q, k, v, log_decay, s0, lengths):
    """o_t = scale * q_t S_t with S_t = exp(log_decay) S_(t-1) + k_t v_t^T, in chunks: pairs inside a chunk as a masked
    product, what came before it through the state at the chunk's start."""
    b, s, n, h, d = q.shape
    c = min(n, 128)
    nc = -(-n // c)

    def rows(t):          # [b*s, h, chunks, c, d]
        t = t.float().permute(0, 1, 3, 2, 4).reshape(b * s, h, n, d)
        return torch.nn.functional.pad(t, (0, 0, 0, nc * c - n)).view(b * s, h, nc, c, d)

    qf, kf, vf = rows(q), rows(k), rows(v)
    g = log_decay.view(1, h, 1, 1)
    at = torch.arange(nc * c, device=q.device)
    length = torch.full((b * s,), n, device=q.device) if lengths is None else lengths.reshape(-1).long()
    live = (at[None, :] < length[:, None]).view(b * s, 1, nc, c, 1)
    kf = kf * live
    i = torch.arange(c, device=q.device, dtype=torch.float32)
    gap = i[:, None] - i[None, :]
    decay = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), 0.0).view(1, h, 1, c, c)
    o = ((qf @ kf.transpose(-1, -2)) * decay) @ vf
    if nc > 1 or s0 is not None:
        u = (kf * torch.exp(g * (c - 1 - i)).view(1, h, 1, c, 1)).transpose(-1, -2) @ vf       # what a chunk adds
        j = torch.arange(nc, device=q.device, dtype=torch.float32)
        ago = j[:, None] - 1 - j[None, :]
        w = torch.where(ago >= 0, torch.exp(g * c * ago.clamp(min=0)), 0.0).view(1, h, nc, nc)
        start = (w @ u.reshape(b * s, h, nc, d * d)).view(b * s, h, nc, d, d)
        if s0 is not None:
            start = start + torch.exp(g * c * j).view(1, h, nc, 1, 1) * s0.reshape(b * s, h, 1, d, d)
        o = o + torch.exp(g * (i + 1)).view(1, h, 1, c, 1) * (qf @ start)
    o = (o * live).view(b * s, h, nc * c, d)[:, :, :n] * d ** -0.5
    o = o.view(b, s, h, n, d).permute(0, 1, 3, 2, 4).to(q.dtype)
    last = None
    if s0 is not None:
        left = (length[:, None] - 1 - at[None, :]).clamp(min=0).view(b * s, 1, nc * c)
        w = torch.exp(log_decay.view(1, h, 1) * left).unsqueeze(-1)
        last = (kf.view(b * s, h, nc * c, d) * w).transpose(-1, -2) @ vf.view(b * s, h, nc * c, d)
        last = last + torch.exp(log_decay.view(1, h) * length.view(-1, 1)).view(b * s, h, 1, 1) * s0.view(b * s, h, d, d)
        last = last.view(b, s, h, d, d)
    return o, last


EPS = 1e-5


def _unit(x, kind):
    """x centred (layer) and divided by its root mean square, and that division's factor."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    f = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    return x * f, f


def _unit_grad(dn, n, f, kind):
    g = dn - n * (dn * n).mean(-1, keepdim=True)
    return f * (g - dn.mean(-1, keepdim=True) if kind == "layer" else g)


def _norm(st, case):
    """out = alpha x + gate * norm(h) * post_weight; y = norm(out) * weight * (1 + scale) + shift; in training the gradients
    of all seven inputs."""
    kind, alpha, dt = case["kind"], case["alpha"], st["x"].dtype
    gate, scale, shift = (st[k][:, None] for k in ("gate", "scale", "shift"))
    pw, w = st["post_weight"], st["weight"]
    hn, hf = _unit(st["h"].float(), kind)
    out = alpha * st["x"].float() + gate * (hn * pw)
    on, of = _unit(out, kind)
    out, y = out.to(dt), (on * w * (1 + scale) + shift).to(dt)
    if not case["train"]:
        return out, y
    dy = st["dy"].float()
    dx = st["dout"].float() + _unit_grad(dy * (w * (1 + scale)), on, of, kind)
    dh = _unit_grad(dx * (gate * pw), hn, hf, kind)
    by_y, by_h = (dy * on).sum(1), (dx * hn).sum(1)
    return (out, y, (alpha * dx).to(dt), dh.to(dt), (by_h * st["gate"]).sum(0), by_h * pw, (by_y * (1 + st["scale"])).sum(0),
            by_y * w, dy.sum(1))


def _rows8(x):
    """x as 8-bit values (4 exponent, 3 fraction bits, at most 448) times a power of two per 32 channels: the smallest one
    that holds the group's largest magnitude."""
    r, c = x.shape
    t = torch.nn.functional.pad(x.float(), (0, -c % 32)).view(r, -1, 32)
    m, e = torch.frexp(t.abs().amax(-1, keepdim=True))
    e = (e - 9 + (m > 0.875).int()).clamp(-118, 119)
    t = torch.ldexp(t, -e).to(torch.float8_e4m3fn).float()
    return torch.ldexp(t, e).view(r, -1)[:, :c]


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"decay": _exact_decay, "step": _exact_step, "norm": _exact_norm, "keep": _exact_rows8, "linear": _exact_rows8}[
        case["op"]](st, case)


def _exact_decay(st, case):
    b, s, n, h, d = st["q"].shape

    def rows(t):
        return t.double().permute(0, 1, 3, 2, 4).reshape(b * s, h, n, d)

    def back(t):
        return t.view(b, s, h, n, d).permute(0, 1, 3, 2, 4)

    q, k, v = rows(st["q"]), rows(st["k"]), rows(st["v"])
    g = st["log_decay"].double()
    length = (torch.full((b * s,), n, device=DEV) if st["lengths"] is None else st["lengths"].reshape(-1)).double()
    c = min(n, 96)
    m = d ** -0.5
    zero = torch.zeros(b * s, h, d, d, device=DEV, dtype=torch.float64)
    cur = zero if st["state"] is None else st["state"].double().view(b * s, h, d, d)
    starts, out = [], torch.zeros_like(q)

    def piece(t0):
        t = torch.arange(t0, min(n, t0 + c), device=DEV, dtype=torch.float64)
        on = (t[None] < length[:, None]).double()[:, None, :, None]              # live tokens of the piece
        left = (torch.minimum(t[-1] + 1, length)[:, None] - 1 - t[None]).clamp(min=0)       # live tokens after each
        span = (length - t0).clamp(0, t.numel())
        gap = t[:, None] - t[None, :]
        pair = torch.exp(g.view(h, 1, 1) * gap.clamp(min=0)) * (gap >= 0)
        into = torch.exp(g.view(h, 1) * (t - t0 + 1)).view(1, h, -1, 1)
        keep = torch.exp(g.view(1, h, 1) * left[:, None]).unsqueeze(-1) * on
        return slice(t0, min(n, t0 + c)), on, pair, into, keep, torch.exp(g.view(1, h) * span[:, None])[..., None, None]

    for t0 in range(0, n, c):
        at, on, pair, into, keep, whole = piece(t0)
        starts.append(cur)
        out[:, :, at] = m * on * (((q[:, :, at] @ k[:, :, at].mT) * pair) @ v[:, :, at] + into * (q[:, :, at] @ cur))
        cur = whole * cur + (keep * k[:, :, at]).mT @ v[:, :, at]
    got = [back(out)] + ([cur.view(b, s, h, d, d)] if case["state"] else [])
    if not case["train"]:
        return tuple(got) if case["state"] else got[0]
    do = rows(st["do"])
    ds = zero if st["dstate"] is None else st["dstate"].double().view(b * s, h, d, d)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    for t0 in reversed(range(0, n, c)):
        at, on, pair, into, keep, whole = piece(t0)
        e, qa, ka, va = m * on * do[:, :, at], q[:, :, at], k[:, :, at], v[:, :, at]
        a, p = (e @ va.mT) * pair, (qa @ ka.mT) * pair
        dq[:, :, at] = a @ ka + into * (e @ starts[-1].mT)
        dk[:, :, at] = a.mT @ qa + keep * (va @ ds.mT)
        dv[:, :, at] = p.mT @ e + keep * (ka @ ds)
        ds = whole * ds + (into * qa).mT @ e
        starts.pop()
    got += [back(dq), back(dk), back(dv)]
    return tuple(got + ([ds.view(b, s, h, d, d)] if case["state"] else []))


def _exact_step(st, case):
    q, k, v = (st[x].double() for x in ("q", "k", "v"))
    s = torch.exp(st["log_decay"].double())[None, :, None, None] * st["state"].double() + torch.einsum("bhi,bhj->bhij", k, v)
    return torch.einsum("bhi,bhij->bhj", q, s) / math.sqrt(case["d"]), s


def _exact_norm(st, case):
    c, layer = case["c"], case["kind"] == "layer"
    D = {k: t.double() for k, t in st.items() if torch.is_tensor(t)}

    def stats(t):
        mean = t.sum(-1, keepdim=True) / c if layer else torch.zeros_like(t[..., :1])
        return mean, ((t - mean).pow(2).sum(-1, keepdim=True) / c + EPS).pow(-0.5)

    def norm_back(dn, t, mean, f):
        n = (t - mean) * f
        r = dn - n * ((dn * n).sum(-1, keepdim=True) / c)
        return f * (r - dn.sum(-1, keepdim=True) / c) if layer else f * r

    up = {k: D[k].unsqueeze(1) for k in ("gate", "scale", "shift")}
    hm, hf = stats(D["h"])
    hn = (D["h"] - hm) * hf
    out = D["x"] * case["alpha"] + up["gate"] * D["post_weight"] * hn
    om, of = stats(out)
    on = (out - om) * of
    y = on * D["weight"] * (1 + up["scale"]) + up["shift"]
    if not case["train"]:
        return out, y
    total = D["dout"] + norm_back(D["dy"] * D["weight"] * (1 + up["scale"]), out, om, of)
    return (out, y, total * case["alpha"], norm_back(total * up["gate"] * D["post_weight"], D["h"], hm, hf),
            (total * up["gate"] * hn).sum((0, 1)), (total * D["post_weight"] * hn).sum(1),
            (D["dy"] * on * (1 + up["scale"])).sum((0, 1)), (D["dy"] * on * D["weight"]).sum(1), D["dy"].sum(1))


def _exact_rows8(st, case):
    x = st["x"].double()
    r, c = x.shape
    groups = -(-c // 32)
    t = torch.zeros(r, groups * 32, device=DEV, dtype=torch.float64)
    t[:, :c] = x
    t = t.view(r, groups, 32)
    top = t.abs().max(-1, keepdim=True).values
    # the least power of two u with top <= 448 u
    u = torch.exp2(torch.ceil(torch.log2((top / 448).clamp(min=2.0 ** -118))))
    u = torch.where(top <= 448 * u / 2, u / 2, torch.where(top > 448 * u, 2 * u, u)).clamp(min=2.0 ** -118)
    a = t / u
    # steps of an eighth of the power of two below, at least 2^-9; ties to the even step
    step = torch.exp2(torch.floor(torch.log2(a.abs().clamp(min=2.0 ** -6))) - 3)
    kept = (torch.round(a / step) * step * u).view(r, -1)[:, :c]
    if case["op"] == "keep":
        return kept
    return st["dy"].double().mT @ kept
