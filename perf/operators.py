"""Cases and plain forms of the conditioned-block operators: cross attention to an encoder's
states, rotary positions on several axes, and the norms around a block with its gate and
residual scale.  `run` computes them in elementary torch operations, or, with `own` true, by
the calls that a user makes of mdgen_finetune_amd.cross_hip."""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one new token of one trajectory reads a short encoder (latency)
        dict(name="attn_token_short", op="attn", train=False, dtype="bf16", B=1, Nq=1, Nk=256, H=16, Hk=16, D=24,
             pad="none", store="tokens"),
        # single tokens of a batch of long contexts with shared k/v heads, cached head by head, ragged lengths
        dict(name="attn_token_long", op="attn", train=False, dtype="bf16", B=16, Nq=1, Nk=16384, H=32, Hk=8, D=128,
             pad="len", store="heads"),
        # the denoiser's tokens (T = 1000 frames x L = 4 residues, B = 8) on a padded residue encoder of crop 256
        dict(name="attn_frames", op="attn", train=False, dtype="bf16", B=8, Nq=4000, Nk=256, H=16, Hk=16, D=24,
             pad="mask", store="packed"),
        # a long prompt on a long encoder, wide heads: the matrix cores' case
        dict(name="attn_prompt", op="attn", train=False, dtype="bf16", B=2, Nq=4096, Nk=8192, H=16, Hk=4, D=128,
             pad="none", store="tokens"),
        # fp32 training at odd lengths, head_dim 48 (embed 384, 8 heads), rows masked
        dict(name="attn_train_f32", op="attn", train=True, dtype="f32", B=2, Nq=1001, Nk=333, H=8, Hk=8, D=48,
             pad="mask", store="tokens"),
        # bf16 training, shared k/v heads, ragged encoder lengths
        dict(name="attn_train", op="attn", train=True, dtype="bf16", B=4, Nq=4096, Nk=2048, H=16, Hk=4, D=64,
             pad="len", store="packed"),
        # the next token of four sequences: q and k of one position each
        dict(name="rope_token", op="rope", train=False, dtype="bf16", B=4, N=1, H=32, Hk=8, D=128, rot=128, axes=3,
             pairs="half", store="tokens", far=True),
        # the training batch B = 8 x T = 1000 x L = 4 on (frame, residue) axes, forward and backward
        dict(name="rope_frames_train", op="rope", train=True, dtype="bf16", B=8, N=4000, H=16, Hk=16, D=24, rot=24,
             axes=2, pairs="axis", store="packed", far=False),
        # a video-like grid of long clips, time / height / width, part of the head left unrotated, odd length
        dict(name="rope_grid_f32", op="rope", train=False, dtype="f32", B=2, N=50001, H=12, Hk=4, D=64, rot=48, axes=3,
             pairs="interleaved", store="tokens", far=True),
        # a token's row through the norms (latency)
        dict(name="norm_token", op="norm", train=False, dtype="bf16", res="f32", G=4, rows=1, C=384, post="rms",
             pre="layer", affine=False),
        # the training batch: fp32 residual, bf16 branch, adaLN rows per trajectory
        dict(name="norm_frames_train", op="norm", train=True, dtype="bf16", res="f32", G=8, rows=4000, C=384,
             post="rms", pre="layer", affine=True),
        # wide rows, everything in bf16, an odd number of rows
        dict(name="norm_wide", op="norm", train=False, dtype="bf16", res="bf16", G=3, rows=5461, C=4096, post="layer",
             pre="rms", affine=True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "rope", "norm"])
    if op == "attn":
        train = rng.random() < 0.5
        dtype = rng.choice(["bf16", "bf16", "f32"])
        Hk = rng.choice([1, 2, 4, 8, 16])
        G = rng.choice([1, 1, 2, 4, 8]) if Hk <= 8 else 1
        c = dict(op="attn", train=train, dtype=dtype, B=rng.randint(1, 8),
                 Nq=rng.choice([1, _logint(rng, 1, 40), _logint(rng, 33, 4096)]),
                 # (the gradients of q and k over one state are zero: a training encoder has some of them)
                 Nk=_logint(rng, 24 if train else 1, 8192), H=G * Hk,
                 Hk=Hk, D=rng.choice([16, 20, 24, 32, 40, 48, 64, 72, 80, 96, 128]),
                 pad=rng.choice(["none", "len", "mask"]), store=rng.choice(["tokens", "heads", "packed"]))
        # no drawn case costs more than the largest listed one; fp32 products run at a sixteenth of bf16's rate
        cap = 0.5 * work(listed()[3])["flops"] / (8 if dtype == "f32" else 1)
        while work(c)["flops"] > cap or c["B"] * c["H"] * c["Nq"] * c["Nk"] > 5e8:
            c["Nq"] = max(1, c["Nq"] * 2 // 3)
            c["Nk"] = max(24, c["Nk"] * 3 // 4)
        return c
    if op == "rope":
        axes = rng.randint(1, 4)
        D = rng.choice([16, 24, 32, 48, 64, 96, 128])
        rot = rng.choice([D, D, D // 2 // 2 * 2])
        Hk = rng.choice([1, 2, 4, 8, 16])
        H = Hk * rng.choice([1, 2, 4])
        B = rng.randint(1, 8)
        N = max(1, min(_logint(rng, 1, 40000), 60_000_000 // (B * (H + Hk) * D)))
        return dict(op="rope", train=rng.random() < 0.5, dtype=rng.choice(["bf16", "f32"]), B=B, N=N, H=H, Hk=Hk, D=D,
                    rot=rot, axes=axes, pairs=rng.choice(["half", "interleaved", "axis"]),
                    store=rng.choice(["tokens", "heads", "packed"]), far=rng.random() < 0.5)
    C = rng.choice([_logint(rng, 16, 6000), 64 * rng.randint(1, 64), 8 * rng.randint(1, 512)])
    G = rng.randint(1, 8)
    rows = max(1, min(_logint(rng, 1, 8000), 60_000_000 // (G * C)))
    dtype = rng.choice(["bf16", "f32"])
    return dict(op="norm", train=rng.random() < 0.5, dtype=dtype, res=rng.choice(["f32", dtype]), G=G, rows=rows, C=C,
                post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["none", "rms", "layer", "layer"]),
                affine=rng.random() < 0.5)


def _sections(c):
    n, a = c["rot"] // 2, c["axes"]
    return [n // a + (1 if i < n % a else 0) for i in range(a)]


def work(c):
    e = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "attn":
        # ragged lengths and masks leave three quarters of the keys on average
        nk = c["Nk"] * (1.0 if c["pad"] == "none" else 0.75)
        qe, ke = c["B"] * c["Nq"] * c["H"] * c["D"], c["B"] * nk * c["Hk"] * c["D"]
        pairs = c["B"] * c["H"] * c["Nq"] * nk * c["D"]
        if c["train"]:  # q, k, v, do read; o, dq, dk, dv written
            return {"bytes": int(e * (4 * qe + 4 * ke)), "flops": int(14 * pairs)}
        return {"bytes": int(e * (2 * qe + 2 * ke)), "flops": int(4 * pairs)}
    if c["op"] == "rope":
        n = c["B"] * c["N"] * (c["H"] + c["Hk"])
        f = 2 if c["train"] else 1
        pos = 4 * c["B"] * c["N"] * c["axes"]
        return {"bytes": f * (2 * n * c["D"] * e + pos), "flops": f * 3 * n * c["rot"]}
    r = 2 if c["res"] == "bf16" else 4
    m = c["G"] * c["rows"] * c["C"]
    has_pre = c["pre"] != "none"
    fwd = m * (2 * r + e + (e if has_pre else 0))  # h, y read; h', xn written
    bwd = m * (3 * r + 2 * e + (e if has_pre else 0)) if c["train"] else 0  # dh', dxn, h, y read; dh, dy written
    return {"bytes": fwd + bwd, "flops": m * (16 if not c["train"] else 48)}


# ---------------------------------------------------------------------------- inputs
def _heads(g, c, n, h, dt, dev):
    """[B, n, h, D] as it lies in a program: token-major, or a head-major cache seen token-major."""
    x = torch.randn(c["B"], *((h, n) if c["store"] == "heads" else (n, h)), c["D"], generator=g, device=dev).to(dt)
    return x.transpose(1, 2) if c["store"] == "heads" else x


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = _DT[c["dtype"]]
    st = {"case": c}
    if c["op"] == "attn":
        B, Nk = c["B"], c["Nk"]
        st["q"] = _heads(g, c, c["Nq"], c["H"], dt, dev)
        if c["store"] == "packed":  # one projection of the states gives k and v side by side
            kv = torch.randn(B, Nk, 2, c["Hk"], c["D"], generator=g, device=dev).to(dt)
            st["k"], st["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            st["k"], st["v"] = _heads(g, c, Nk, c["Hk"], dt, dev), _heads(g, c, Nk, c["Hk"], dt, dev)
        st["kv_len"] = st["mask"] = None
        if c["pad"] == "len":
            st["kv_len"] = torch.randint((Nk + 1) // 2, Nk + 1, (B,), generator=g, device=dev, dtype=torch.int32)
        elif c["pad"] == "mask":  # the framework's padding mask: 1.0 where a residue is there
            st["mask"] = (torch.rand(B, Nk, generator=g, device=dev) < 0.75).float()
        st["scale"] = c["D"] ** -0.5
        if c["train"]:
            st["do"] = torch.randn(B, c["Nq"], c["H"], c["D"], generator=g, device=dev).to(dt)
            for k in ("q", "k", "v"):
                st[k] = st[k].detach().requires_grad_(True)
    elif c["op"] == "rope":
        B, N = c["B"], c["N"]
        if c["store"] == "packed":
            qk = torch.randn(B, N, c["H"] + c["Hk"], c["D"], generator=g, device=dev).to(dt)
            st["q"], st["k"] = qk[:, :, :c["H"]], qk[:, :, c["H"]:]
        else:
            st["q"], st["k"] = _heads(g, c, N, c["H"], dt, dev), _heads(g, c, N, c["Hk"], dt, dev)
        # positions of a grid walked in order, the first axis slowest; `far` starts the first axis a long way out
        side = max(1, round(N ** (1.0 / c["axes"])))
        i = torch.arange(N, device=dev)
        cols = []
        for a in range(c["axes"]):
            p = i // side ** (c["axes"] - 1 - a)
            cols.append(p if a == 0 else p % side)
        pos = torch.stack(cols, -1)[None].repeat(B, 1, 1)
        off = torch.randint(0, 1_000_000 if c["far"] else 50, (B, 1), generator=g, device=dev)
        pos[..., 0] += off
        st["pos"] = pos.to(torch.int32).contiguous()
        sec = _sections(c)
        # per axis the frequencies 10000^(-i/n) of its n pairs
        st["freq"] = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device=dev) / max(n, 1))
                                for n in sec])
        st["axis"] = torch.cat([torch.full((n,), a, dtype=torch.int64, device=dev) for a, n in enumerate(sec)])
        st["first"], st["second"] = _pair_index(c, dev)
        if own:
            from mdgen_finetune_amd.cross_hip import RopeAxes

            st["plan"] = RopeAxes(sec, base=10000.0, pairs=c["pairs"], device=dev)
        if c["train"]:
            st["gq"] = torch.randn(B, N, c["H"], c["D"], generator=g, device=dev).to(dt)
            st["gk"] = torch.randn(B, N, c["Hk"], c["D"], generator=g, device=dev).to(dt)
            st["q"], st["k"] = st["q"].detach().requires_grad_(True), st["k"].detach().requires_grad_(True)
    else:
        G, R, C = c["G"], c["rows"], c["C"]
        rd = _DT[c["res"]]
        st["h"] = (2.0 * torch.randn(G, R, C, generator=g, device=dev) + 0.3).to(rd)
        st["y"] = (torch.randn(G, R, C, generator=g, device=dev) + 0.1).to(dt)
        mods = 0.5 * torch.randn(G, 3 * C, generator=g, device=dev)  # one adaLN row per group: gate | shift | scale
        st["mods"] = mods
        st["rs"] = 0.9
        st["w"] = {}
        if c["affine"]:
            for side in ("post", "pre"):
                if c[side] != "none":
                    st["w"][side + "_w"] = 1.0 + 0.2 * torch.randn(C, generator=g, device=dev)
                    if c[side] == "layer":
                        st["w"][side + "_b"] = 0.2 * torch.randn(C, generator=g, device=dev)
        if c["train"]:
            st["gh"] = torch.randn(G, R, C, generator=g, device=dev).to(rd)
            st["gx"] = torch.randn(G, R, C, generator=g, device=dev).to(dt) if c["pre"] != "none" else None
            for k in ("h", "y", "mods"):
                st[k].requires_grad_(True)
            for t in st["w"].values():
                t.requires_grad_(True)
    return st


def _pair_index(c, dev):
    """Columns (first, second) of each rotated pair, in the order of the sections' pairs."""
    n = c["rot"] // 2
    p = torch.arange(n, device=dev)
    if c["pairs"] == "half":
        return p, p + n
    if c["pairs"] == "interleaved":
        return 2 * p, 2 * p + 1
    first, base = [], 0
    second = []
    for s in _sections(c):
        i = torch.arange(s, device=dev)
        first.append(base + i)
        second.append(base + s + i)
        base += 2 * s
    return torch.cat(first), torch.cat(second)


# ---------------------------------------------------------------------------- one pass
def run(st):
    op = st["case"]["op"]
    if own:
        return {"attn": _own_attn, "rope": _own_rope, "norm": _own_norm}[op](st)
    with torch.no_grad():
        return {"attn": _plain_attn, "rope": _plain_rope, "norm": _plain_norm}[op](st)


def _own_attn(st):
    from mdgen_finetune_amd.cross_hip import cross_attention

    c = st["case"]
    if not c["train"]:
        with torch.no_grad():
            return cross_attention(st["q"], st["k"], st["v"], mask=st["mask"], kv_len=st["kv_len"], scale=st["scale"])
    o = cross_attention(st["q"], st["k"], st["v"], mask=st["mask"], kv_len=st["kv_len"], scale=st["scale"])
    return (o.detach(), *torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"]))


def _own_rope(st):
    from mdgen_finetune_amd.cross_hip import rope_axes

    if not st["case"]["train"]:
        with torch.no_grad():
            return rope_axes(st["plan"], st["pos"], st["q"], st["k"])
    q, k = rope_axes(st["plan"], st["pos"], st["q"], st["k"])
    return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (st["q"], st["k"]), (st["gq"], st["gk"])))


def _own_norm(st):
    from mdgen_finetune_amd.cross_hip import gate_residual_norm

    c = st["case"]
    C = c["C"]

    def call():
        gate, shift, scale = st["mods"].split(C, -1)
        if c["pre"] == "none":
            shift = scale = None
        return gate_residual_norm(st["h"], st["y"], gate=gate, resid_scale=st["rs"], post=c["post"], pre=c["pre"],
                                  shift=shift, scale=scale, eps=1e-6, **st["w"])

    if not c["train"]:
        with torch.no_grad():
            h, xn = call()
        return h if xn is None else (h, xn)
    h, xn = call()
    ws = [st["w"][k] for k in sorted(st["w"])]
    outs, gs = ((h,), (st["gh"],)) if xn is None else ((h, xn), (st["gh"], st["gx"]))
    grads = torch.autograd.grad(outs, (st["h"], st["y"], st["mods"], *ws), gs)
    return tuple(o.detach() for o in outs) + tuple(grads)


# plain forms: 32 bits throughout, rounded once at the end
def _keep(st):
    c = st["case"]
    keep = torch.ones(c["B"], c["Nk"], dtype=torch.bool, device=st["q"].device)
    if st["kv_len"] is not None:
        keep = torch.arange(c["Nk"], device=keep.device)[None] < st["kv_len"][:, None]
    if st["mask"] is not None:
        keep = keep & (st["mask"] != 0)
    return keep


def _plain_attn(st):
    c = st["case"]
    B, Nq, Nk, H, Hk, D = (c[k] for k in ("B", "Nq", "Nk", "H", "Hk", "D"))
    G = H // Hk
    dt = st["q"].dtype
    keep = _keep(st)

    def rows(x):  # [B, Nq, H, D] -> [B * Hk, G * Nq, D]
        return x.float().reshape(B, Nq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, G * Nq, D)

    def back(x):
        return x.reshape(B, Hk, G, Nq, D).permute(0, 3, 1, 2, 4).reshape(B, Nq, H, D).to(dt)

    def keys(x):
        x = torch.where(keep[:, :, None, None], x.float(), 0.0)
        return x.permute(0, 2, 1, 3).reshape(B * Hk, Nk, D)

    def unkeys(x):
        return x.reshape(B, Hk, Nk, D).permute(0, 2, 1, 3).contiguous().to(dt)

    q, k, v = rows(st["q"]), keys(st["k"]), keys(st["v"])
    kt = k.transpose(1, 2).contiguous()
    s = torch.bmm(q, kt) * st["scale"]
    s = s.reshape(B, Hk, G * Nq, Nk).masked_fill_(~keep[:, None, None, :], -math.inf).reshape(B * Hk, G * Nq, Nk)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    del s
    l = p.sum(-1, keepdim=True)
    p /= torch.where(l == 0, 1.0, l)
    o = torch.bmm(p, v)
    if not c["train"]:
        return back(o)
    do = rows(st["do"])
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do)
    ds = torch.bmm(do, v.transpose(1, 2).contiguous())
    ds = p * (ds - (do * o).sum(-1, keepdim=True)) * st["scale"]
    dq = torch.bmm(ds, k)
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q)
    return back(o), back(dq), unkeys(dk), unkeys(dv)


def _plain_rope(st):
    ang = st["pos"].double()[..., st["axis"]] * st["freq"]  # far positions: the angle in 64 bits
    cos, sin = ang.cos().float()[:, :, None], ang.sin().float()[:, :, None]

    def rotate(x, sign):
        x32 = x.float()
        a, b = x32[..., st["first"]], x32[..., st["second"]]
        out = x32.clone()
        out[..., st["first"]] = a * cos - b * (sign * sin)
        out[..., st["second"]] = b * cos + a * (sign * sin)
        return out.to(x.dtype)

    out = (rotate(st["q"], 1.0), rotate(st["k"], 1.0))
    if st["case"]["train"]:
        out += (rotate(st["gq"], -1.0), rotate(st["gk"], -1.0))
    return out


def _plain_norm(st):
    c = st["case"]
    w, rs, eps = st["w"], st["rs"], 1e-6
    gate, shift, scale = (t[:, None] for t in st["mods"].split(c["C"], -1))
    h, y = st["h"].float(), st["y"].float()

    def norm(x, kind):  # (x - mean) * rstd, rstd
        if kind == "none":
            return x, None
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        return x * r, r

    def affine(x, side):
        if side + "_w" in w:
            x = x * w[side + "_w"]
        if side + "_b" in w:
            x = x + w[side + "_b"]
        return x

    def norm_bwd(g, xh, r, kind):
        if kind == "none":
            return g
        g = g - xh * (g * xh).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == "layer" else 0.0)
        return g * r

    yh, ry = norm(y, c["post"])
    u = affine(yh, "post")
    h2 = rs * h + gate * u
    outs = [h2.to(st["h"].dtype)]
    if c["pre"] != "none":
        xh, rx = norm(h2, c["pre"])
        z = affine(xh, "pre")
        outs.append((z * (1 + scale) + shift).to(st["y"].dtype))
    if not c["train"]:
        return outs[0] if len(outs) == 1 else tuple(outs)
    g = st["gh"].float()
    dw = {}
    dshift = dscale = torch.zeros_like(st["mods"][:, :c["C"]])
    if c["pre"] != "none":
        gx = st["gx"].float()
        dshift, dscale = gx.sum(1), (gx * z).sum(1)
        gz = gx * (1 + scale)
        dw["pre_w"], dw["pre_b"] = (gz * xh).sum((0, 1)), gz.sum((0, 1))
        g = g + norm_bwd(gz * w["pre_w"] if "pre_w" in w else gz, xh, rx, c["pre"])
    gu = g * gate
    dw["post_w"], dw["post_b"] = (gu * yh).sum((0, 1)), gu.sum((0, 1))
    dy = norm_bwd(gu * w["post_w"] if "post_w" in w else gu, yh, ry, c["post"])
    dmods = torch.cat([(g * u).sum(1), dshift, dscale], -1)
    return tuple(outs) + ((rs * g).to(st["h"].dtype), dy.to(st["y"].dtype), dmods) + tuple(dw[k] for k in sorted(w))


# ---------------------------------------------------------------------------- from the definition, in 64 bits
def exact(c, seed):
    st = prepare(c, seed)
    with torch.enable_grad():
        return {"attn": _exact_attn, "rope": _exact_rope, "norm": _exact_norm}[c["op"]](st)


def _leaf(x, train):
    return x.detach().double().requires_grad_(train)


def _exact_attn(st):
    c = st["case"]
    G, train = c["H"] // c["Hk"], c["train"]
    keep = _keep(st)
    o = torch.zeros(c["B"], c["Nq"], c["H"], c["D"], dtype=torch.float64, device=st["q"].device)
    grads = [torch.zeros(st[n].shape, dtype=torch.float64, device=o.device) for n in "qkv"] if train else []
    for b in range(c["B"]):
        idx = keep[b].nonzero()[:, 0]
        if idx.numel() == 0:
            continue
        for h in range(c["H"]):  # one head at a time, over the keys that are there
            q, k, v = (_leaf(t, train) for t in (st["q"][b, :, h], st["k"][b, idx, h // G], st["v"][b, idx, h // G]))
            out = torch.softmax(st["scale"] * (q @ k.T), -1) @ v
            o[b, :, h] = out.detach()
            if train:
                gq, gk, gv = torch.autograd.grad(out, (q, k, v), st["do"][b, :, h].double())
                grads[0][b, :, h] = gq
                grads[1][b, :, h // G].index_add_(0, idx, gk)
                grads[2][b, :, h // G].index_add_(0, idx, gv)
    return (o, *grads) if train else o


def _exact_rope(st):
    ang = st["pos"].double()[..., st["axis"]] * st["freq"]
    turn = torch.polar(torch.ones_like(ang), ang)[:, :, None]

    def rotate(x, z):
        out = x.detach().double()
        w = torch.complex(out[..., st["first"]], out[..., st["second"]]) * z
        out[..., st["first"]], out[..., st["second"]] = w.real, w.imag
        return out

    res = (rotate(st["q"], turn), rotate(st["k"], turn))
    if st["case"]["train"]:
        res += (rotate(st["gq"], turn.conj()), rotate(st["gk"], turn.conj()))
    return res


def _exact_norm(st):
    c, train = st["case"], st["case"]["train"]
    h, y, mods = (_leaf(st[k], train) for k in ("h", "y", "mods"))
    w = {k: _leaf(t, train) for k, t in st["w"].items()}

    def norm(x, kind, side):
        if kind == "layer":
            x = torch.nn.functional.layer_norm(x, (c["C"],), eps=1e-6)
        elif kind == "rms":
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6)
        return x * w.get(side + "_w", 1.0) + w.get(side + "_b", 0.0)

    gate, shift, scale = (mods[:, i * c["C"]:(i + 1) * c["C"]].unsqueeze(1) for i in range(3))
    outs = [st["rs"] * h + gate * norm(y, c["post"], "post")]
    if c["pre"] != "none":
        outs.append(norm(outs[0], c["pre"], "pre") * (1 + scale) + shift)
    if not train:
        return outs[0] if len(outs) == 1 else tuple(outs)
    gs = [st["gh"].double()] + ([st["gx"].double()] if len(outs) > 1 else [])
    leaves = (h, y, mods, *[w[k] for k in sorted(w)])
    return tuple(o.detach() for o in outs) + torch.autograd.grad(outs, leaves, gs)
