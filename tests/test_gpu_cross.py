"""The conditioned block's operators on the GPU against plain implementations in 64 bits.

Tolerances (u = half a rounding step relative to the value: bf16 2^-8, fp32 2^-24) are bounds on what
the kernels round, element by element, from the magnitudes that enter each sum:
  * an output of type t: u_t |value|;
  * a sum of n fp32 products: n 2^-24 sum |terms|;
  * bf16 attention: the probabilities (and dS) are rounded to bf16 before their product, u_bf16 of
    sum |terms|; delta = do . (o + o_lo) carries o to 2^-16;
  * scores are fp32 sums of D products: P changes by the factor exp of their error (and of the 2^-22
    of exp2 and its argument's rounding at the scores met here, below 2^7)."""
import functools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32, U16 = 2.0 ** -24, 2.0 ** -8


def X():
    from mdgen_finetune_amd import cross_hip

    return cross_hip


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _near(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), what
    if not got.numel():
        return
    bad = (got - want).abs() - tol
    assert bad.max().item() <= 0, (what, (got - want).abs().max().item(), bad.max().item())


# ------------------------------------------------------------------------------------------ attention
def _layout(x, store):
    """The same values in another layout on the GPU."""
    if store == "heads":
        return x.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    if store == "odd":  # rows that start off any 16-byte boundary
        B, n, h, d = x.shape
        buf = torch.full((B, n, h, d + 3), float("nan"), dtype=x.dtype, device="cuda")
        buf[..., 1:d + 1] = x.cuda()
        return buf[..., 1:d + 1]
    if store == "dfirst":  # the head dim is not contiguous: the call copies
        return x.cuda().permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    return x.cuda()


def _attn_inputs(B, Nq, Nk, H, Hk, D, dt, pad, seed):
    g = _gen(seed)
    q, k, v, do = (torch.randn(B, n, h, D, generator=g).to(dt) for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
    keep = torch.ones(B, Nk, dtype=torch.bool)
    qkeep = torch.ones(B, Nq, dtype=torch.bool)
    kw = {}
    if "len" in pad:
        ln = torch.randint(0, Nk + 1, (B,), generator=g, dtype=torch.int32)
        ln[0] = Nk
        keep &= torch.arange(Nk)[None] < ln[:, None]
        kw["kv_len"] = ln
    if "q" in pad:
        ln = torch.randint(0, Nq + 1, (B,), generator=g, dtype=torch.int32)
        qkeep &= torch.arange(Nq)[None] < ln[:, None]
        kw["q_len"] = ln
    if "mask" in pad:
        m = torch.rand(B, Nk, generator=g) < 0.6
        m[-1] = False  # a sequence whose mask leaves nothing
        keep &= m
        kw["mask"] = m if "bool" in pad else m.float()
    # what lies at keys that are not there is garbage of the worst kind
    if Nk:
        k[~keep] = float("nan")
        v[~keep] = float("inf")
    return q, k, v, do, keep, qkeep, kw


def _attn_oracle(q, k, v, do, keep, qkeep, scale, dt):
    """o, dq, dk, dv and their tolerances, float64 on the CPU."""
    B, Nq, H, D = q.shape
    Nk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    z = lambda t: torch.where(keep[:, :, None, None], t.double(), 0.0)  # noqa: E731
    qh = torch.where(qkeep[:, :, None, None], q.double(), 0.0).transpose(1, 2)
    gh = torch.where(qkeep[:, :, None, None], do.double(), 0.0).transpose(1, 2)
    kh, vh = (z(t).transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
    s = scale * (qh @ kh.transpose(-1, -2))
    live = (keep[:, None, None, :] & qkeep[:, None, :, None]).expand(B, H, Nq, Nk)
    s = s.masked_fill(~live, -math.inf)
    m = s.amax(-1, keepdim=True) if Nk else torch.zeros(B, H, Nq, 1, dtype=torch.float64)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    p = p / torch.where(l == 0, 1.0, l)
    o = p @ vh
    uo = U16 if dt == torch.bfloat16 else U32
    up = U16 if dt == torch.bfloat16 else 0.0
    # relative error of P: the scores' fp32 sums, exp2 and the normaliser's sum of Nk terms
    smag = scale * (qh.abs() @ kh.abs().transpose(-1, -2))
    ep = 2 * ((D + 4) * U32 * (smag.amax(-1, keepdim=True) if Nk else 0.0) + (Nk + 16) * U32 + 2.0 ** -20)
    av = p @ vh.abs()
    t_o = uo * o.abs() + (up + ep + (Nk + 8) * U32) * av
    dv = p.transpose(-1, -2) @ gh
    dvm = p.transpose(-1, -2) @ gh.abs()
    t_dv = uo * dv.abs() + ((up + Nq * U32) * dvm + (p * ep).transpose(-1, -2) @ gh.abs())
    dp = gh @ vh.transpose(-1, -2)
    delta = (gh * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # error of dS: P's, the fp32 sums of dp and delta, and o + o_lo (2^-16 of the rounded o, with its own P's error)
    dpm = gh.abs() @ vh.abs().transpose(-1, -2)
    dm = (gh.abs() * o.abs()).sum(-1, keepdim=True)
    e_o = (gh.abs() * ((2.0 ** -16 if up else U32) * o.abs() + (up + ep + (Nk + 8) * U32) * av)).sum(-1, keepdim=True)
    e_ds = up * ds.abs() + ep * ds.abs() + p * ((D + 4) * U32 * (dpm + dm) + e_o)
    dq, t_dq = scale * (ds @ kh), scale * ((e_ds + Nk * U32 * ds.abs()) @ kh.abs())
    dk = scale * (ds.transpose(-1, -2) @ qh)
    t_dk = scale * ((e_ds + Nq * G * U32 * ds.abs()).transpose(-1, -2) @ qh.abs())
    fold = lambda t: t.reshape(B, Hk, G, Nk, D).sum(2).transpose(1, 2)  # noqa: E731
    dk, t_dk, dv, t_dv = fold(dk), fold(t_dk), fold(dv), fold(t_dv)
    dq, t_dq, o, t_o = (t.transpose(1, 2) for t in (dq, t_dq, o, t_o))
    tiny = 1e-30
    return (o, dq, dk, dv), (t_o + tiny, t_dq + uo * dq.abs() + tiny, t_dk + uo * dk.abs() + tiny, t_dv + tiny)


ATTN = [  # B, Nq, Nk, H, Hk, D, padding, layout
    (1, 1, 1, 1, 1, 1, "", "tokens"),
    (2, 1, 7, 4, 4, 24, "len", "tokens"),
    (2, 1, 300, 8, 2, 128, "len", "heads"),
    (3, 5, 33, 4, 2, 20, "mask", "odd"),
    (2, 8, 64, 4, 1, 32, "q", "tokens"),        # exactly 32 packed rows
    (2, 33, 65, 3, 3, 33, "mask bool", "dfirst"),
    (1, 130, 31, 2, 1, 48, "len q", "heads"),
    (2, 64, 129, 6, 3, 64, "mask len q", "tokens"),
    (1, 257, 200, 2, 2, 96, "", "odd"),
    (1, 40, 700, 2, 1, 128, "len", "tokens"),
    (4, 3, 5, 2, 2, 16, "len mask q", "tokens"),
    (1, 2, 0, 2, 1, 8, "", "tokens"),           # an encoder without states
    # enough rows for the wide blocks of each head width
    (8, 300, 100, 16, 16, 24, "mask", "tokens"),
    (4, 520, 161, 32, 16, 64, "len q", "heads"),
    (4, 260, 133, 32, 32, 128, "mask len", "tokens"),
    (16, 257, 31, 16, 16, 40, "", "tokens"),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: "-".join(str(x) for x in c))
def test_cross_attention_forward_backward(case, dt):
    B, Nq, Nk, H, Hk, D, pad, store = case
    q, k, v, do, keep, qkeep, kw = _attn_inputs(B, Nq, Nk, H, Hk, D, dt, pad, 11)
    scale = 0.7 * D ** -0.5
    want, tol = _attn_oracle(q, k, v, do, keep, qkeep, scale, dt)
    kw = {n: t.cuda() for n, t in kw.items()}
    qc, kc, vc = (_layout(t, store) for t in (q, k, v))
    with torch.no_grad():
        _near(X().cross_attention(qc, kc, vc, scale=scale, **kw), want[0], tol[0], "o (inference)")
    leaves = [t.detach().requires_grad_(True) for t in (qc, kc, vc)]
    o = X().cross_attention(*leaves, scale=scale, **kw)
    dout = do.cuda()
    dout[~qkeep.cuda()] = float("nan")  # (not read)
    grads = torch.autograd.grad(o, leaves, dout)
    for n, got, w, t in zip(("o", "dq", "dk", "dv"), (o, *grads), want, tol):
        _near(got, w, t, n)


# at most 32 rows per key head: the backward in one pass over the keys, its waves and splits, ends of sequences
FEW = [
    (1, 1, 33, 1, 1, 64, "", "tokens"),
    (2, 32, 257, 2, 2, 32, "len q", "tokens"),
    (3, 4, 700, 16, 2, 128, "len mask", "heads"),
    (2, 17, 1300, 2, 2, 96, "mask", "tokens"),
    (4, 1, 2100, 16, 4, 64, "len", "odd"),
    (2, 2, 1111, 15, 1, 36, "mask bool len q", "dfirst"),
    (1, 31, 3000, 1, 1, 72, "len", "heads"),
    (2, 6, 96, 5, 1, 128, "mask len q", "odd"),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", FEW, ids=lambda c: "-".join(str(x) for x in c))
def test_cross_attention_few_rows(case, dt):
    test_cross_attention_forward_backward(case, dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("Nq,Nk,G", [(1, 5000, 4), (2, 20000, 1), (45, 6000, 1)])
def test_cross_attention_splits_a_long_key_axis(Nq, Nk, G, dt):
    """Few rows over many keys: the splits' partial softmaxes joined, ragged lengths (0 and 1 among them)."""
    B, Hk, D = 3, 2, 40
    q, k, v, do, keep, qkeep, _ = _attn_inputs(B, Nq, Nk, Hk * G, Hk, D, dt, "", 5)
    ln = torch.tensor([Nk - 3, 0, 1], dtype=torch.int32)
    keep = torch.arange(Nk)[None] < ln[:, None]
    want, tol = _attn_oracle(q, k, v, do, keep, qkeep, D ** -0.5, dt)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = X().cross_attention(*leaves, kv_len=ln.cuda())
    grads = torch.autograd.grad(o, leaves, do.cuda())
    for n, got, w, t in zip(("o", "dq", "dk", "dv"), (o, *grads), want, tol):
        _near(got, w, t, n)
    with torch.no_grad():
        assert torch.equal(X().cross_attention(*leaves, kv_len=ln.cuda()), o)


def test_cross_attention_broadcast_inputs_and_frozen_encoder():
    """k / v shared by the batch (stride 0): their gradient is the batch's sum; a frozen encoder gets none and
    dq is the same bits."""
    B, Nq, Nk, H, D = 3, 37, 50, 2, 24
    q, k, v, do, *_ = _attn_inputs(B, Nq, Nk, H, H, D, torch.float32, "", 3)
    k1, v1 = k[:1], v[:1]
    ke, ve = k1.expand(B, -1, -1, -1), v1.expand(B, -1, -1, -1)
    ones = torch.ones(B, Nk, dtype=torch.bool)
    want, tol = _attn_oracle(q, ke, ve, do, ones, torch.ones(B, Nq, dtype=torch.bool), D ** -0.5, torch.float32)
    ql, kl, vl = (t.cuda().requires_grad_(True) for t in (q, k1, v1))
    o = X().cross_attention(ql, kl.expand(B, -1, -1, -1), vl.expand(B, -1, -1, -1))
    dq, dk, dv = torch.autograd.grad(o, (ql, kl, vl), do.cuda())
    _near(o, want[0], tol[0], "o")
    _near(dk, want[2].sum(0, keepdim=True), tol[2].sum(0, keepdim=True) + 4 * U32 * want[2].abs().sum(0), "dk")
    _near(dv, want[3].sum(0, keepdim=True), tol[3].sum(0, keepdim=True) + 4 * U32 * want[3].abs().sum(0), "dv")
    of = X().cross_attention(ql, kl.detach().expand(B, -1, -1, -1), vl.detach().expand(B, -1, -1, -1))
    (dqf,) = torch.autograd.grad(of, ql, do.cuda())
    assert torch.equal(dqf, dq)
    # a gradient that arrives expanded (as of a sum) and one in another order
    (ds,) = torch.autograd.grad(X().cross_attention(ql, kl.detach().expand(B, -1, -1, -1), vl.detach().expand(B, -1, -1, -1)).sum(), ql)
    assert torch.isfinite(ds).all()


@pytest.mark.parametrize("dt,D", [(torch.bfloat16, 128), (torch.bfloat16, 24), (torch.float32, 64)], ids=str)
def test_cross_attention_few_rows_frozen_broadcast_captured(dt, D):
    """Three query tokens in two splits: what masked keys hold (NaN) is without effect, a frozen encoder's dq is the
    same bits, k and v shared by the batch, and a captured pass replayed on new inputs."""
    B, Nq, Nk, H, Hk = 2, 3, 900, 4, 2
    g = _gen(77)
    q, k, v, do = (torch.randn(B, n, h, D, generator=g).to(dt).cuda() for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
    ln = torch.tensor([900, 411], dtype=torch.int32, device="cuda")
    mask = (torch.rand(B, Nk, generator=g) < 0.8).cuda()
    gone = ~mask | (torch.arange(Nk, device="cuda")[None] >= ln[:, None])

    def grads(q, k, v, do, **kw):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(X().cross_attention(*leaves, mask=mask, kv_len=ln, **kw), leaves, do)

    base = grads(q, k, v, do)
    kn, vn = (torch.where(gone[..., None, None], float("nan"), t) for t in (k, v))
    again = grads(q, kn, vn, do)
    assert all(torch.equal(a, b) for a, b in zip(base, again))
    assert not base[1][gone].any() and not base[2][gone].any()
    ql = q.clone().requires_grad_(True)
    (dq,) = torch.autograd.grad(X().cross_attention(ql, k, v, mask=mask, kv_len=ln), ql, do)
    assert torch.equal(dq, base[0])
    wide = [t.expand(B, -1, -1, -1) for t in (k[:1], v[:1])]
    assert all(torch.equal(a, b) for a, b in zip(grads(q, *wide, do), grads(q, *(t.contiguous() for t in wide), do)))

    static = [t.clone() for t in (q, k, v, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(*static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads(*static)
    for turn in range(4):
        new = [torch.randn(t.shape, generator=g).to(dt).cuda() for t in static]
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        want = grads(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_cross_attention_gradient_against_differences():
    B, Nq, Nk, H, D = 1, 3, 6, 2, 8
    q, k, v, do, *_ = _attn_inputs(B, Nq, Nk, H, 1, D, torch.float32, "", 9)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(X().cross_attention(*leaves), leaves, do.cuda())
    f = lambda xs: (X().cross_attention(*xs).double() * do.cuda().double()).sum().item()  # noqa: E731
    eps = 2.0 ** -6
    with torch.no_grad():
        for which, at in ((0, (0, 1, 1, 3)), (1, (0, 4, 0, 2)), (2, (0, 2, 0, 7))):
            hi, lo = ([t.detach().clone() for t in leaves] for _ in range(2))
            hi[which][at] += eps
            lo[which][at] -= eps
            num = (f(hi) - f(lo)) / (2 * eps)
            # the difference's own error: eps^2 / 6 of a third derivative below 8, and 48 fp32 outputs' rounding over 2 eps
            assert abs(num - grads[which][at].item()) < eps * eps / 6 * 8 + 48 * 8 * U32 * 4 / eps


def test_cross_attention_large_scores_and_ties():
    """Scores far above and below zero (a raised maximum in later tiles), and equal scores."""
    B, Nq, Nk, D = 1, 40, 300, 16
    q = torch.ones(B, Nq, 1, D)
    k = torch.zeros(B, Nk, 1, D)
    k[0, :, 0, 0] = torch.linspace(-300, 300, Nk).round()
    v = torch.randn(B, Nk, 1, D, generator=_gen(0))
    one = torch.ones(B, Nk, dtype=torch.bool)
    for dt in (torch.float32, torch.bfloat16):
        args = [t.to(dt) for t in (q, k, v)]
        want, tol = _attn_oracle(*args, args[0], one, torch.ones(B, Nq, dtype=torch.bool), 1.0, dt)
        # exponents up to 600 * log2 e < 2^10: the argument of exp2 is rounded by 2^-14
        _near(X().cross_attention(*(t.cuda() for t in args), scale=1.0), want[0], tol[0] + 2.0 ** -13 * 4, "o")
        z = torch.zeros_like(args[1])
        w2, t2 = _attn_oracle(args[0], z, args[2], args[0], one, torch.ones(B, Nq, dtype=torch.bool), 1.0, dt)
        _near(X().cross_attention(args[0].cuda(), z.cuda(), args[2].cuda(), scale=1.0), w2[0], t2[0], "ties")
    # a NaN among the keys that are there stays one
    k[0, 7] = float("nan")
    assert torch.isnan(X().cross_attention(q.cuda(), k.cuda(), v.cuda(), scale=1.0)).all()
    assert torch.isnan(X().cross_attention(q[:, :1].cuda(), k.cuda(), v.cuda(), scale=1.0)).all()


def test_cross_attention_offsets_past_32_bits():
    """A single token over a cache whose last keys lie past 2^31 elements, and lengths clamped to the cache."""
    B, Nk, H, D = 1, 140000, 130, 128  # 2.3e9 elements each of k and v in bf16
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GiB")
    kv = torch.zeros(Nk, H, D, dtype=torch.bfloat16, device="cuda")[None]
    q = torch.ones(B, 1, H, D, dtype=torch.bfloat16, device="cuda")
    kv[0, -1] = 4.0  # score 4 * 128 / sqrt(128) above the rest: the last key takes the whole softmax
    o = X().cross_attention(q, kv, kv, kv_len=torch.tensor([2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert (o - 4.0).abs().max().item() <= 4 * U16
    o = X().cross_attention(q, kv, kv, kv_len=torch.tensor([Nk - 1], dtype=torch.int32, device="cuda"))
    assert o.abs().max().item() == 0
    o = X().cross_attention(q, kv, kv, kv_len=torch.tensor([-5], dtype=torch.int32, device="cuda"))
    assert o.abs().max().item() == 0


# ------------------------------------------------------------------------------------------ rotary
def _rope_oracle(x, pos, sections, pairs, base, sign):
    cols = X().RopeAxes(sections, pairs=pairs, device="cpu").cols.long()
    n = sum(sections)
    axis = torch.cat([torch.full((s,), a) for a, s in enumerate(sections)]).long()
    freq = torch.tensor([base ** (-i / s) for s in sections for i in range(s)], dtype=torch.float64)
    ang = (pos.double()[..., axis] * freq)[:, :, None]
    out = x.double().clone()
    a, b = x.double()[..., cols[:n]], x.double()[..., cols[n:]]
    out[..., cols[:n]] = a * ang.cos() - sign * b * ang.sin()
    out[..., cols[n:]] = b * ang.cos() + sign * a * ang.sin()
    mag = out.abs().clone()
    mag[..., cols[:n]] = mag[..., cols[n:]] = a.abs() + b.abs()
    return out, mag


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("pairs", ["half", "interleaved", "axis"])
@pytest.mark.parametrize("B,N,H,Hk,D,sections,store", [  # (runs of one or two pairs in whole 16-byte pieces)
    (2, 300, 5, 3, 64, [11, 11, 9], "tokens"), (1, 77, 2, 1, 24, [6, 6], "heads"), (3, 40, 40, 8, 32, [3, 5], "tokens"),
    (1, 2, 300, 20, 16, [1, 0, 6], "tokens"), (5, 1, 1, 1, 8, [1, 1], "heads"), (2, 700, 3, 1, 128, [14, 18, 2], "tokens"),
    (1, 5, 48, 12, 128, [7, 9], "tokens"), (1, 3, 64, 64, 128, [5, 5, 3], "tokens"),
])
def test_rope_axes_short_runs(B, N, H, Hk, D, sections, store, pairs, dt):
    test_rope_axes_forward_backward(B, N, H, Hk, D, sections, store, pairs, dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("pairs", ["half", "interleaved", "axis"])
@pytest.mark.parametrize("B,N,H,Hk,D,sections,store", [
    (1, 1, 1, 1, 2, [1], "tokens"), (2, 5, 4, 2, 24, [6, 6], "tokens"), (3, 7, 2, 1, 64, [8, 8, 16], "heads"),
    (2, 9, 3, 3, 33, [3, 5, 0, 7], "odd"), (1, 300, 12, 4, 128, [16, 24, 24], "tokens"), (2, 4, 40, 8, 48, [16], "dfirst"),
    (1, 6001, 8, 8, 64, [16, 16], "tokens"),
])
def test_rope_axes_forward_backward(B, N, H, Hk, D, sections, store, pairs, dt):
    g = _gen(2)
    q, k, gq, gk = (torch.randn(B, N, h, D, generator=g).to(dt) for h in (H, Hk, H, Hk))
    pos = torch.randint(-1000, 1_000_000, (B, N, len(sections)), generator=g)
    plan = X().RopeAxes(sections, pairs=pairs, device="cuda")
    u = U16 if dt == torch.bfloat16 else U32
    # per output: its rounding, two fp32 products and their sum, and 2^-22 of cos / sin (the reduced angle in fp32)
    lim = lambda o, m: u * o.abs() + (4 * U32 + 2.0 ** -22) * m + 1e-30  # noqa: E731
    ql, kl = (_layout(t, store).detach().requires_grad_(True) for t in (q, k))
    for p in (pos.to(torch.int32).cuda(), pos.cuda()):
        qo, ko = X().rope_axes(plan, p, ql, kl)
        for got, x in ((qo, q), (ko, k)):
            w, m = _rope_oracle(x, pos, sections, pairs, 10000.0, 1.0)
            _near(got, w, lim(w, m), "rotated")
    dq, dk = torch.autograd.grad((qo, ko), (ql, kl), (gq.cuda(), gk.cuda()))
    for got, x in ((dq, gq), (dk, gk)):
        w, m = _rope_oracle(x, pos, sections, pairs, 10000.0, -1.0)
        _near(got, w, lim(w, m), "gradient")
    with torch.no_grad():  # one tensor, the inverse, in place, shared positions
        one = X().rope_axes(plan, pos.cuda(), ql)
        assert torch.equal(one, qo)
        back = X().rope_axes(plan, pos.cuda(), gq.cuda(), inverse=True)
        assert torch.equal(back, dq)
        if store != "dfirst":
            buf = _layout(q, store).clone(memory_format=torch.preserve_format)
            kb = _layout(k, "tokens").clone()
            r = X().rope_axes(plan, pos.cuda(), buf, kb, inplace=True)
            assert r[0] is buf and torch.equal(buf, qo) and torch.equal(kb, ko)
        sh = X().rope_axes(plan, pos[:1].cuda(), ql)
        w, m = _rope_oracle(q, pos[:1].expand(B, -1, -1), sections, pairs, 10000.0, 1.0)
        _near(sh, w, lim(w, m), "shared positions")


def test_rope_axes_inplace_refusals():
    plan = X().RopeAxes([4], device="cuda")
    x = torch.zeros(1, 3, 2, 8, device="cuda")
    pos = torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        X().rope_axes(plan, pos, x.requires_grad_(True), inplace=True)
    with pytest.raises(ValueError):
        X().rope_axes(plan, pos, x.detach()[:, :1].expand(1, 3, 2, 8), inplace=True)
    with pytest.raises(TypeError):
        X().rope_axes(plan, pos.float(), x.detach())
    with pytest.raises(ValueError):
        X().rope_axes(plan, pos[:2], x.detach())
    with pytest.raises(ValueError):
        X().rope_axes(plan, pos.cpu(), x.detach())
    assert X().rope_axes(plan, pos[:0], x.detach()[:, :0]).shape == (1, 0, 2, 8)


# ------------------------------------------------------------------------------------------ norms
def _grn_oracle(t, G, post, pre, rs, eps, gh, gx):
    """float64 autograd from the definition: outputs, gradients by name."""
    leaf = {n: (None if x is None else x.double().requires_grad_(True)) for n, x in t.items()}
    C = t["h"].shape[-1]
    h, y = leaf["h"].reshape(G, -1, C), None if leaf["y"] is None else leaf["y"].reshape(G, -1, C)

    def norm(x, kind, w, b):
        if kind == "layer":
            x = x - x.mean(-1, keepdim=True)
        if kind != "none":
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + eps)
        x = x if w is None else x * w
        return x if b is None else x + b

    row = lambda n: leaf[n][:, None]  # noqa: E731
    ho = rs * h
    if y is not None:
        u = norm(y, post, leaf["post_w"], leaf["post_b"])
        ho = ho + (u if leaf["gate"] is None else row("gate") * u)
    outs, gs = [ho], [gh.double().reshape(G, -1, C)]
    if pre != "none":
        z = norm(ho, pre, leaf["pre_w"], leaf["pre_b"])
        z = z if leaf["scale"] is None else z * (1 + row("scale"))
        outs.append(z if leaf["shift"] is None else z + row("shift"))
        gs.append(gx.double().reshape(G, -1, C))
    names = [n for n, x in leaf.items() if x is not None]
    grads = torch.autograd.grad(outs, [leaf[n] for n in names], gs, allow_unused=True)
    return [o.detach().reshape(t["h"].shape) for o in outs], dict(zip(names, grads))


GRN = [  # G, rows, C, post, pre, gate/mod/affine, type of h
    (1, 1, 1, "none", "rms", "", "f32"),
    (4, 1, 384, "rms", "layer", "gate mod", "f32"),
    (2, 33, 64, "layer", "rms", "gate mod affine", "same"),
    (3, 70, 24, "rms", "none", "gate", "f32"),
    (2, 5, 129, "layer", "layer", "gate mod affine", "f32"),
    (1, 9, 3001, "rms", "layer", "affine", "same"),
    (5, 40, 1000, "rms", "rms", "mod", "same"),
    (2, 3, 4096, "layer", "rms", "gate mod affine", "same"),
    (1, 2, 8192, "none", "layer", "gate mod affine", "f32"),
    (1, 300, 512, "layer", "layer", "", "f32"),
    (1, 4, 2050, "rms", "rms", "gate mod affine", "same"),
    (7, 1, 200, "noy", "layer", "mod affine", "same"),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", GRN, ids=lambda c: "-".join(str(x) for x in c))
def test_gate_residual_norm_forward_backward(case, dt):
    G, rows, C, post, pre, opts, res = case
    rdt = torch.float32 if res == "f32" else dt
    g = _gen(4)
    rs, eps = 0.75, 1e-5
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    noy = post == "noy"
    post = "none" if noy else post
    t = {"h": (2 * rnd(G, rows, C) + 0.5).to(rdt), "y": None if noy else (rnd(G, rows, C) - 0.2).to(dt)}
    t["gate"] = rnd(G, C) if "gate" in opts else None
    t["shift"], t["scale"] = (0.3 * rnd(G, C) if "mod" in opts else None for _ in range(2))
    t["post_w"] = 1 + 0.2 * rnd(C) if "affine" in opts and post != "none" else None
    t["post_b"] = 0.2 * rnd(C) if "affine" in opts and post == "layer" else None
    t["pre_w"] = 1 + 0.2 * rnd(C) if "affine" in opts else None
    t["pre_b"] = 0.2 * rnd(C) if "affine" in opts and pre == "layer" else None
    xdt = rdt if noy else dt
    gh, gx = rnd(G, rows, C).to(rdt), rnd(G, rows, C).to(xdt)
    outs, grads = _grn_oracle(t, G, post, pre, rs, eps, gh, gx)
    dev = {n: (None if x is None else x.cuda().requires_grad_(True)) for n, x in t.items()}
    kw = {n: x for n, x in dev.items() if n not in ("h", "y")}
    ho, xn = X().gate_residual_norm(dev["h"], dev["y"], resid_scale=rs, post=post, pre=pre, eps=eps, **kw)
    got_o = [ho] if xn is None else [ho, xn]
    names = [n for n, x in dev.items() if x is not None]
    got_g = torch.autograd.grad(got_o, [dev[n] for n in names], [gh.cuda(), gx.cuda()][:len(got_o)])
    u = lambda d: U16 if d == torch.bfloat16 else U32  # noqa: E731
    # fp32 rows: sums of C terms (mean, variance) scale every value of the row, a few products follow; the
    # magnitudes of the terms are bounded by the row's own largest ones
    f32 = (C + 64) * U32
    for n, o, w in zip(("h_out", "xn"), got_o, outs):
        _near(o, w, u(o.dtype) * w.abs() + f32 * (4 + w.abs().amax(-1, keepdim=True)), n)
    M = G * rows
    for n, o in zip(names, got_g):
        w = grads[n]
        if n in ("h", "y"):
            # C = 1 rows and rows of tiny variance: gradients of a norm scale with 1 / std
            big = w.abs().amax(-1, keepdim=True) + 4
            _near(o, w, u(o.dtype) * w.abs() + 4 * f32 * big, n)
        else:  # column sums over the rows: terms up to 5 * 5 in magnitude, M of them, fp32
            k = M if n in ("post_w", "post_b", "pre_w", "pre_b") else rows
            _near(o, w, (k + C + 64) * U32 * 16 * math.sqrt(k) * 4, n)
    with torch.no_grad():
        h2, x2 = X().gate_residual_norm(dev["h"], dev["y"], resid_scale=rs, post=post, pre=pre, eps=eps, **kw)
        assert torch.equal(h2, ho) and (xn is None or torch.equal(x2, xn))


def test_gate_residual_norm_strided_rows_and_partial_gradients():
    """h and y as column slices of wider rows, adaLN rows as chunks of one projection; gradients of some inputs only,
    and of one output only."""
    g = _gen(8)
    G, R, C = 3, 11, 96
    wide = torch.randn(G, R, 3 * C, generator=g).cuda()
    mods = torch.randn(G, 3 * C, generator=g).cuda().requires_grad_(True)
    h, y = wide[..., C:2 * C], wide[..., 2 * C:]
    gate, shift, scale = mods.split(C, -1)
    ho, xn = X().gate_residual_norm(h, y, gate=gate, shift=shift, scale=scale, post="rms")
    hc, xc = X().gate_residual_norm(h.contiguous(), y.contiguous(), gate=gate.contiguous(), shift=shift.contiguous(),
                                    scale=scale.contiguous(), post="rms")
    assert torch.equal(ho, hc) and torch.equal(xn, xc)
    (d1,) = torch.autograd.grad(xn.sum() + (ho * 2).sum(), mods, retain_graph=True)
    (d2,) = torch.autograd.grad(xc.sum() + (hc * 2).sum(), mods)
    assert torch.equal(d1, d2)
    (dh_only,) = torch.autograd.grad(ho.sum(), mods, retain_graph=True)
    assert dh_only[:, C:].abs().max().item() == 0 and dh_only[:, :C].abs().max().item() > 0
    hl = h.detach().clone().requires_grad_(True)
    _, x1 = X().gate_residual_norm(hl, pre="rms")
    (gr,) = torch.autograd.grad(x1, hl, torch.ones_like(x1))
    h64 = hl.detach().double().cpu().requires_grad_(True)
    w = h64 / torch.sqrt((h64 ** 2).mean(-1, keepdim=True) + 1e-6)
    (wg,) = torch.autograd.grad(w.sum(), h64)
    _near(gr, wg, 4 * (C + 64) * U32 * (wg.abs().amax(-1, keepdim=True) + 4), "dh of a pre norm alone")


def test_gate_residual_norm_empty_and_constant_rows():
    e = torch.zeros(2, 0, 16, device="cuda", requires_grad=True)
    ho, xn = X().gate_residual_norm(e, e.detach(), gate=torch.zeros(2, 16, device="cuda"))
    assert ho.shape == xn.shape == (2, 0, 16)
    c = torch.full((3, 48), 7.0, device="cuda")  # a layer norm of equal values: zeros, eps in the root
    _, xn = X().gate_residual_norm(c, pre="layer")
    assert xn.abs().max().item() <= 48 * U32 * 7 / 1e-3
    _, xz = X().gate_residual_norm(torch.zeros(3, 48, device="cuda"), pre="rms")
    assert xz.abs().max().item() == 0


# ------------------------------------------------------------------------------------------ together
def _block(x, states, mask, P, plan, pos, ops):
    """A conditioned block: tokens on (frame, residue) axes attend to an encoder's states, then an MLP."""
    B, N, C = x.shape
    H, Hk = 4, 2
    D = C // H
    gate, shift, scale, gate2 = P["mods"].split(C, -1)
    _, xn = ops.gate_residual_norm(x, pre="rms", pre_w=P["w0"], shift=shift, scale=scale)
    q = (xn @ P["wq"]).reshape(B, N, H, D)
    k, v = (states @ P["wkv"]).reshape(B, -1, 2, Hk, D).unbind(2)
    q = ops.rope_axes(plan, pos, q)
    y = ops.cross_attention(q, k, v, mask=mask).reshape(B, N, C) @ P["wo"]
    x, xn = ops.gate_residual_norm(x, y, gate=gate, post="rms", post_w=P["w1"], pre="layer")
    y = torch.nn.functional.gelu(xn @ P["w_up"]) @ P["w_dn"]
    x, _ = ops.gate_residual_norm(x, y, gate=gate2, post="layer", pre="none")
    return x


class _Plain:
    """The three operators in elementary 64-bit operations."""

    @staticmethod
    def gate_residual_norm(h, y=None, gate=None, shift=None, scale=None, post="none", pre="layer", post_w=None, pre_w=None):
        def norm(x, kind, w):
            if kind == "layer":
                x = x - x.mean(-1, keepdim=True)
            if kind != "none":
                x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + 1e-6)
            return x if w is None else x * w

        if y is not None:
            u = norm(y, post, post_w)
            h = h + (u if gate is None else gate[:, None] * u)
        if pre == "none":
            return h, None
        xn = norm(h, pre, pre_w)
        return h, xn if scale is None else xn * (1 + scale[:, None]) + shift[:, None]

    @staticmethod
    def rope_axes(plan, pos, x):
        c, n = plan.cols.long().cpu(), plan.npairs
        ang = (pos.double().cpu()[..., plan.axis.long().cpu()] * plan.turns.cpu() * 2 * math.pi)[:, :, None]
        a, b = x[..., c[:n]], x[..., c[n:]]
        out = x.clone()
        out[..., c[:n]] = a * ang.cos() - b * ang.sin()
        out[..., c[n:]] = b * ang.cos() + a * ang.sin()
        return out

    @staticmethod
    def cross_attention(q, k, v, mask):
        G = q.shape[2] // k.shape[2]
        kh, vh = (t.transpose(1, 2).repeat_interleave(G, 1) for t in (k, v))
        s = q.transpose(1, 2) @ kh.transpose(-1, -2) * q.shape[-1] ** -0.5
        p = torch.softmax(s.masked_fill(~mask.cpu().bool()[:, None, None], -math.inf), -1)
        return (p @ vh).transpose(1, 2)


def _block_case(seed=1):
    g = _gen(seed)
    B, T, L, C, S, Cs = 2, 9, 4, 96, 21, 40
    x, states = torch.randn(B, T * L, C, generator=g), torch.randn(B, S, Cs, generator=g)
    w = lambda i, o: torch.randn(i, o, generator=g) / math.sqrt(i)  # noqa: E731
    P = {"mods": 0.5 * torch.randn(B, 4 * C, generator=g), "w0": 1 + 0.1 * torch.randn(C, generator=g),
         "w1": 1 + 0.1 * torch.randn(C, generator=g), "wq": w(C, C), "wkv": w(Cs, 2 * 2 * (C // 4)), "wo": w(C, C),
         "w_up": w(C, 2 * C), "w_dn": w(2 * C, C)}
    mask = (torch.rand(B, S, generator=g) < 0.7).float()
    n = torch.arange(T * L)
    pos = torch.stack([n // L, n % L], -1)[None].to(torch.int32)
    return x, states, P, mask, pos


def test_conditioned_block_forward_and_gradients():
    x, states, P, mask, pos = _block_case()
    plan = X().RopeAxes([8, 4], device="cuda")

    def run(dev, dt, ops):
        leaf = {n: t.to(dev, dt).requires_grad_(True) for n, t in {"x": x, "states": states, **P}.items()}
        out = _block(leaf["x"], leaf["states"], mask.to(dev), leaf, plan, pos.to(dev), ops)
        go = torch.linspace(-1, 1, out.numel(), device=dev, dtype=dt).reshape(out.shape)
        return out, dict(zip(leaf, torch.autograd.grad(out, list(leaf.values()), go)))

    got, gg = run("cuda", torch.float32, X())
    want, wg = run("cpu", torch.float64, _Plain)
    # six products of up to 192 terms and four norms, each within (terms + 64) 2^-24 of its row's magnitude and
    # amplified at most 4x by the next: 10 * 256 * 4 * 2^-24 of the largest value
    lim = 10 * 256 * 4 * U32
    _near(got, want.detach(), lim * want.abs().max().item(), "block")
    for n in wg:
        _near(gg[n], wg[n], 4 * lim * wg[n].abs().max().item(), "d" + n)


def test_conditioned_block_captured_and_replayed():
    """Forward and backward in one graph, replayed with new inputs between eager runs; every replay equals the
    eager bits."""
    x, states, P, mask, pos = _block_case()
    plan = X().RopeAxes([8, 4], device="cuda")
    mask, pos = mask.cuda(), pos.cuda()
    static = {n: t.cuda().requires_grad_(True) for n, t in {"x": x, "states": states, **P}.items()}
    go = torch.randn(x.shape, generator=_gen(6)).cuda()

    def step(leaf):
        out = _block(leaf["x"], leaf["states"], mask, leaf, plan, pos, X())
        return (out.detach(), *torch.autograd.grad(out, list(leaf.values()), go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i in range(4):
        fresh = {n: (t.detach() * (1 + 0.1 * i) + 0.01 * i) for n, t in static.items()} if i else None
        if fresh:
            with torch.no_grad():
                for n in static:
                    static[n].copy_(fresh[n])
        graph.replay()
        torch.cuda.synchronize()
        eager = step({n: t.detach().clone().requires_grad_(True) for n, t in static.items()})
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), i


def test_operators_on_another_stream_and_repeatable():
    q, k, v, do, *_ = _attn_inputs(2, 150, 333, 4, 2, 48, torch.bfloat16, "", 21)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    do = do.cuda()

    def once():
        o = X().cross_attention(*leaves)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    base = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(base, once()))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    res = []
    for s in (s1, s2):  # two calls at once on streams of their own
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            res.append(once())
    torch.cuda.synchronize()
    for r in res:
        assert all(torch.equal(a, b) for a, b in zip(base, r))


# ------------------------------------------------------------------------------------------ autograd's corners
def _small(seed=2):
    g = _gen(seed)
    q, k, v = (torch.randn(2, n, 2, 16, generator=g).cuda() for n in (5, 9, 9))
    h, y = torch.randn(2, 5, 32, generator=g).cuda(), torch.randn(2, 5, 32, generator=g).cuda()
    gate = torch.randn(2, 32, generator=g).cuda()
    plan = X().RopeAxes([4, 4], device="cuda")
    pos = torch.randint(0, 50, (5, 2), generator=g).cuda()
    return [(lambda q, k, v: X().cross_attention(q, k, v), (q, k, v)),
            (lambda q: X().rope_axes(plan, pos, q), (q,)),
            (lambda h, y, gate: sum(X().gate_residual_norm(h, y, gate=gate, post="rms")), (h, y, gate))]


@pytest.mark.parametrize("which", range(3), ids=["attention", "rope", "norms"])
def test_once_differentiable(which):
    """create_graph returns the same gradients; differentiating them raises, and so does a second backward."""
    f, ins = _small()[which]
    leaves = [t.clone().requires_grad_(True) for t in ins]
    base = torch.autograd.grad(f(*leaves).sum(), leaves)
    again = torch.autograd.grad(f(*leaves).sum(), leaves, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(base, again))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(sum(a.sum() for a in again), leaves)
    out = f(*leaves)
    out.sum().backward()
    with pytest.raises(RuntimeError):
        out.sum().backward()


@pytest.mark.parametrize("which", range(3), ids=["attention", "rope", "norms"])
def test_saved_tensors_moved_to_the_host(which):
    """Saved tensors that come back at other addresses (offloaded to the host between the passes)."""
    f, ins = _small()[which]
    leaves = [t.clone().requires_grad_(True) for t in ins]
    base = torch.autograd.grad(f(*leaves).sum(), leaves)
    with torch.autograd.graph.save_on_cpu():
        out = f(*leaves)
    junk = [torch.full_like(t, float("nan")) for t in ins]
    assert all(torch.equal(a, b) for a, b in zip(base, torch.autograd.grad(out.sum(), leaves)))
    del junk


def test_a_changed_input_is_noticed():
    f, ins = _small()[0]
    leaves = [t.clone().requires_grad_(True) for t in ins]
    mask = torch.ones(2, 9, device="cuda")
    out = X().cross_attention(*leaves, mask=mask)
    mask[0, 3] = 0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


def test_rope_plan_copies_and_gradient_of_one_output():
    import copy
    import pickle

    plan = X().RopeAxes([3, 5], pairs="axis", device="cuda")
    x = torch.randn(1, 7, 2, 16, device="cuda")
    pos = torch.randint(0, 99, (7, 2), device="cuda", dtype=torch.int32)
    want = X().rope_axes(plan, pos, x)
    for p in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        assert torch.equal(X().rope_axes(p, pos, x), want)
    q, k = (x.clone().requires_grad_(True) for _ in range(2))
    qo, ko = X().rope_axes(plan, pos, q, k)
    dq, dk = torch.autograd.grad(ko.sum(), (q, k), allow_unused=True)
    assert dq is None and torch.isfinite(dk).all()
    with torch.inference_mode():
        y = x.clone()
        X().rope_axes(plan, pos, y, inplace=True)
        assert torch.equal(y, want)


def test_refusals_on_the_gpu():
    x = torch.zeros(2, 3, 4, 8, device="cuda")
    for kw in (dict(mask=torch.ones(2, 4, device="cuda")), dict(mask=torch.ones(2, 3, device="cuda").half()),
               dict(kv_len=torch.ones(2, device="cuda")), dict(q_len=torch.ones(3, dtype=torch.int32, device="cuda")),
               dict(mask=torch.ones(2, 3)), dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            X().cross_attention(x, x, x, **kw)
    h = torch.zeros(6, 8, device="cuda")
    for kw in (dict(gate=torch.ones(4, 8, device="cuda")), dict(gate=torch.ones(2, 7, device="cuda")), dict(pre_w=torch.ones(9, device="cuda")),
               dict(gate=torch.ones(2, 8, device="cuda"), shift=torch.ones(3, 8, device="cuda")), dict(eps=-1.0),
               dict(resid_scale=float("inf")), dict(scale=torch.ones(2, 8, device="cuda").half())):
        with pytest.raises(ValueError):
            X().gate_residual_norm(h, h, **kw)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_operators_on_a_device_that_is_not_current():
    f, ins = _small()[0]
    torch.cuda.set_device(0)
    with torch.cuda.device(1):
        other = [t.to("cuda:1") for t in ins]
    assert torch.equal(f(*other).cpu(), f(*ins).cpu()) and torch.cuda.current_device() == 0


def test_rope_inplace_on_views_of_one_memory():
    """q and k packed in one projection, by heads or interleaved, shared heads, a head-major cache: rotated where
    they lie; views that share an element are refused."""
    plan = X().RopeAxes([2, 2], device="cuda")
    g = _gen(31)
    pos = torch.randint(0, 99, (5, 2), generator=g).cuda()

    def views(make, q, k):
        base = make()
        a, b = q(base), k(base)
        wa, wb = X().rope_axes(plan, pos[: a.shape[1]], a.clone(), b.clone())
        X().rope_axes(plan, pos[: a.shape[1]], a, b, inplace=True)
        assert torch.equal(a, wa) and torch.equal(b, wb)

    packed = lambda: torch.randn(2, 5, 10, 8, generator=g).cuda()
    views(packed, lambda x: x[:, :, :8], lambda x: x[:, :, 8:9])
    views(packed, lambda x: x[:, :, :5], lambda x: x[:, :, 5:])
    views(packed, lambda x: x[:, :, ::2], lambda x: x[:, :, 1::2])
    views(packed, lambda x: x[:, :1, :4], lambda x: x[:, :1, 4:8])
    views(packed, lambda x: x[:1], lambda x: x[1:])
    views(lambda: torch.randn(2, 10, 5, 8, generator=g).cuda(), lambda x: x[:, :6].transpose(1, 2), lambda x: x[:, 6:].transpose(1, 2))
    views(lambda: torch.randn(2, 5, 4, 16, generator=g).cuda(), lambda x: x[..., :8], lambda x: x[..., 8:])
    x = packed()
    for q, k in ((x, x), (x[:, :, :5], x[:, :, 4:9]), (x[:, :, ::2], x[:, :, 2:3]), (x[:, :, :4], x[:, :, 3:9:2])):
        with pytest.raises(ValueError, match="share memory"):
            X().rope_axes(plan, pos, q, k, inplace=True)
    with pytest.raises(ValueError, match="share|shared"):
        X().rope_axes(plan, pos, x.reshape(-1).as_strided((2, 5, 2, 8), (200, 8, 8, 1)), inplace=True)


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwad

    for f, ins in _small():
        with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            f(fwad.make_dual(ins[0], torch.ones_like(ins[0])), *ins[1:])


@pytest.mark.parametrize("which", range(3), ids=["attention", "rope", "norms"])
def test_backward_twice_with_retain_graph(which):
    f, ins = _small()[which]
    leaves = [t.clone().requires_grad_(True) for t in ins]
    out = f(*leaves)
    w = torch.randn_like(out)
    one = torch.autograd.grad(out, leaves, w, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(one, torch.autograd.grad(out, leaves, w)))


@pytest.mark.parametrize("R", [1 << 30, (1 << 31) - 1])
def test_norm_backward_of_one_long_group(R):
    """rows_per_mod past the rows' count, at the C entry: one group, the results of rows_per_mod = M bit for bit."""
    import ctypes

    from mdgen_finetune_amd import _lib

    lib, M, C, g = _lib.load(), 3000, 96, _gen(31)
    h, y, dho, dxn = (torch.randn(M, C, generator=g).cuda() for _ in range(4))
    gate, scale = (torch.randn(1, C, generator=g).cuda() for _ in range(2))
    got = []
    for rows in (M, R):
        outs = {n: torch.full((M, C), 7.0, device="cuda") for n in ("h_out", "xn", "dh", "dy")}
        outs.update({n: torch.full((C,), 7.0, device="cuda") for n in ("dgate", "dscale", "dpost_w", "dpre_w")})
        d = _lib.MdgGateResNorm(dtype=0, res_dtype=0, M=M, C=C, rows_per_mod=rows, post=1, pre=2, resid_scale=0.9, eps=1e-6,
                                h=h.data_ptr(), y=y.data_ptr(), ldh=C, ldy=C, gate=gate.data_ptr(), scale=scale.data_ptr(),
                                mod_stride=C, dmod_stride=C, dh_out=dho.data_ptr(), dxn=dxn.data_ptr(),
                                **{n: t.data_ptr() for n, t in outs.items()})
        stream = torch.cuda.current_stream().cuda_stream
        need = lib.mdg_gate_res_norm_bwd_workspace_bytes(ctypes.byref(d))
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        assert lib.mdg_gate_res_norm(ctypes.byref(d), stream) == 0, lib.mdg_last_error_string()
        assert lib.mdg_gate_res_norm_bwd(ctypes.byref(d), ws.data_ptr(), need, stream) == 0, lib.mdg_last_error_string()
        got.append((need, outs))
    assert got[0][0] == got[1][0]
    for n, t in got[0][1].items():
        assert torch.equal(t, got[1][1][n]), n
        assert not (t == 7.0).all(), n


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,D", [
    (2, 1, 40, 4, 2, 24),       # single tokens: one wave's tile
    (2, 3, 3000, 4, 1, 64),     # their splits
    (2, 1, 900, 2, 2, 128),
    (2, 70, 50, 2, 2, 40),      # 128-row blocks
    (2, 40, 1500, 2, 1, 24),    # their splits
    (40, 260, 130, 16, 16, 72),  # 256-row blocks of wide bf16 heads
    (2, 260, 1500, 1, 1, 128),  # their splits
])
def test_no_keys_and_a_query_that_is_not_finite(B, Nq, Nk, H, Hk, D, dt):
    """A mask that leaves nothing and kv_len 0 say the same: o = 0 and dq = 0 whatever q and dout hold, and the other
    sequences are as they are beside finite ones."""
    g = _gen(41)
    q, k, v, do = (torch.randn(B, n, h, D, generator=g).to(dt).cuda() for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
    mask = torch.rand(B, Nk, generator=g).cuda() < 0.7
    mask[-1] = False
    bad = torch.tensor([float("nan"), float("inf"), float("-inf")], device="cuda").to(dt)
    ln = torch.full((B,), Nk, dtype=torch.int32, device="cuda")
    ln[-1] = 0
    res = []
    for fill, kw in ((None, dict(mask=mask)), (bad, dict(mask=mask)), (bad, dict(kv_len=ln, mask=mask | (ln == 0)[:, None]))):
        ql, gl = q.clone(), do.clone()
        if fill is not None:
            ql[-1] = fill[torch.arange(D, device="cuda") % 3]
            gl[-1] = fill[0]
        leaves = [t.clone().requires_grad_(True) for t in (ql, k, v)]
        o = X().cross_attention(*leaves, **kw)
        with torch.no_grad():
            assert torch.equal(X().cross_attention(*leaves, **kw), o)
        res.append((o.detach(), *torch.autograd.grad(o, leaves, gl)))
        for n, t in zip(("o", "dq", "dk", "dv"), res[-1]):
            assert (t[-1] == 0).all(), n
            assert torch.isfinite(t).all() and (t[0] != 0).any(), n
    for n, a, b, c in zip(("o", "dq", "dk", "dv"), *res):
        assert torch.equal(a, b) and torch.equal(a, c), n


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,D", [(2, 3, 40, 4, 2, 24), (2, 6, 3000, 4, 1, 64), (2, 200, 50, 2, 2, 128), (2, 90, 1500, 1, 1, 48)])
def test_rows_past_q_len_beside_a_key_that_is_not_finite(B, Nq, Nk, H, Hk, D, dt):
    """A key that is there and holds infinities makes its sequence's rows NaN, not those past q_len: o and dq are 0 there."""
    g = _gen(43)
    q, k, v, do = (torch.randn(B, n, h, D, generator=g).to(dt).cuda() for n, h in ((Nq, H), (Nk, Hk), (Nk, Hk), (Nq, H)))
    k[0, Nk // 2], v[0, Nk // 2] = float("inf"), float("nan")
    ln = torch.tensor([Nq // 2, Nq - 1], dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = X().cross_attention(*leaves, q_len=ln)
    dq, dk, dv = torch.autograd.grad(o, leaves, do)
    for t in (o, dq):
        assert (t[0, Nq // 2:] == 0).all() and (t[1, Nq - 1:] == 0).all()
        assert not torch.isfinite(t[0, :Nq // 2]).any() and torch.isfinite(t[1]).all() and (t[1, : Nq - 1] != 0).any()
    assert torch.isfinite(dk[1]).all() and torch.isfinite(dv[1]).all()


@pytest.mark.parametrize("Nq", [1, 40])
def test_cross_attention_on_the_longest_key_axis(Nq):
    """2^31 - 8192 keys, the most that is not refused: equal scores, v = 1 at the last 2^21 keys.  Every count is a
    whole number of 8192s below 2^31, exact in fp32, and the probabilities are powers of two: o is its own rounding
    (2^-8) and those of a reciprocal and a product in fp32."""
    Nk, last = (1 << 31) - 8192, 1 << 21
    q = torch.ones(1, Nq, 1, 1, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(1, 1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(1, Nk, 1, 1)
    v = torch.zeros(1, Nk, 1, 1, dtype=torch.bfloat16, device="cuda")
    v[:, Nk - last:] = 1
    with torch.no_grad():
        o = X().cross_attention(q, k, v)
    want = torch.full((1, Nq, 1, 1), last / Nk, dtype=torch.float64)
    _near(o, want, (U16 + 4 * U32) * want, "o")


@pytest.mark.parametrize("mdt", [torch.bool, torch.uint8, torch.float32], ids=str)
@pytest.mark.parametrize("mB", [1, 3])
def test_an_empty_mask_of_an_encoder_without_states(mB, mdt):
    q = torch.randn(3, 5, 2, 24, device="cuda", requires_grad=True)
    k, v = (torch.randn(3, 0, 1, 24, device="cuda", requires_grad=True) for _ in range(2))
    mask, ln = torch.zeros(mB, 0, dtype=mdt, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    for kw in (dict(mask=mask), dict(mask=mask, kv_len=ln)):
        o = X().cross_attention(q, k, v, **kw)
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
        assert (o == 0).all() and (dq == 0).all() and dk.shape == dv.shape == k.shape
    with pytest.raises(ValueError):
        X().cross_attention(q, k, v, mask=torch.zeros(2, 0, dtype=mdt, device="cuda"))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_all_that_attention_keeps_passes_the_saved_tensor_hooks(dt):
    """Moved to the host by the hooks, nothing of the forward stays allocated but its output, and the gradients are the same."""
    B, Nq, Nk, H, D = 2, 4096, 64, 8, 64
    g = _gen(47)
    q, k, v = (torch.randn(B, n, H, D, generator=g).to(dt).cuda().requires_grad_(True) for n in (Nq, Nk, Nk))
    do = torch.ones(B, Nq, H, D, dtype=dt, device="cuda")
    want = torch.autograd.grad(X().cross_attention(q, k, v), (q, k, v), do)
    # (bytes as they were asked for: what counts as allocated is whole cached blocks, up to 1 MiB larger where one is not
    # split; o took the 8651264 bytes of an earlier lse and residual, 262656 more than its own 8388608)
    asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]  # noqa: E731
    at = asked()
    with torch.autograd.graph.save_on_cpu():
        o = X().cross_attention(q, k, v)
    kept = asked() - at
    assert kept < o.numel() * o.element_size() + (1 << 18), kept  # (lse alone is B H Nq 4 bytes, o's residual as large as o)
    got = torch.autograd.grad(o, (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(o, (q, k, v), do)


@pytest.mark.parametrize("which", range(3), ids=["attention", "rope", "norms"])
def test_negated_views(which):
    """Views that hold their values negated (as z.conj().imag does), as inputs and as gradients."""
    f, ins = _small()[which]
    neg = lambda t: torch._neg_view(-t)  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in ins]
    out = f(*leaves)
    up = torch.randn_like(out)
    base = torch.autograd.grad(out, leaves, up)
    twins = [neg(t).requires_grad_(True) for t in ins]
    assert all(t.is_neg() and torch.equal(t, u) for t, u in zip(twins, ins))
    got = f(*twins)
    assert torch.equal(got, out)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, twins, neg(up)), base))


def test_negated_views_rotated_in_place():
    plan = X().RopeAxes([4, 4])
    q, pos = torch.randn(2, 5, 3, 16, device="cuda"), torch.arange(10, device="cuda", dtype=torch.int32).reshape(5, 2)
    want = X().rope_axes(plan, pos, q)
    twin = torch._neg_view(-q)
    assert torch.equal(X().rope_axes(plan, pos, twin, inplace=True), want) and torch.equal(twin, want)


# wide bf16 heads over 256 rows and more: key tiles of 64 through two and three buffers, 4 to 8 of them per block (a
# buffer is written again from the fourth on), alone and in splits, rows of grouped heads and rows past q_len
WIDE = [  # B, Nq, Nk, H, Hk, D, padding, layout
    (4, 130, 461, 128, 64, 72, "", "tokens"),           # one split, 8 tiles
    (4, 260, 449, 32, 32, 96, "mask len q", "heads"),
    (2, 520, 401, 64, 32, 128, "mask", "tokens"),
    (1, 100, 1500, 4, 1, 128, "", "heads"),             # 6 splits of 4 tiles
    (1, 65, 1777, 8, 1, 80, "mask bool q", "tokens"),
    (2, 150, 3000, 16, 8, 96, "mask len", "tokens"),    # 8 splits of 6 tiles
]


@pytest.mark.parametrize("case", WIDE, ids=lambda c: "-".join(str(x) for x in c))
def test_cross_attention_wide_heads(case):
    test_cross_attention_forward_backward(case, torch.bfloat16)


@pytest.mark.parametrize("D", [72, 128])
def test_cross_attention_wide_heads_ragged_splits(D):
    """Lengths of 0, 1, one tile and all keys where every sequence's keys are shared out over splits."""
    B, Nq, Nk, Hk, G, dt = 4, 75, 2100, 1, 4, torch.bfloat16
    q, k, v, do, *_ = _attn_inputs(B, Nq, Nk, Hk * G, Hk, D, dt, "", 21)
    ln = torch.tensor([Nk, 0, 1, 64], dtype=torch.int32)
    keep = torch.arange(Nk)[None] < ln[:, None]
    k[~keep], v[~keep] = float("nan"), float("inf")
    want, tol = _attn_oracle(q, k, v, do, keep, torch.ones(B, Nq, dtype=torch.bool), D ** -0.5, dt)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = X().cross_attention(*leaves, kv_len=ln.cuda())
    for n, got, w, t in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, do.cuda())), want, tol):
        _near(got, w, t, n)


@pytest.mark.parametrize("B,H,Nk", [(1, 1, 2000), (64, 2, 461)])
def test_cross_attention_wide_heads_maximum_raised_late(B, H, Nk):
    """Scores that rise over the tiles for one row and fall for its neighbour, by 8 and more in log2 per tile or less."""
    Nq, D, dt = 300, 128, torch.bfloat16
    q, k = torch.zeros(B, Nq, H, D), torch.zeros(B, Nk, H, D)
    r = torch.arange(Nq)
    q[..., 0] = (torch.where(r % 2 == 0, 1.0, -1.0) * 2.0 ** -(r % 5).float())[None, :, None]
    k[..., 0] = torch.linspace(-256, 256, Nk).round()[None, :, None]  # (whole numbers, exact in bf16)
    v = torch.randn(B, Nk, H, D, generator=_gen(6))
    args = [t.to(dt) for t in (q, k, v)]
    want, tol = _attn_oracle(*args, args[0], torch.ones(B, Nk, dtype=torch.bool), torch.ones(B, Nq, dtype=torch.bool), 1.0, dt)
    # exponents up to 512 * log2 e < 2^10: the argument of exp2 is rounded by 2^-14, in the sum and in its normaliser
    _near(X().cross_attention(*(t.cuda() for t in args), scale=1.0), want[0], tol[0] + 2.0 ** -13 * v.abs().max().item(), "o")


def test_cross_attention_gradients_that_arrive_expanded_or_in_another_order():
    """An expanded gradient (of a sum) and one whose head dim is not contiguous: the bits of their contiguous copies."""
    for B, Nq, Nk, H, Hk, D in ((3, 37, 50, 2, 1, 24), (2, 5, 70, 2, 2, 64)):
        q, k, v, do, *_ = _attn_inputs(B, Nq, Nk, H, Hk, D, torch.float32, "", 3)
        leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
        grads = lambda up: torch.autograd.grad(X().cross_attention(*leaves), leaves, up)  # noqa: E731
        one = torch.ones(1, device="cuda")
        flipped = do.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0).cuda()
        assert flipped.stride(-1) != 1 and one.expand(B, Nq, H, D).stride(-1) == 0
        for up in (one.expand(B, Nq, H, D), flipped, flipped[:1].expand(B, -1, -1, -1)):
            assert all(torch.equal(a, b) and (a != 0).any() for a, b in zip(grads(up), grads(up.contiguous())))


# the norms' other widths per thread and team: one, four and eight columns, odd numbers of rows (two share a wide block)
GRN_WIDTHS = [  # G, rows, C, post, pre, gate/mod/affine, type of h
    (1, 3, 257, "rms", "layer", "gate mod affine", "same"),
    (1, 5, 1001, "layer", "rms", "gate mod affine", "f32"),
    (3, 1, 1537, "layer", "layer", "gate mod affine", "f32"),
    (1, 7, 1999, "rms", "rms", "gate mod", "same"),
    (3, 3, 400, "rms", "layer", "gate mod affine", "same"),
    (1, 5, 600, "layer", "layer", "gate mod affine", "same"),
    (1, 3, 700, "layer", "rms", "gate mod affine", "f32"),
    (3, 1, 1200, "rms", "rms", "gate mod affine", "same"),
    (1, 7, 1800, "layer", "layer", "gate mod affine", "same"),
    (1, 7, 2000, "layer", "layer", "gate mod affine", "f32"),
    (1, 5, 2500, "rms", "layer", "gate mod affine", "same"),
    (3, 5, 5000, "rms", "layer", "gate mod affine", "same"),
    (1, 5, 6000, "layer", "rms", "gate affine", "f32"),
    (1, 3, 7000, "none", "layer", "gate mod affine", "same"),
]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("case", GRN_WIDTHS, ids=lambda c: "-".join(str(x) for x in c))
def test_gate_residual_norm_widths(case, dt):
    test_gate_residual_norm_forward_backward(case, dt)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,Nk,H,D", [(1, 1, 40, 2, 16), (1, 2, 3000, 1, 128), (1, 100, 50, 2, 24), (1, 40, 1500, 1, 64), (64, 260, 70, 2, 128)])
def test_scores_past_fp32_are_not_a_row_without_keys(B, Nq, Nk, H, D, dt):
    """q . k = 2^74 D is finite, scaled by 2^56 it is not (2^134 and more): NaN as in a plain softmax, where 0 would hide it.
    Rows beside them are as they were."""
    scale = 2.0 ** 56
    q = torch.full((B, Nq, H, D), 2.0 ** 37, dtype=dt, device="cuda")
    q[:, 0] = 0
    k = torch.full((B, Nk, H, D), 2.0 ** 37, dtype=dt, device="cuda")
    v = torch.ones(B, Nk, H, D, dtype=dt, device="cuda")
    o = X().cross_attention(q, k, v, scale=scale)
    assert torch.isnan(o[:, 1:]).all() and (o[:, 0] == 1).all()
