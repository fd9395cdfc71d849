"""A conditioned block's operators on libmdgen_hip.so, forward and backward: cross attention to an
encoder's states, rotary positions on several axes, and the norms around a block with its gate and
residual scale.

    q, k = rope_axes(plan, pos, q, k)                      # plan = RopeAxes((pairs per axis, ...))
    o = cross_attention(q, k, v, mask=mask)                # [B, Nq, H, D] over [B, Nk, Hk, D]
    h, xn = gate_residual_norm(h, y, gate=gate, post="rms", pre="layer", shift=shift, scale=scale)

The reference's MultiheadAttention takes key and value inputs of their own (mha.py:161-264), rotates
by one axis (mha.py:356-357) and its block keeps LayerNorm -> branch -> gated residual
(latent_model.py:456-493).  Here the key side has its own length, heads and mask, a token has a
position on each of several axes (frame, residue, ...), and the branch is normalised on both sides.

Tensors are fp32 or bf16 on a ROCm device, any strides with a contiguous last dim (other orders are
copied).  Calls run on the current stream of the tensors' device, allocate only outputs and
workspaces through torch's caching allocator (so they may be captured into a HIP graph), and are
differentiable where an input requires grad.  Wrong types and shapes raise TypeError / ValueError
before any launch; a missing library or a CPU tensor raises RuntimeError (there is no other path).
"""
from __future__ import annotations

import functools
import math
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.MDG_F32, torch.bfloat16: _lib.MDG_BF16}
_NORMS = {"none": _lib.MDG_NORM_NONE, "rms": _lib.MDG_NORM_RMS, "layer": _lib.MDG_NORM_LAYER}
_PAIRS = {"half": _lib.MDG_ROPE_HALF, "interleaved": _lib.MDG_ROPE_INTERLEAVED, "axis": _lib.MDG_ROPE_AXIS}
_MASKS = {torch.bool: _lib.MDG_MASK_U8, torch.uint8: _lib.MDG_MASK_U8, torch.float32: _lib.MDG_MASK_F32}

# The descriptors' images (include/mdgen_hip.h), packed by one call each: filling the ctypes mirrors
# field by field costs several times a small launch.
_CROSS = struct.Struct("<8if4x42q")
_ROPE = struct.Struct("<20i22q")
_GRN = struct.Struct("<7i2f4x26q")
_NO_HEADS = (0, 0, 0, 0)


def _check_device(t, *others):
    dev = t.device
    if dev.type != "cuda":
        raise RuntimeError("mdgen_finetune_amd.cross_hip runs on a ROCm device; got a tensor on " + str(dev))
    for o in others:
        if o is not None and o.device != dev:
            raise ValueError(f"tensors on {dev} and {o.device}")


def _stream(dev):
    """(the device index to go back to, or -1; the current stream of the tensors' device, which is current now)."""
    idx, cur = dev.index, torch._C._cuda_getDevice()
    if cur == idx:
        return -1, torch._C._cuda_getCurrentRawStream(idx)
    torch._C._cuda_setDevice(idx)
    return cur, torch._C._cuda_getCurrentRawStream(idx)


def _done(back, rc, what):
    if back >= 0:
        torch._C._cuda_setDevice(back)
    if rc != 0:
        _lib.check(rc, what)


def _launch(fn, what, dev, *args):
    """One library call on the current stream of dev (made current for it where it is not)."""
    back, stream = _stream(dev)
    _done(back, fn(*args, stream), what)


def _twice(backward):
    """Autograd formula of a Function whose backward has no derivative of its own: once_differentiable's
    wrapping only where a caller asks for a graph of the backward (create_graph)."""
    once = once_differentiable(backward)

    def call(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return staticmethod(call)


def _unit(t):
    """The tensor with its last dim contiguous (a copy only where it is not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _heads(t):
    s = t.stride()
    return t.data_ptr(), s[0], s[1], s[2]


def _ws(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


_LIB = None


def _library():
    global _LIB
    if _LIB is None:
        _LIB = _lib.load()
    return _LIB


# ------------------------------------------------------------------------------------------
# cross attention

@functools.lru_cache(maxsize=512)
def _cross_ws_bytes(dtype, B, Nq, Nk, H, Hk, D, backward):
    n = _library().mdg_attn_cross_workspace_bytes(_CROSS.pack(dtype, B, Nq, Nk, H, Hk, D, 0, 1.0, *([0] * 42)), backward)
    if n == _lib.SIZE_MAX:
        _lib.check(1, "mdg_attn_cross_workspace_bytes")
    return n


def _cross_desc(q, k, v, o, side, mask, q_len, kv_len, scale, grads=_NO_HEADS * 4):
    """side: (o_lo address or 0, lse address or 0); both contiguous as o [B, Nq, H, D] and [B, H, Nq]."""
    B, Nq, H, D = q.shape
    o_lo, lse = side
    return _CROSS.pack(_DTYPES[q.dtype], B, Nq, k.shape[1], H, k.shape[2], D, 0 if mask is None else _MASKS[mask.dtype], scale,
                       *_heads(q), *_heads(k), *_heads(v), *_heads(o), o_lo, Nq * H * D, H * D, D, *grads,
                       0 if q_len is None else q_len.data_ptr(), 0 if kv_len is None else kv_len.data_ptr(),
                       *((0, 0, 0) if mask is None else (mask.data_ptr(), *mask.stride())), lse)


def _cross_fwd(q, k, v, o, side, mask, q_len, kv_len, scale):
    B, Nq, H, D = q.shape
    nbytes = _cross_ws_bytes(_DTYPES[q.dtype], B, Nq, k.shape[1], H, k.shape[2], D, 0)
    ws = _ws(nbytes, q.device)
    _launch(_library().mdg_attn_cross_fwd, "mdg_attn_cross_fwd", q.device,
            _cross_desc(q, k, v, o, side, mask, q_len, kv_len, scale), _lib.ptr(ws), nbytes)


class _CrossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, q_len, kv_len, scale):
        q, k, v = _unit(q), _unit(k), _unit(v)
        n, dev = q.numel(), q.device
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
        # what the backward reads beside o, one allocation: lse [B, H, Nq] fp32, then bf16's o_lo as o
        low = q.dtype == torch.bfloat16
        rows = (n // q.shape[3] + 3) // 4 * 16  # bytes of lse, o_lo aligned behind it
        side = torch.empty(rows + (2 * n if low else 0), dtype=torch.uint8, device=dev)
        if n:
            at = side.data_ptr()
            _cross_fwd(q, k, v, o, (at + rows if low else 0, at), mask, q_len, kv_len, scale)
        ctx.save_for_backward(q, k, v, o, mask, q_len, kv_len)
        ctx.rest = side, rows if low else -1, scale
        return o

    @_twice
    def backward(ctx, dout):
        q, k, v, o, mask, q_len, kv_len = ctx.saved_tensors
        q, k, v, o = _unit(q), _unit(k), _unit(v), _unit(o)
        side, low, scale = ctx.rest
        need = ctx.needs_input_grad
        dev = q.device
        dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
        dk = dv = None
        if need[1] or need[2]:  # (a frozen encoder leaves the key side's pass out)
            dk = torch.empty(k.shape, dtype=k.dtype, device=dev)
            dv = torch.empty(v.shape, dtype=v.dtype, device=dev)
        if q.numel():
            dout = _unit(dout)
            B, Nq, H, D = q.shape
            nbytes = _cross_ws_bytes(_DTYPES[q.dtype], B, Nq, k.shape[1], H, k.shape[2], D, 1)
            ws = _ws(nbytes, dev)
            keys = _NO_HEADS * 2 if dk is None else (*_heads(dk), *_heads(dv))
            at = side.data_ptr()
            desc = _cross_desc(q, k, v, o, (at + low if low >= 0 else 0, at), mask, q_len, kv_len, scale,
                               (*_heads(dout), *_heads(dq), *keys))
            _launch(_library().mdg_attn_cross_bwd, "mdg_attn_cross_bwd", dev, desc, _lib.ptr(ws), nbytes)
        elif dk is not None:
            dk.zero_(), dv.zero_()
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def _check_len(name, t, B):
    if t.dtype != torch.int32 or tuple(t.shape) != (B,) or not t.is_contiguous():
        raise ValueError(f"cross_attention: {name} must be a contiguous int32 [{B}], got {t.dtype} {tuple(t.shape)}")


def cross_attention(q, k, v, mask=None, q_len=None, kv_len=None, scale=None):
    """softmax(scale q k^T) v over the keys that are there: q [B, Nq, H, D], k / v [B, Nk, Hk, D] with
    H % Hk == 0 (query head h reads key head h // (H / Hk)) and D <= 128; returns [B, Nq, H, D].

    mask [B, Nk] or [1, Nk] (bool, uint8 or fp32; nonzero: the key is there), kv_len / q_len int32 [B]:
    the sequences' own lengths.  What k and v hold at keys that are not there is without effect (NaN
    too) and has gradient 0; a row without keys gives 0, and so do query rows past q_len.  scale
    defaults to D ** -0.5.  Accumulation and the softmax are fp32; with bf16 inputs the probabilities
    are rounded to bf16 before their product with v."""
    if not q.dim() == k.dim() == v.dim() == 4:
        raise ValueError(f"cross_attention: q, k, v must be [B, N, heads, D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"cross_attention: q, k, v must be fp32 or bf16 of one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    B, Nq, H, D = q.shape
    kB, Nk, Hk, kD = k.shape
    if k.shape != v.shape or kB != B or kD != D or Hk == 0 or H % Hk or not 1 <= D <= 128:
        raise ValueError(f"cross_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}")
    _check_device(q, k, v, mask, q_len, kv_len)
    if mask is not None:
        if mask.dtype not in _MASKS or mask.dim() != 2 or mask.shape[1] != Nk or mask.shape[0] not in (1, B):
            raise ValueError(f"cross_attention: mask must be bool, uint8 or fp32 [{B} or 1, {Nk}], got {mask.dtype} "
                             f"{tuple(mask.shape)}")
        if mask.shape[0] != B:
            mask = mask.expand(B, Nk)
    if q_len is not None:
        _check_len("q_len", q_len, B)
    if kv_len is not None:
        _check_len("kv_len", kv_len, B)
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-18 <= scale <= 1e18:
        raise ValueError(f"cross_attention: scale {scale}")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossFn.apply(q, k, v, mask, q_len, kv_len, scale)
    q, k, v = _unit(q), _unit(k), _unit(v)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if o.numel():
        _cross_fwd(q, k, v, o, (0, 0), mask, q_len, kv_len, scale)
    return o


# ------------------------------------------------------------------------------------------
# rotary positions with several axes

class RopeAxes:
    """The rotary plan of a head: sections[a] pairs of columns turn by a token's position on axis a, pair i
    of an axis with n pairs at frequency base ** (-i / n) (or freq: one frequency per pair, all sections in
    order).  pairs: "half" couples column p with p + sum(sections), "interleaved" 2p with 2p + 1, "axis"
    halves within each axis's own section.  Columns past 2 * sum(sections) pass through."""

    def __init__(self, sections, base=10000.0, pairs="half", freq=None, device=None):
        sections = [int(s) for s in sections]
        if not 1 <= len(sections) <= _lib.MDG_ROPE_MAX_AXES or min(sections) < 0 or sum(sections) < 1:
            raise ValueError(f"RopeAxes: sections {sections}")
        if pairs not in _PAIRS:
            raise ValueError(f"RopeAxes: pairs {pairs!r} (one of {sorted(_PAIRS)})")
        n = sum(sections)
        if freq is None:
            freq = [float(base) ** (-i / s) for s in sections for i in range(s)]
        freq = torch.as_tensor(freq, dtype=torch.float64).cpu()
        if tuple(freq.shape) != (n,):
            raise ValueError(f"RopeAxes: {n} pairs but freq {tuple(freq.shape)}")
        first, second, at = [], [], 0
        for s in sections:
            first += [at + i for i in range(s)]
            second += [at + s + i for i in range(s)]
            at += 2 * s
        if pairs == "half":
            first, second = list(range(n)), list(range(n, 2 * n))
        elif pairs == "interleaved":
            first, second = list(range(0, 2 * n, 2)), list(range(1, 2 * n, 2))
        self.sections, self.pairs, self.npairs = sections, pairs, n
        device = torch.device("cuda" if device is None else device)
        self.turns = (freq / (2.0 * math.pi)).to(device)
        self.axis = torch.tensor([a for a, s in enumerate(sections) for _ in range(s)], dtype=torch.int32).to(device)
        self.cols = torch.tensor(first + second, dtype=torch.int32).to(device)
        self._code = _PAIRS[pairs]
        self._sections8 = tuple(sections + [0] * (_lib.MDG_ROPE_MAX_AXES - len(sections)))


def _rope_call(plan, pos, xs, outs, inverse):
    q, o = xs[0], outs[0]
    B, N, H, D = q.shape
    if len(xs) == 2:
        H2, k2, o2 = xs[1].shape[2], _heads(xs[1]), _heads(outs[1])
    else:
        H2, k2, o2 = 0, _NO_HEADS, _NO_HEADS
    ps = pos.stride()
    desc = _ROPE.pack(_DTYPES[q.dtype], plan._code, len(xs), B, N, D, plan.npairs, len(plan.sections), pos.dtype == torch.int64,
                      inverse, H, H2, *plan._sections8, pos.data_ptr(), 0 if pos.shape[0] == 1 else ps[0], ps[1],
                      plan.turns.data_ptr(), plan.axis.data_ptr(), plan.cols.data_ptr(), *_heads(q), *k2, *_heads(o), *o2)
    _launch(_library().mdg_rope_axes, "mdg_rope_axes", q.device, desc)


def _rope_new(plan, pos, xs, inverse):
    xs = [_unit(t) for t in xs]
    outs = [torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in xs]
    if xs[0].shape[0] and xs[0].shape[1]:
        _rope_call(plan, pos, xs, outs, inverse)
    return outs


class _RopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, plan, pos, inverse, *xs):
        ctx.plan, ctx.inverse = plan, inverse
        ctx.save_for_backward(pos)
        return tuple(_rope_new(plan, pos, xs, inverse))

    @_twice
    def backward(ctx, *gs):  # the rotation's transpose is the rotation by the negative angle
        (pos,) = ctx.saved_tensors
        return (None, None, None, *_rope_new(ctx.plan, pos, gs, 1 - ctx.inverse))


def rope_axes(plan, pos, q, k=None, inverse=False, inplace=False):
    """q (and k, in the same launch) [B, N, heads, D] rotated by their tokens' positions: pos [N, axes],
    [1, N, axes] or [B, N, axes], int32 or int64.  Returns q or (q, k).  inverse: by the negative angle.
    inplace: writes into q and k (no gradient through the call then)."""
    xs = (q,) if k is None else (q, k)
    for t in xs:
        if t.dim() != 4 or t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise TypeError(f"rope_axes: tensors must be fp32 or bf16 [B, N, heads, D] of one type, got {t.dtype} "
                            f"{tuple(t.shape)}")
        s = t.shape
        if s[0] != q.shape[0] or s[1] != q.shape[1] or s[3] != q.shape[3] or not 1 <= s[2] <= 1024:
            raise ValueError(f"rope_axes: q {tuple(q.shape)}, k {tuple(s)}")
    B, N, _, D = q.shape
    if 2 * plan.npairs > D or D > 1024:
        raise ValueError(f"rope_axes: {plan.npairs} pairs in a head of {D}")
    _check_device(q, k, pos, plan.turns)
    if pos.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"rope_axes: pos must be int32 or int64, got {pos.dtype}")
    if pos.dim() == 2:
        pos = pos[None]
    if pos.dim() != 3 or pos.shape[0] not in (1, B) or pos.shape[1] != N or pos.shape[2] != len(plan.sections):
        raise ValueError(f"rope_axes: pos {tuple(pos.shape)} for tokens [{B}, {N}] on {len(plan.sections)} axes")
    pos = _unit(pos)
    inverse = int(bool(inverse))
    grad = torch.is_grad_enabled() and any(t.requires_grad for t in xs)
    if inplace:
        if grad:
            raise ValueError("rope_axes: inplace on a tensor that requires grad")
        for t in xs:
            if (t.stride(-1) != 1 and D > 1) or any(t.stride(i) == 0 and t.shape[i] > 1 for i in range(3)):
                raise ValueError("rope_axes: inplace needs a contiguous head dim and no shared memory between tokens or heads")
        if B and N:
            _rope_call(plan, pos, xs, xs, inverse)
        outs = xs
    else:
        outs = _RopeFn.apply(plan, pos, inverse, *xs) if grad else _rope_new(plan, pos, xs, inverse)
    return outs[0] if k is None else tuple(outs)


# ------------------------------------------------------------------------------------------
# the norms around a block, its gate and residual scale

def _rows2d(t, C):
    """(t as rows [M, C] with a contiguous last dim, their stride)."""
    if t.is_contiguous():
        return t, C
    t = t.reshape(-1, C)
    if (t.stride(1) == 1 or C == 1) and (t.stride(0) >= C or t.shape[0] == 1):
        return t, (t.stride(0) if t.shape[0] > 1 else C)
    return t.contiguous(), C


def _same_rows(gate, shift, scale):
    """gate / shift / scale with one common row stride (copied where they differ), and that stride."""
    some = gate if gate is not None else shift if shift is not None else scale
    if some is None:
        return gate, shift, scale, 0
    st, C = some.stride(), some.shape[1]
    if (st[1] == 1 or C == 1) and st[0] >= C and (shift is None or shift.stride() == st) and (
            scale is None or scale.stride() == st):
        return gate, shift, scale, st[0]
    return (*(None if t is None else t.contiguous() for t in (gate, shift, scale)), C)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _grn_ins(cfg, h, y, gate, shift, scale, post_w, post_b, pre_w, pre_b):
    """The inputs' part of the descriptor, and the tensors that it points into.  cfg: (dtype code of y, of h,
    rows per group, post, pre, resid_scale, eps, type of xn)."""
    C = h.shape[-1]
    h, ldh = _rows2d(h, C)
    y, ldy = (None, 0) if y is None else _rows2d(y, C)
    gate, shift, scale, ms = _same_rows(gate, shift, scale)
    return (cfg[0], cfg[1], h.numel() // C, C, *cfg[2:7], h.data_ptr(), _ptr(y), ldh, ldy, _ptr(gate), _ptr(shift), _ptr(scale),
            ms, _ptr(post_w), _ptr(post_b), _ptr(pre_w), _ptr(pre_b)), (h, y, gate, shift, scale, post_w, post_b, pre_w, pre_b)


def _grn_fwd(cfg, h, y, *par):
    head, ins = _grn_ins(cfg, h, y, *par)
    ho = None if y is None and cfg[5] == 1.0 and cfg[4] else torch.empty(h.shape, dtype=h.dtype, device=h.device)
    xn = torch.empty(h.shape, dtype=cfg[7], device=h.device) if cfg[4] else None
    if h.numel():
        desc = _GRN.pack(*head, _ptr(ho), _ptr(xn), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        _launch(_library().mdg_gate_res_norm, "mdg_gate_res_norm", h.device, desc)
    return ins, ho, xn


class _GrnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, h, y, *par):
        ins, ho, xn = _grn_fwd(cfg, h, y, *par)
        ctx.save_for_backward(*ins)
        ctx.cfg, ctx.shape = cfg, h.shape
        ctx.set_materialize_grads(False)
        return (h.view_as(h) if ho is None else ho), xn  # (without y, h itself goes on)

    @_twice
    def backward(ctx, dho, dxn):
        need = ctx.needs_input_grad[1:]
        if dho is None and dxn is None:
            return (None,) * 10
        head, saved = _grn_ins(ctx.cfg, *ctx.saved_tensors)
        h, y, gate, shift, scale, *ws = saved
        C, dev = h.shape[-1], h.device
        dho = None if dho is None else dho.contiguous()
        dxn = None if dxn is None else dxn.contiguous()
        dh = torch.empty(ctx.shape, dtype=h.dtype, device=dev) if need[0] else None
        dy = torch.empty(ctx.shape, dtype=y.dtype, device=dev) if need[1] else None
        ins = (gate, shift, scale, *ws)
        pre = (False, True, True, False, False, True, True)  # the pre norm's parameters: none without dxn
        live = [need[2 + i] and not (pre[i] and dxn is None) and h.numel() > 0 for i in range(7)]
        par = [None if live[i] or not need[2 + i] else torch.zeros(ins[i].shape, device=dev) for i in range(7)]
        for part in (range(3), range(3, 7)):  # the rows' gradients in one allocation, the weights' in another
            at = [i for i in part if live[i]]
            if at:
                for i, t in zip(at, torch.empty((len(at), *ins[at[0]].shape), device=dev).unbind(0)):
                    par[i] = t
        if h.numel():
            at = [par[i].data_ptr() if live[i] else 0 for i in range(7)]
            desc = _GRN.pack(*head, 0, 0, _ptr(dho), _ptr(dxn), _ptr(dh), _ptr(dy), *at[:3], C, *at[3:])
            lib = _library()
            nbytes = lib.mdg_gate_res_norm_bwd_workspace_bytes(desc)
            if nbytes == _lib.SIZE_MAX:
                _lib.check(1, "mdg_gate_res_norm_bwd_workspace_bytes")
            wsp = _ws(nbytes, dev)
            _launch(lib.mdg_gate_res_norm_bwd, "mdg_gate_res_norm_bwd", dev, desc, _lib.ptr(wsp), nbytes)
        return (None, dh, dy, *par)


def gate_residual_norm(h, y=None, gate=None, shift=None, scale=None, resid_scale=1.0, post="none", pre="layer",
                       post_w=None, post_b=None, pre_w=None, pre_b=None, eps=1e-6):
    """(h_out, xn) with h_out = resid_scale h + gate u, u = post(y) post_w + post_b, and
    xn = (pre(h_out) pre_w + pre_b) (1 + scale) + shift: the branch's own norm, its gated way back into the
    residual stream and the next block's input in one pass.

    h [..., C] fp32 or y's type; y [..., C] fp32 or bf16 (None: only the norm before a block; xn then has
    h's type); post / pre "none", "rms" or "layer" (pre "none": xn is None).  gate / shift / scale fp32
    [G, C], one row per run of rows (the rows' count is a multiple of G); weights fp32 [C].  C <= 8192.
    Statistics and sums are fp32; xn is formed from h_out before its rounding."""
    if h.dtype not in _DTYPES or h.dim() < 1:
        raise TypeError(f"gate_residual_norm: h must be fp32 or bf16 [..., C], got {h.dtype} {tuple(h.shape)}")
    C = h.shape[-1]
    if not 1 <= C <= 8192:
        raise ValueError(f"gate_residual_norm: C = {C}")
    if post not in _NORMS or pre not in _NORMS:
        raise ValueError(f"gate_residual_norm: post {post!r}, pre {pre!r} (one of {sorted(_NORMS)})")
    if y is None:
        if post != "none" or gate is not None:
            raise ValueError("gate_residual_norm: a post norm or gate without y")
        if pre == "none":
            raise ValueError("gate_residual_norm: nothing to do without y and a pre norm")
    elif y.shape != h.shape or y.dtype not in _DTYPES or h.dtype not in (torch.float32, y.dtype):
        raise TypeError(f"gate_residual_norm: h {h.dtype} {tuple(h.shape)}, y {y.dtype} {tuple(y.shape)}")
    if post == "none" and (post_w is not None or post_b is not None):
        raise ValueError("gate_residual_norm: post weights without a post norm")
    if pre == "none" and any(t is not None for t in (pre_w, pre_b, shift, scale)):
        raise ValueError("gate_residual_norm: pre weights or modulation without a pre norm")
    _check_device(h, y, gate, shift, scale, post_w, post_b, pre_w, pre_b)
    M, G = h.numel() // C, 0
    for t in (gate, shift, scale):
        if t is not None:
            if t.dtype != torch.float32 or t.dim() != 2 or t.shape[1] != C or (G and t.shape[0] != G):
                raise ValueError(f"gate_residual_norm: gate, shift and scale must be fp32 [G, {C}], got {t.dtype} "
                                 f"{tuple(t.shape)}")
            G = t.shape[0]
            if not G:
                raise ValueError("gate_residual_norm: gate, shift or scale without rows")
    G = G or 1
    if M % G or (M == 0 and G > 1 and h.shape[0] != G):
        raise ValueError(f"gate_residual_norm: {M} rows in {G} groups")
    for t in (post_w, post_b, pre_w, pre_b):
        if t is not None and (t.dtype != torch.float32 or t.dim() != 1 or t.shape[0] != C or not t.is_contiguous()):
            raise ValueError(f"gate_residual_norm: weights must be contiguous fp32 [{C}], got {t.dtype} {tuple(t.shape)}")
    eps, rs = float(eps), float(resid_scale)
    if not (0.0 <= eps < math.inf and math.isfinite(rs)):
        raise ValueError(f"gate_residual_norm: eps {eps}, resid_scale {rs}")
    ct = h.dtype if y is None else y.dtype
    cfg = (_DTYPES[ct], _DTYPES[h.dtype], M // G or 1, _NORMS[post], _NORMS[pre], rs, eps, ct)
    if torch.is_grad_enabled():
        for t in (h, y, gate, shift, scale, post_w, post_b, pre_w, pre_b):
            if t is not None and t.requires_grad:
                return _GrnFn.apply(cfg, h, y, gate, shift, scale, post_w, post_b, pre_w, pre_b)
    _, ho, xn = _grn_fwd(cfg, h, y, gate, shift, scale, post_w, post_b, pre_w, pre_b)
    return (h if ho is None else ho), xn
