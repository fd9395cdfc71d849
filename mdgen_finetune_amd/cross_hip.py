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
workspaces through torch's caching allocator (so they may be captured into a HIP graph; a backward pass
only while no eager graph of the same leaves is alive, whose accumulation torch ties to its own stream), and
are differentiable, once, where an input requires grad; forward-mode tangents and tracing (torch.jit.trace,
make_fx, fake tensors) raise RuntimeError.  Wrong types and shapes raise TypeError / ValueError
before any launch; a missing library or a CPU tensor raises RuntimeError (there is no other path).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib

_PAIRS = {"half": _lib.MDG_ROPE_HALF, "interleaved": _lib.MDG_ROPE_INTERLEAVED, "axis": _lib.MDG_ROPE_AXIS}
_ENTRIES = ("mdg_attn_cross_workspace_bytes", "mdg_attn_cross_fwd", "mdg_attn_cross_bwd", "mdg_rope_axes", "mdg_gate_res_norm",
            "mdg_gate_res_norm_bwd_workspace_bytes", "mdg_gate_res_norm_bwd", "mdg_last_error_string")
_C = None


def _ext():
    """The host side (csrc/cross_torch.cpp), bound to the library's entry points once."""
    global _C
    if _C is None:
        lib = _lib.load()
        try:
            from . import _cross
        except ImportError as e:
            raise RuntimeError("mdgen_finetune_amd/_cross.so is missing or does not load: build it with `make -C "
                               "mdgen_finetune_amd/csrc` (there is no other path)") from e
        _cross.bind([ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _ENTRIES])
        _C = _cross
    return _C


def cross_attention(q, k, v, mask=None, q_len=None, kv_len=None, scale=None):
    """softmax(scale q k^T) v over the keys that are there: q [B, Nq, H, D], k / v [B, Nk, Hk, D] with
    H % Hk == 0 (query head h reads key head h // (H / Hk)) and D <= 128; returns [B, Nq, H, D].

    mask [B, Nk] or [1, Nk] (bool, uint8 or fp32; nonzero: the key is there), kv_len / q_len int32 [B]:
    the sequences' own lengths.  What k and v hold at keys that are not there is without effect (NaN
    too) and has gradient 0; a row without keys gives 0, and so do query rows past q_len.  scale
    defaults to D ** -0.5.  Accumulation and the softmax are fp32; with bf16 inputs the probabilities
    are rounded to bf16 before their product with v."""
    return (_C or _ext()).cross_attention(q, k, v, mask, q_len, kv_len, scale)


class RopeAxes:
    """The rotary plan of a head: sections[a] pairs of columns turn by a token's position on axis a, pair i
    of an axis with n pairs at frequency base ** (-i / n) (or freq: one frequency per pair, all sections in
    order, constants).  pairs: "half" couples column p with p + sum(sections), "interleaved" 2p with 2p + 1, "axis"
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
        if freq.requires_grad:
            raise ValueError("RopeAxes: frequencies are constants of the plan and get no gradient, detach them first")
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
        self.sections, self.pairs, self.npairs = tuple(sections), pairs, n
        axis = [a for a, s in enumerate(sections) for _ in range(s)]
        # one copy to the device: the frequencies in turns (fp64), then three int32 tables
        tables = torch.cat([(freq / (2.0 * math.pi)).view(torch.int32), torch.tensor(axis + first + second, dtype=torch.int32)])
        tables = tables.to(torch.device("cuda" if device is None else device))
        self.turns, self.axis, self.cols = tables[: 2 * n].view(torch.float64), tables[2 * n : 3 * n], tables[3 * n :]
        self._plan = None

    def __setattr__(self, name, value):
        # (the extension's handle holds the tables, and the kernels trust their columns)
        if name in self.__dict__ and name in ("sections", "pairs", "npairs", "turns", "axis", "cols"):
            raise AttributeError(f"RopeAxes: {name} of a plan is fixed, make another plan")
        super().__setattr__(name, value)

    def __getstate__(self):
        return {**self.__dict__, "_plan": None}  # (the extension's handle is made anew where it is needed)


def rope_axes(plan, pos, q, k=None, inverse=False, inplace=False):
    """q (and k, in the same launch) [B, N, heads, D] rotated by their tokens' positions: pos [N, axes],
    [1, N, axes] or [B, N, axes], int32 or int64.  Returns q or (q, k).  inverse: by the negative angle.
    inplace: writes into q and k (no gradient through the call then)."""
    ext = _C or _ext()
    handle = plan._plan
    if handle is None:
        handle = plan._plan = ext.RopePlan(plan.turns, plan.axis, plan.cols, plan.sections, _PAIRS[plan.pairs])
    return ext.rope_axes(handle, pos, q, k, inverse, inplace)


def gate_residual_norm(h, y=None, gate=None, shift=None, scale=None, resid_scale=1.0, post="none", pre="layer",
                       post_w=None, post_b=None, pre_w=None, pre_b=None, eps=1e-6):
    """(h_out, xn) with h_out = resid_scale h + gate u, u = post(y) post_w + post_b, and
    xn = (pre(h_out) pre_w + pre_b) (1 + scale) + shift: the branch's own norm, its gated way back into the
    residual stream and the next block's input in one pass.

    h [..., C] fp32 or y's type; y [..., C] fp32 or bf16 (None: only the norm before a block; xn then has
    h's type); post / pre "none", "rms" or "layer" (pre "none": xn is None).  gate / shift / scale fp32
    [G, C], one row per run of rows (the rows' count is a multiple of G; the backward slows down for runs shorter than
    32 rows); weights fp32 [C].  C <= 8192.
    Statistics and sums are fp32; xn is formed from h_out before its rounding."""
    return (_C or _ext()).gate_residual_norm(h, y, gate, shift, scale, resid_scale, post, pre, post_w, post_b, pre_w, pre_b, eps)
