"""The conditioned block's operators without a GPU: descriptor layouts, size queries, and every
refusal (before any launch) of the Python calls and of the C entry points."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from mdgen_finetune_amd import _lib
from mdgen_finetune_amd import cross_hip as X
from tests.conftest import REPO


def test_descriptor_layouts_match_header():
    prog = r"""
#include <stdio.h>
#include <stddef.h>
#include "mdgen_hip.h"
int main(void){
 printf("%zu %zu %zu %zu %zu %zu\n", sizeof(mdg_heads), sizeof(mdg_attn_cross), offsetof(mdg_attn_cross, q),
        offsetof(mdg_attn_cross, dv), offsetof(mdg_attn_cross, q_len), offsetof(mdg_attn_cross, lse));
 printf("%zu %zu %zu %zu %zu\n", sizeof(mdg_rope_axes_desc), offsetof(mdg_rope_axes_desc, section),
        offsetof(mdg_rope_axes_desc, pos), offsetof(mdg_rope_axes_desc, x), offsetof(mdg_rope_axes_desc, out));
 printf("%zu %zu %zu %zu %zu %zu\n", sizeof(mdg_gate_res_norm_desc), offsetof(mdg_gate_res_norm_desc, h),
        offsetof(mdg_gate_res_norm_desc, mod_stride), offsetof(mdg_gate_res_norm_desc, h_out),
        offsetof(mdg_gate_res_norm_desc, dmod_stride), offsetof(mdg_gate_res_norm_desc, dpre_b));
 return 0; }
"""
    with tempfile.TemporaryDirectory() as td:
        c = os.path.join(td, "t.c")
        open(c, "w").write(prog)
        subprocess.check_call(["gcc", "-I", os.path.join(REPO, "include"), c, "-o", os.path.join(td, "t")])
        got = [int(v) for v in subprocess.check_output([os.path.join(td, "t")]).split()]
    A, R, G = _lib.MdgAttnCross, _lib.MdgRopeAxes, _lib.MdgGateResNorm
    assert got == [ctypes.sizeof(_lib.MdgHeads), ctypes.sizeof(A), A.q.offset, A.dv.offset, A.q_len.offset, A.lse.offset,
                   ctypes.sizeof(R), R.section.offset, R.pos.offset, R.x.offset, R.out.offset,
                   ctypes.sizeof(G), G.h.offset, G.mod_stride.offset, G.h_out.offset, G.dmod_stride.offset, G.dpre_b.offset]


def _cross(**kw):
    a = _lib.MdgAttnCross(dtype=1, B=2, Nq=5, Nk=7, H=4, Hk=2, D=24, mask_type=0, scale=0.2)
    for n in ("q", "k", "v", "o"):
        setattr(a, n, _lib.MdgHeads(0x1000, 1000, 100, 24))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=2), b"dtype"), (dict(B=0), b"B=0"), (dict(Nq=0), b"Nq=0"), (dict(Nk=-1), b"Nk=-1"), (dict(H=5), b"H=5"),
    (dict(Hk=0), b"Hk=0"), (dict(D=0), b"D=0"), (dict(D=129), b"D=129"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("nan")), b"scale"), (dict(scale=-1.0), b"scale"), (dict(mask_type=3), b"mask_type"),
    (dict(mask_type=1), b"mask_type"), (dict(mask=0x1000), b"mask_type"), (dict(q=_lib.MdgHeads(None, 1, 1, 1)), b"null q"),
    (dict(k=_lib.MdgHeads(None, 1, 1, 1)), b"null k"), (dict(v=_lib.MdgHeads(0x1001, 1, 1, 1)), b"aligned"),
    (dict(q=_lib.MdgHeads(0x1000, -1, 1, 1)), b"strides"), (dict(B=1 << 20, Nq=1 << 20), b"grid"),
    (dict(B=1, Nq=(1 << 31) - 100), b"grid"), (dict(B=1, Nk=(1 << 31) - 100), b"grid"), (dict(B=1 << 23, Nq=1), b"grid"),
])
def test_cross_entry_refuses(kw, word):
    lib = _lib.load()
    a = _cross(**kw)
    assert lib.mdg_attn_cross_fwd(ctypes.byref(a), None, 0, None) != 0
    assert word in lib.mdg_last_error_string()


def test_cross_entry_refuses_backward_and_workspace():
    lib = _lib.load()
    assert lib.mdg_attn_cross_fwd(None, None, 0, None) != 0
    assert lib.mdg_attn_cross_bwd(ctypes.byref(_cross()), None, 0, None) != 0 and b"lse" in lib.mdg_last_error_string()
    hd = _lib.MdgHeads(0x1000, 1000, 100, 24)
    a = _cross(lse=0x1000, dout=hd, dq=hd, dk=hd)
    assert lib.mdg_attn_cross_bwd(ctypes.byref(a), None, 0, None) != 0 and b"together" in lib.mdg_last_error_string()
    a = _cross(lse=0x1000, dout=hd, dq=hd, dk=hd, dv=hd)
    need = lib.mdg_attn_cross_workspace_bytes(ctypes.byref(a), 1)
    assert 0 < need < 1 << 20
    assert lib.mdg_attn_cross_bwd(ctypes.byref(a), 0x1000, need - 1, None) != 0 and b"workspace" in lib.mdg_last_error_string()
    assert lib.mdg_attn_cross_bwd(ctypes.byref(a), 0x1004, need, None) != 0 and b"aligned" in lib.mdg_last_error_string()
    long = _cross(B=1, Nq=1, Nk=100000)  # a single token over a long cache splits its keys
    need = lib.mdg_attn_cross_workspace_bytes(ctypes.byref(long), 0)
    assert need > 0 and lib.mdg_attn_cross_fwd(ctypes.byref(long), None, 0, None) != 0
    bad = _cross(D=200)
    assert lib.mdg_attn_cross_workspace_bytes(ctypes.byref(bad), 0) == _lib.SIZE_MAX
    assert lib.mdg_attn_cross_workspace_bytes(ctypes.byref(_cross(Nk=0)), 1) < 1 << 20


def _rope(**kw):
    hd = _lib.MdgHeads(0x1000, 1000, 100, 24)
    r = _lib.MdgRopeAxes(dtype=1, pairs=0, nseg=1, B=2, N=3, D=24, npairs=12, naxes=2, pos=0x1000, pos_sb=6, pos_sn=2,
                         turns=0x1000, axis=0x1000, cols=0x1000)
    r.H[0], r.section[0], r.section[1], r.x[0], r.out[0] = 4, 6, 6, hd, hd
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(r, k)[v[0]] = v[1]
        else:
            setattr(r, k, v)
    return r


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=5), b"dtype"), (dict(N=0), b"N=0"), (dict(npairs=13), b"npairs"), (dict(naxes=9), b"naxes"),
    (dict(nseg=3), b"nseg"), (dict(section=(0, 5)), b"sections"), (dict(section=(0, -1)), b"section"), (dict(pairs=3), b"pairs"),
    (dict(pos=None), b"null pos"), (dict(turns=0x1004), b"aligned"), (dict(pos_i64=1, pos=0x1004), b"aligned"),
    (dict(pos_sn=-1), b"strides of pos"), (dict(H=(0, 0)), b"H[0]"), (dict(x=(0, _lib.MdgHeads(None, 1, 1, 1))), b"null x"),
    (dict(out=(0, _lib.MdgHeads(0x1000, 1000, 100, 48))), b"in place"), (dict(B=(1 << 31) - 1, N=(1 << 31) - 1), b"grid"),
    (dict(B=1 << 25, N=1, H=(0, 1024)), b"grid"),
])
def test_rope_entry_refuses(kw, word):
    lib = _lib.load()
    assert lib.mdg_rope_axes(ctypes.byref(_rope(**kw)), None) != 0
    assert word in lib.mdg_last_error_string()
    assert lib.mdg_rope_axes(None, None) != 0


def _grn(**kw):
    g = _lib.MdgGateResNorm(dtype=1, res_dtype=0, M=8, C=64, rows_per_mod=4, post=1, pre=2, resid_scale=1.0, eps=1e-6,
                            h=0x1000, y=0x2000, ldh=64, ldy=64, h_out=0x3000, xn=0x4000)
    for k, v in kw.items():
        setattr(g, k, v)
    return g


@pytest.mark.parametrize("kw, word", [
    (dict(dtype=2), b"dtype"), (dict(dtype=0, res_dtype=1), b"residual dtype"), (dict(M=0), b"M=0"), (dict(C=0), b"C=0"),
    (dict(C=8193), b"C=8193"), (dict(rows_per_mod=0), b"rows_per_mod"), (dict(post=3), b"post 3"), (dict(pre=-1), b"pre -1"),
    (dict(eps=-1.0), b"eps"), (dict(resid_scale=float("inf")), b"resid_scale"), (dict(h=None), b"null h"), (dict(ldh=63), b"ldh"),
    (dict(ldy=1), b"ldy"), (dict(y=None), b"without y"), (dict(post=0, post_w=0x1000), b"post weights"),
    (dict(pre=0), b"without a pre norm"), (dict(gate=0x1000, mod_stride=3), b"mod_stride"), (dict(h=0x1002), b"aligned"),
    (dict(gate=0x1002, mod_stride=64), b"aligned"), (dict(xn=None), b"no output"), (dict(h_out=0x1000, ldh=128), b"in place"),
    (dict(M=1 << 30), b"grid"), (dict(M=(1 << 31) - 1, C=1), b"grid"),
])
def test_grn_entry_refuses(kw, word):
    lib = _lib.load()
    assert lib.mdg_gate_res_norm(ctypes.byref(_grn(**kw)), None) != 0
    assert word in lib.mdg_last_error_string()


@pytest.mark.parametrize("kw, word", [
    (dict(), b"incoming"), (dict(dh_out=0x1000, dshift=0x1000), b"without dxn"),
    (dict(dxn=0x1000, dgate=0x1000, dmod_stride=2), b"dmod_stride"),
    (dict(dxn=0x1000, dgate=0x1000, dmod_stride=64), b"workspace"),
    (dict(dxn=0x1000, dscale=0x1000, dmod_stride=64, M=1 << 23, rows_per_mod=1), b"grid"),
])
def test_grn_backward_refuses(kw, word):
    lib = _lib.load()
    assert lib.mdg_gate_res_norm_bwd(ctypes.byref(_grn(**kw)), None, 0, None) != 0
    assert word in lib.mdg_last_error_string()


def test_grn_workspace_only_for_parameter_gradients():
    lib = _lib.load()
    assert lib.mdg_gate_res_norm_bwd_workspace_bytes(ctypes.byref(_grn(dxn=0x1000, dh=0x1000))) == 0
    assert lib.mdg_gate_res_norm_bwd_workspace_bytes(ctypes.byref(_grn(dxn=0x1000, dscale=0x1000))) > 0
    assert lib.mdg_gate_res_norm_bwd_workspace_bytes(ctypes.byref(_grn(C=9000))) == _lib.SIZE_MAX


def _z(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("args, kw, err", [
    ((_z(2, 3, 8), _z(2, 4, 1, 8), _z(2, 4, 1, 8)), {}, ValueError),
    ((_z(2, 3, 4, 8), _z(2, 4, 3, 8), _z(2, 4, 3, 8)), {}, ValueError),
    ((_z(2, 3, 4, 8), _z(2, 4, 4, 9), _z(2, 4, 4, 9)), {}, ValueError),
    ((_z(2, 3, 4, 8), _z(2, 4, 4, 8), _z(2, 5, 4, 8)), {}, ValueError),
    ((_z(1, 3, 4, 130), _z(1, 4, 4, 130), _z(1, 4, 4, 130)), {}, ValueError),
    ((_z(2, 3, 4, 8, dtype=torch.float16),) * 3, {}, TypeError),
    ((_z(2, 3, 4, 8), _z(2, 3, 4, 8, dtype=torch.bfloat16), _z(2, 3, 4, 8)), {}, TypeError),
    ((_z(2, 3, 4, 8),) * 3, {}, RuntimeError),  # a CPU tensor
])
def test_cross_attention_refuses(args, kw, err):
    with pytest.raises(err):
        X.cross_attention(*args, **kw)


def test_other_calls_refuse():
    with pytest.raises(ValueError):
        X.RopeAxes([], device="cpu")
    with pytest.raises(ValueError):
        X.RopeAxes([4], pairs="other", device="cpu")
    with pytest.raises(ValueError):
        X.RopeAxes([4, 4], freq=[1.0] * 7, device="cpu")
    plan = X.RopeAxes([4, 4], device="cpu")
    with pytest.raises(TypeError):
        X.rope_axes(plan, _z(3, 2, dtype=torch.int32), _z(1, 3, 2, 16, dtype=torch.float16))
    with pytest.raises(ValueError):
        X.rope_axes(plan, _z(3, 2, dtype=torch.int32), _z(1, 3, 2, 14))
    with pytest.raises(RuntimeError):
        X.rope_axes(plan, _z(3, 2, dtype=torch.int32), _z(1, 3, 2, 16))
    h = _z(4, 8)
    for kw in (dict(post="rms"), dict(pre="none"), dict(gate=_z(1, 8)), dict(y=h, post_w=_z(8)), dict(y=h, pre="none", scale=_z(1, 8)),
               dict(y=h, pre="other")):
        with pytest.raises(ValueError):
            X.gate_residual_norm(h, **kw)
    with pytest.raises(TypeError):
        X.gate_residual_norm(h.bfloat16(), h)
    with pytest.raises(TypeError):
        X.gate_residual_norm(h, _z(4, 9))
    with pytest.raises(RuntimeError):
        X.gate_residual_norm(h, h)


def test_rope_plan_tables():
    p = X.RopeAxes([2, 3], base=100.0, pairs="axis", device="cpu")
    assert p.cols.tolist() == [0, 1, 4, 5, 6, 2, 3, 7, 8, 9] and p.axis.tolist() == [0, 0, 1, 1, 1]
    want = torch.tensor([1.0, 100.0 ** -0.5, 1.0, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)], dtype=torch.float64) / (2 * torch.pi)
    assert torch.allclose(p.turns, want, rtol=1e-15)
    assert X.RopeAxes([2, 1], pairs="half", device="cpu").cols.tolist() == [0, 1, 2, 3, 4, 5]
    assert X.RopeAxes([2, 1], pairs="interleaved", device="cpu").cols.tolist() == [0, 2, 4, 1, 3, 5]


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
def test_forward_mode_tangents_are_refused_whatever_the_grad_mode(grad):
    """no_grad does not switch forward mode off (x * 2 keeps its tangent there): no call may drop one."""
    import torch.autograd.forward_ad as fwd

    plan = X.RopeAxes([4], device="cpu")
    pos = _z(3, 1, dtype=torch.int32)
    x, h = torch.randn(1, 3, 2, 8), torch.randn(4, 8)
    with torch.set_grad_enabled(grad), fwd.dual_level():
        dx, dh, dm = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, h, torch.ones(1, 8)))
        assert fwd.unpack_dual(dx * 2).tangent is not None
        for call in (lambda: X.cross_attention(dx, x, x), lambda: X.cross_attention(x, dx, x), lambda: X.cross_attention(x, x, dx),
                     lambda: X.rope_axes(plan, pos, dx), lambda: X.rope_axes(plan, pos, x, dx),
                     lambda: X.rope_axes(plan, pos, dx, inplace=True), lambda: X.gate_residual_norm(dh),
                     lambda: X.gate_residual_norm(h, dh), lambda: X.gate_residual_norm(h, h, gate=dm)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


@pytest.mark.parametrize("grads", [dict(dscale=0x1000), dict(dpost_w=0x1000), dict(dgate=0x1000, gate=0x1000, mod_stride=64)])
@pytest.mark.parametrize("M", [1, 8, 1000, 100000])
def test_grn_workspace_of_one_long_group(M, grads):
    """rows_per_mod at or past M is one group of M rows, whatever its value."""
    lib = _lib.load()
    kw = dict(dxn=0x1000, dmod_stride=64, M=M, **grads)
    want = lib.mdg_gate_res_norm_bwd_workspace_bytes(ctypes.byref(_grn(rows_per_mod=M, **kw)))
    assert 0 < want <= 770 * 4 * 64 * 4  # (at most 768 chunks, and the sums)
    for R in (M + 1, 1 << 30, (1 << 31) - 20, (1 << 31) - 1):
        assert lib.mdg_gate_res_norm_bwd_workspace_bytes(ctypes.byref(_grn(rows_per_mod=R, **kw))) == want


def test_tracing_is_refused():
    """A trace would hold an output's allocation without the call that fills it."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    plan, pos = X.RopeAxes([4], device="cpu"), _z(3, 1, dtype=torch.int32)
    for f, x in ((lambda t: X.cross_attention(t, t, t), _z(1, 3, 2, 8)), (lambda t: X.rope_axes(plan, pos, t), _z(1, 3, 2, 8)),
                 (lambda t: X.gate_residual_norm(t)[1], _z(4, 8))):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(f, (x,))
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(f)(x)
        with FakeTensorMode(), pytest.raises(RuntimeError, match="traced"):
            f(torch.empty(x.shape))


def test_rope_plan_refuses_frequencies_that_require_grad():
    freq = torch.ones(4, dtype=torch.float64, requires_grad=True)
    for f in (freq, freq * 2, torch.nn.Parameter(torch.ones(4))):
        with pytest.raises(ValueError, match="gradient"):
            X.RopeAxes([2, 2], freq=f, device="cpu")
    assert torch.equal(X.RopeAxes([2, 2], freq=freq.detach(), device="cpu").turns, freq.detach() / (2 * torch.pi))


def test_rope_plan_is_fixed():
    """A call keeps the tables behind a handle: assigning others is refused, not ignored."""
    import copy

    plan = X.RopeAxes([2, 2], device="cpu")
    for n in ("turns", "axis", "cols", "sections", "pairs", "npairs"):
        with pytest.raises(AttributeError, match="fixed"):
            setattr(plan, n, getattr(plan, n))
    with pytest.raises(TypeError):
        plan.sections[0] = 3
    plan.note = 1
    plan.note = 2  # (what a user adds is the user's)
    twin = copy.deepcopy(plan)
    assert torch.equal(twin.turns, plan.turns) and twin.sections == plan.sections == (2, 2)
