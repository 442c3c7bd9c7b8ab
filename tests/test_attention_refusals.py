"""What the attention operators refuse, on the host and before any HIP call (no GPU)."""
import ctypes as C

from deepx_amd import lib as dx

OK, DTYPE, ARG, SHAPE, WORKSPACE, ALIGN = 0, -1, -2, -3, -4, -5


def heads(ptr=4096, row=1024, head=64):
    return dx.Heads(ptr, row, head)


def norm_part(**kw):
    p = dx.NormropePart(heads(), heads(8192), heads(16384), 256, 512, 4, 1, dx.BF16)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def rotary(**kw):
    r = dx.Rotary(256, 512, 1024, 100, 64, 0, dx.I32)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def test_normrope():
    L = dx.load()

    def fwd(part=None, rot=None, dtype=dx.BF16, n=1, rows=0, dim=64, eps=1e-6):
        parts = (dx.NormropePart * 1)(part or norm_part())
        return L.dxh_normrope(dtype, parts, n, rows, dim, eps, rot, None)

    assert fwd() == OK and fwd(rot=rotary()) == OK  # no rows: checked, nothing launched
    assert fwd(dtype=dx.F64) == DTYPE and fwd(dtype=dx.I32) == DTYPE and fwd(dtype=dx.F8E4M3) == DTYPE
    assert fwd(n=0) == ARG and fwd(n=5) == ARG and fwd(rows=-1) == ARG and fwd(eps=-1.0) == ARG and fwd(eps=float("nan")) == ARG
    assert L.dxh_normrope(dx.BF16, None, 1, 0, 64, 1e-6, None, None) == ARG
    for dim in (0, 8, 24, 272, -16):
        assert fwd(dim=dim) == SHAPE
    assert fwd(rot=rotary(dim=66)) == SHAPE and fwd(rot=rotary(dim=7)) == SHAPE and fwd(rot=rotary(dim=-2)) == SHAPE
    assert fwd(rot=rotary(interleaved=2)) == ARG and fwd(rot=rotary(position_dtype=dx.F32)) == DTYPE
    assert fwd(rot=rotary(cos=None), rows=1) == ARG and fwd(rot=rotary(table_rows=0), rows=1) == ARG
    assert fwd(rot=rotary(sin=258)) == ALIGN and fwd(rot=rotary(positions=1026)) == ALIGN and fwd(rot=rotary(positions=1028, position_dtype=dx.I64)) == ALIGN
    assert fwd(rot=rotary(dim=0, cos=None)) == OK  # no rotation: tables are not looked at
    assert fwd(norm_part(heads=-1)) == ARG and fwd(norm_part(norm=2)) == ARG and fwd(norm_part(weight_dtype=dx.F16)) == DTYPE
    assert fwd(norm_part(weight_dtype=dx.F32)) == OK and fwd(norm_part(weight=None, weight_dtype=0)) == OK
    assert fwd(norm_part(weight=264)) == ALIGN
    assert fwd(norm_part(x=dx.Heads()), rows=1) == ARG and fwd(norm_part(y=dx.Heads()), rows=1) == ARG
    for bad in (heads(4098), heads(row=1025), heads(head=68)):
        assert fwd(norm_part(x=bad), rows=1) == ALIGN and fwd(norm_part(y=bad), rows=1) == ALIGN


def test_normrope_backward():
    L = dx.load()
    parts = (dx.NormropePart * 1)(norm_part())
    n = C.c_size_t(1)
    assert L.dxh_normrope_backward_workspace_bytes(dx.BF16, parts, 1, 100, 64, C.byref(n)) == OK and n.value > 0
    assert L.dxh_normrope_backward_workspace_bytes(dx.BF16, parts, 1, 0, 64, C.byref(n)) == OK and n.value == 0
    assert L.dxh_normrope_backward_workspace_bytes(dx.BF16, parts, 1, 100, 64, None) == ARG
    assert L.dxh_normrope_backward_workspace_bytes(dx.BF16, parts, 1, -1, 64, C.byref(n)) == ARG
    assert L.dxh_normrope_backward_workspace_bytes(dx.BF16, parts, 1, 1, 40, C.byref(n)) == SHAPE
    assert L.dxh_normrope_backward_workspace_bytes(dx.I8, parts, 1, 1, 64, C.byref(n)) == DTYPE
    back = lambda part, ws, nbytes: L.dxh_normrope_backward(dx.BF16, (dx.NormropePart * 1)(part), 1, 100, 64, 1e-6, None, ws, nbytes, None)  # noqa: E731
    assert back(norm_part(), None, 0) == WORKSPACE and back(norm_part(), 4096, 16) == WORKSPACE and back(norm_part(), 4100, 1 << 30) == WORKSPACE
    assert back(norm_part(dx=dx.Heads()), 4096, 1 << 30) == ARG and back(norm_part(dx=heads(4100)), 4096, 1 << 30) == ALIGN and back(norm_part(dweight=513), 4096, 1 << 30) == ALIGN
    assert L.dxh_normrope_backward_workspace_bytes(dx.BF16, (dx.NormropePart * 1)(norm_part(dweight=None)), 1, 100, 64, C.byref(n)) == OK and n.value == 0
