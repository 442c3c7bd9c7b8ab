"""Which attention calls are cut into slices, from the workspace that the query asks for (host only, no GPU)."""
import ctypes as C

import pytest

from deepx_amd import lib as dx

DT = {"f32": dx.F32, "f16": dx.F16, "bf16": dx.BF16}


def slices(name, page, dim, heads, q_heads, batch, longest, rows, max_rows):
    per = -(-longest // page)
    cache = dx.KvCache(4096, 1 << 20, 256, 512, 1024, batch * per + 2, per, page, heads, dim, dx.I8)
    desc, need = dx.KvRows(256, 512, rows, batch, max_rows), C.c_size_t(1)
    dx.check(dx.load().dxh_kvcache_attention_workspace_bytes(cache, desc, DT[name], q_heads, C.byref(need)))
    each = rows * q_heads * (dim + 2) * 4  # one slice's partial results, all of them rounded up to 256 bytes
    return -(-(need.value - 255) // each) if need.value else 1


@pytest.mark.parametrize("name,page,dim,batch,longest,rows", [("bf16", 16, 64, 2, 1500, 531), ("f16", 64, 128, 2, 2000, 431), ("f32", 16, 64, 1, 1000, 201), ("bf16", 64, 256, 1, 2200, 131), ("f32", 32, 96, 2, 900, 154),
                                                              ("bf16", 128, 192, 1, 3000, 34)], ids=str)
def test_prompts_whose_tiles_leave_cus_idle(name, page, dim, batch, longest, rows):
    """room for as many rows as leave some CUs idle, more work than the kernel for few rows is given: slices for every head size"""
    assert slices(name, page, dim, 1, 2, batch, longest, rows, 255 * 128 // 2 // batch) > 1


def test_few_rows():
    assert slices("bf16", 16, 64, 2, 14, 1, 777, 1, 1) == 1  # fewer tiles than one slice has
    assert slices("bf16", 16, 64, 1, 3, 1, 40000, 2, 2) > 16  # one long sequence: what runs at once
    assert slices("bf16", 64, 128, 8, 32, 64, 16384, 64, 1) == 4  # a batch: eight workgroups a CU
    assert slices("bf16", 64, 128, 8, 32, 4, 4096, 16000, 4096) == 1  # prompts that fill the card
    assert slices("bf16", 64, 64, 1, 2, 1, 1 << 20, 1, 1) <= 128
