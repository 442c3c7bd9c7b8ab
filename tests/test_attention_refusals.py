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


def test_results_that_would_overwrite_other_inputs():
    """two parts whose results meet, or meet the other part's input, are refused (a result in its own input's place is not)"""
    L = dx.load()
    two = lambda x0, y0, x1, y1: (dx.NormropePart * 2)(norm_part(x=heads(x0), y=heads(y0)), norm_part(x=heads(x1), y=heads(y1)))  # noqa: E731
    for ptrs in ((4096, 8192, 16384, 8192), (4096, 16384, 16384, 4096), (4096, 8192, 8192, 16384)):
        assert L.dxh_normrope(dx.BF16, two(*ptrs), 2, 1, 64, 1e-6, None, None) == ARG, ptrs
    assert L.dxh_kvcache_read(cache(), kvrows(rows=1), dx.BF16, heads(), heads(), None) == ARG
    assert L.dxh_kvcache_attention(cache(), kvrows(rows=1), dx.BF16, 14, heads(), heads(), None, 0.125, 1, 0, None, 0, None) == ARG


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


def cache(**kw):
    c = dx.KvCache(4096, 8192, 256, 512, 1024, 100, 8, 16, 2, 64, dx.I8)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def kvrows(**kw):
    r = dx.KvRows(256, 512, 0, 4, 8)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


BAD_CACHE = [(dict(code=dx.I16), DTYPE), (dict(code=dx.BF16), DTYPE), (dict(num_pages=-1), ARG), (dict(pages_per_seq=-1), ARG), (dict(heads=0), ARG), (dict(page_size=8), SHAPE),
             (dict(page_size=48), SHAPE), (dict(page_size=256), SHAPE), (dict(dim=24), SHAPE), (dict(dim=272), SHAPE), (dict(dim=0), SHAPE), (dict(k=4100), ALIGN), (dict(v=8193), ALIGN),
             (dict(k_scale=258), ALIGN), (dict(page_table=1026), ALIGN), (dict(page_table=None, num_pages=31), SHAPE),
             (dict(pages_per_seq=(1 << 26) + 1), -6), (dict(num_pages=1 << 31), -6)]
BAD_ROWS = [(dict(batch=-1), ARG), (dict(rows=-1), ARG), (dict(max_rows=-1), ARG), (dict(offsets=258), ALIGN), (dict(lengths=514), ALIGN), (dict(offsets=None, rows=31), SHAPE),
            (dict(rows=1 << 31), -6), (dict(rows=1, lengths=None), ARG)]


def test_kvcache_write_and_read():
    L = dx.load()
    for fn in (L.dxh_kvcache_write, L.dxh_kvcache_read):
        call = lambda c=None, r=None, dtype=dx.BF16, k=None, v=None: fn(c or cache(), r or kvrows(), dtype, k or heads(), v or heads(16384), None)  # noqa: E731, B023
        assert call() == OK and call(cache(code=dx.F8E4M3)) == OK and call(cache(page_table=None, num_pages=32)) == OK
        for kw, rc in BAD_CACHE:
            assert call(cache(**kw)) == rc, kw
        for kw, rc in BAD_ROWS:
            assert call(r=kvrows(**kw)) == rc, kw
        assert call(r=kvrows(rows=1), c=cache(k=None)) == ARG and call(r=kvrows(rows=1), c=cache(v_scale=None)) == ARG
        assert call(dtype=dx.F64) == DTYPE and call(dtype=dx.I8) == DTYPE
        assert fn(None, kvrows(), dx.BF16, heads(), heads(), None) == ARG and fn(cache(), None, dx.BF16, heads(), heads(), None) == ARG
        assert fn(cache(), kvrows(), dx.BF16, None, heads(), None) == ARG
        assert call(r=kvrows(rows=1), k=dx.Heads()) == ARG and call(k=heads(4100)) == ALIGN and call(v=heads(row=1028)) == ALIGN and call(v=heads(head=60)) == ALIGN
        assert call(r=kvrows(rows=1 << 30, batch=1 << 20, max_rows=1 << 20)) == -6  # more workgroups than a launch has


def test_kvcache_attention():
    L = dx.load()
    n = C.c_size_t(1)

    def att(c=None, r=None, dtype=dx.BF16, q_heads=14, q=None, out=None, lse=None, scale=0.125, causal=1, window=0, ws=None, nbytes=0):
        return L.dxh_kvcache_attention(c or cache(), r or kvrows(), dtype, q_heads, q or heads(), out or heads(8192), lse, scale, causal, window, ws, nbytes, None)

    query = lambda c=None, r=None, dtype=dx.BF16, q_heads=14: L.dxh_kvcache_attention_workspace_bytes(c or cache(), r or kvrows(), dtype, q_heads, C.byref(n))  # noqa: E731
    assert att() == OK and query() == OK and n.value == 0
    for kw, rc in BAD_CACHE:
        assert att(cache(**kw)) == rc and query(cache(**kw)) == rc, kw
    for kw, rc in BAD_ROWS:
        assert att(r=kvrows(**kw)) == rc and query(r=kvrows(**kw)) == rc, kw
    assert att(q_heads=0) == ARG and att(q_heads=15) == SHAPE and query(q_heads=15) == SHAPE and query(q_heads=-2) == ARG and query(dtype=dx.F64) == DTYPE
    assert L.dxh_kvcache_attention_workspace_bytes(cache(), kvrows(), dx.BF16, 14, None) == ARG
    assert att(causal=2) == ARG and att(window=-1) == ARG and att(scale=float("nan")) == ARG and att(scale=float("inf")) == ARG
    assert att(lse=258) == ALIGN and att(q=heads(4098)) == ALIGN and att(out=heads(head=65)) == ALIGN
    assert att(r=kvrows(rows=1), q=dx.Heads()) == ARG and att(r=kvrows(rows=1), out=dx.Heads()) == ARG
    assert att(r=kvrows(rows=1 << 30, batch=1, max_rows=1 << 30), q_heads=14) == -6
    # a long cache under one row is cut: the workspace is asked for and checked
    long = cache(num_pages=100000, pages_per_seq=8192)
    one = kvrows(rows=1, batch=1, max_rows=1)
    assert query(long, one) == OK and n.value > 0
    assert att(long, one) == WORKSPACE and att(long, one, ws=4096, nbytes=n.value - 1) == WORKSPACE and att(long, one, ws=4096 + 16, nbytes=n.value) == WORKSPACE


def test_results_laid_out_unlike_the_input_they_replace():
    """in place only element on element: the same pointer with other strides is refused where a stride is used at all"""
    L = dx.load()
    same = lambda rows, n, row=1024, head=64, **kw: L.dxh_normrope(dx.BF16, (dx.NormropePart * 1)(norm_part(x=heads(4096), y=heads(4096, row, head), heads=n, **kw)), 1, rows, 64, 1e-6, rotary(cos=None), None)  # noqa: E731
    assert same(2, 4, row=2048) == ARG and same(1, 4, head=128) == ARG
    back = lambda dx_: L.dxh_normrope_backward(dx.BF16, (dx.NormropePart * 1)(norm_part(x=heads(4096), y=heads(8192), dx=dx_)), 1, 2, 64, 1e-6, None, 4096, 1 << 30, None)  # noqa: E731
    assert back(heads(8192, row=2048)) == ARG and back(heads(4096, head=128)) == ARG


def test_caches_whose_halves_are_one():
    L = dx.load()
    for kw in (dict(v=4096), dict(v_scale=256)):
        for fn in (L.dxh_kvcache_write, L.dxh_kvcache_read):
            assert fn(cache(**kw), kvrows(rows=1), dx.BF16, heads(), heads(16384), None) == ARG, kw
        assert L.dxh_kvcache_attention(cache(**kw), kvrows(rows=1), dx.BF16, 14, heads(), heads(8192), None, 0.125, 1, 0, None, 0, None) == ARG, kw


def test_sizes_past_one_launch():
    """a launch has fewer than 2^32 work items; a score scale is finite in base 2 too"""
    L, big = dx.load(), -6
    n = C.c_size_t(1)
    rows = kvrows(rows=1 << 26, batch=1 << 23, max_rows=8)
    assert L.dxh_kvcache_write(cache(), rows, dx.BF16, heads(), heads(16384), None) == big  # 2^23 sequences, 2 heads, keys and values, 2 pages each, 64 lanes
    assert L.dxh_kvcache_attention_workspace_bytes(cache(), kvrows(rows=1 << 24, batch=1 << 23, max_rows=1), dx.BF16, 14, C.byref(n)) == big
    assert L.dxh_kvcache_attention(cache(), kvrows(rows=1), dx.BF16, 14, heads(), heads(8192), None, 3e38, 1, 0, None, 0, None) == ARG


def test_counts_whose_products_pass_64_bits():
    """sizes that are each within their limits but not together: too large, not wrapped around into a launch that fits"""
    L, big, top = dx.load(), -6, (1 << 31) - 1
    n = C.c_size_t(1)
    # the second writes 2 x 2^30 heads x (2^27 + 1) slots x 2^30 sequences: of 2^88 + 2^61 workgroups of 64 lanes, none is left in 64 bits
    for heads_, batch, most in ((1 << 26, 1 << 10, top), (1 << 30, 1 << 30, top), (top, top, top), (1 << 20, 1 << 24, 1 << 24)):
        c, r = cache(heads=heads_, pages_per_seq=1), kvrows(rows=1, batch=batch, max_rows=most)
        for fn in (L.dxh_kvcache_write, L.dxh_kvcache_read):
            assert fn(c, r, dx.BF16, heads(), heads(16384), None) == big, (heads_, batch, most)
        for q in (heads_, top // heads_ * heads_):
            assert L.dxh_kvcache_attention_workspace_bytes(c, r, dx.BF16, q, C.byref(n)) == big, (heads_, batch, most)


def test_results_in_the_place_of_weights_tables_scales_and_each_other():
    L = dx.load()
    fwd = lambda *parts: L.dxh_normrope(dx.BF16, (dx.NormropePart * len(parts))(*parts), len(parts), 1, 64, 1e-6, rotary(), None)  # noqa: E731
    other = norm_part(x=heads(32768), y=heads(40960), weight=49152)
    for part in (norm_part(y=heads(256)), norm_part(y=heads(49152)), norm_part(y=heads(512)), norm_part(y=heads(1024))):  # its weight, the other's, sines, positions
        assert fwd(part, other) == ARG and fwd(other, part) == ARG
    assert fwd(norm_part(y=heads(256), weight=2048, norm=0)) == ARG  # cosines
    other = norm_part(x=heads(32768), y=heads(40960), dx=heads(57344), weight=49152, dweight=65536)
    back = lambda *parts: L.dxh_normrope_backward(dx.F32, (dx.NormropePart * len(parts))(*parts), len(parts), 1, 64, 1e-6, rotary(positions=None), 1 << 20, 1 << 30, None)  # noqa: E731
    for part in (norm_part(dx=heads(49152)), norm_part(dx=heads(65536)), norm_part(dweight=57344), norm_part(dweight=16384)):
        part.weight_dtype = other.weight_dtype = dx.F32
        assert back(part, other) == ARG and back(other, part) == ARG
    rows = kvrows(rows=1)
    for lse in (4096, 12288, 8192 + 16384, 256, 512, 1024, 256 * 3):
        assert L.dxh_kvcache_attention(cache(v=12288, k=24576), kvrows(rows=1, lengths=768), dx.BF16, 14, heads(4096), heads(8192), lse, 0.125, 1, 0, None, 0, None) == ARG, lse
    assert L.dxh_kvcache_attention(cache(), rows, dx.BF16, 14, heads(16384), heads(32768), 32768, 0.125, 1, 0, None, 0, None) == ARG
    for out in (4096, 8192):  # the codes
        assert L.dxh_kvcache_attention(cache(), rows, dx.BF16, 14, heads(16384), heads(out), None, 0.125, 1, 0, None, 0, None) == ARG
        for fn in (L.dxh_kvcache_write, L.dxh_kvcache_read):
            assert fn(cache(), rows, dx.BF16, heads(out), heads(16384), None) == ARG and fn(cache(), rows, dx.BF16, heads(16384), heads(out), None) == ARG
    for out in (256, 512, 1024):  # scales and offsets, the page table
        for fn in (L.dxh_kvcache_write, L.dxh_kvcache_read):
            assert fn(cache(), rows, dx.BF16, heads(16384), heads(out), None) == ARG
