"""dxh_kvcache_write and dxh_kvcache_read: every bit against their 32-bit definition (tests/kv_reference.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

from deepx_amd import lib as dx
from tests import kv_reference as R

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def check_cache(c):
    for got, want, what in zip(c.download(), (c.k, c.v, c.ks, c.vs), ("k", "v", "k_scale", "v_scale")):
        got, want = got.view(np.int8), want.view(np.int8)
        if c.code == "e4m3" and "scale" not in what:  # a NaN of either sign
            got, want = np.where(got == -1, 127, got), np.where(want == -1, 127, want)
        bad = np.argwhere(got != want)
        assert not len(bad), f"{what}: {len(bad)} bytes differ, the first at {bad[0]}"


def call_write(L, c, rows, name, k, v):
    """one write through the library and one by the definition"""
    dx.check(L.dxh_kvcache_write(c.desc, rows.upload(), R.DT[name], R.heads(k), R.heads(v), stream()), "write")
    R.write(c, rows, k.float().cpu().numpy(), v.float().cpu().numpy())


LAYOUTS = [  # code, page, heads, dim
    ("i8", 16, 2, 64), ("e4m3", 16, 1, 16), ("i8", 32, 3, 80), ("e4m3", 64, 2, 128), ("i8", 128, 1, 256), ("e4m3", 128, 2, 96), ("e4m3", 32, 1, 48), ("i8", 64, 5, 32)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", LAYOUTS, ids=str)
def test_growing_sequences(dxh, layout, name):
    """prompts of odd lengths, then single tokens, then a few at once, each larger or smaller than before: pages that are new, part
    full, exactly full; scales that grow and scales that stay; one sequence that gets nothing"""
    code, page, heads, dim = layout
    c = R.Cache(code, page, heads, dim, 5, 5, seed=page + dim)
    c.desc = c.upload()
    rng = np.random.default_rng(dim)
    have = [0] * 5
    for counts, size in (((page, page + 1, 3, 0, 2 * page - 1), 1.0), ((1, 1, 1, 0, 1), 3.0), ((1, 1, 1, 1, 1), 0.1), ((2, page, 5, 3, 7), 30.0), ((1, 0, 1, 1, 1), 1e-3)):
        have = [h + n for h, n in zip(have, counts)]
        rows = R.Rows(counts, have, extra=2)
        k, v = (torch.from_numpy((rng.standard_normal((rows.rows, heads, dim)) * size).astype(np.float32)).cuda().to(R.TT[name]) for _ in range(2))
        call_write(dxh, c, rows, name, k, v)
        check_cache(c)
        back = [torch.full_like(k, 7.0), torch.full_like(k, 7.0)]
        dx.check(dxh.dxh_kvcache_read(c.desc, rows.upload(), R.DT[name], R.heads(back[0]), R.heads(back[1]), stream()), "read")
        for which in (0, 1):
            want = R.read(c, rows, which)
            got = back[which].cpu()
            for r in range(rows.rows):
                expect = torch.from_numpy(want[r]).to(R.TT[name]) if r in want else torch.full((heads, dim), 7.0, dtype=R.TT[name])
                assert torch.equal(got[r], expect), (which, r)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_every_16_bit_value(dxh, code):
    """all 65536 bf16 and f16 values (NaN, infinities and subnormals among them), 64 x 16 a page"""
    for name, tt in (("bf16", torch.bfloat16), ("f16", torch.float16)):
        c = R.Cache(code, 64, 1, 16, 1, 64, seed=1)
        c.desc = c.upload()
        x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(tt).view(4096, 1, 16).cuda()
        y = x[torch.randperm(4096, generator=torch.Generator().manual_seed(3)).cuda()].contiguous()
        call_write(dxh, c, R.Rows([4096], [4096]), name, x, y)
        check_cache(c)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_rounding_ties_and_tiny_scales(dxh, code):
    """values at the halves between codes, a page of zeros, pages of subnormal and of huge values"""
    c = R.Cache(code, 16, 1, 64, 1, 5, seed=2)
    c.desc = c.upload()
    x = np.zeros((80, 1, 64), np.float32)
    top = float(R.MAX[code])
    x[:16] = (np.arange(1024).reshape(16, 1, 64) / 1024 * top)
    x[0, 0, 0] = top
    x[16:32] = np.rint(np.random.default_rng(1).uniform(-top, top, (16, 1, 64))) + 0.5
    x[16, 0, 0] = top
    x[48:64] = np.random.default_rng(2).standard_normal((16, 1, 64)) * 1e-42
    x[64:80] = np.random.default_rng(3).uniform(-3.4e38, 3.4e38, (16, 1, 64))
    k = torch.from_numpy(x).cuda()
    call_write(dxh, c, R.Rows([80], [80]), "f32", k, k)
    check_cache(c)


def test_bad_pages_lengths_and_offsets(dxh):
    """page numbers that are none, rows before token 0 and past the table, offsets outside the tensor, more rows than max_rows: nothing
    but the pages that exist is touched, reads of what does not exist give zeros, other rows stay"""
    for code in ("i8", "e4m3"):
        c = R.Cache(code, 16, 2, 32, 4, 3, seed=5, missing=[(0, 1, -1), (1, 0, 14), (2, 2, 2 ** 31 - 1), (3, 1, -2 ** 31)])
        assert c.pages == 14
        c.desc = c.upload()
        # sequence 0: across its missing page; 1: begins before token 0; 2: runs past the table; 3: more rows than max_rows
        rows = R.Rows((40, 20, 30, 45), (44, 12, 60, 45), extra=3, max_rows=40)
        g = torch.Generator(device="cuda").manual_seed(1)
        k, v = (torch.randn(rows.rows, 2, 32, generator=g, device="cuda") for _ in range(2))
        call_write(dxh, c, rows, "f32", k, v)
        check_cache(c)
        back = [torch.full_like(k, 7.0), torch.full_like(k, 7.0)]
        dx.check(dxh.dxh_kvcache_read(c.desc, rows.upload(), dx.F32, R.heads(back[0]), R.heads(back[1]), stream()), "read")
        for which in (0, 1):
            want, got = R.read(c, rows, which), back[which].cpu().numpy()
            for r in range(rows.rows):
                assert np.array_equal(got[r], want[r] if r in want else np.full((2, 32), 7.0, np.float32)), (which, r)
        # wild offsets and lengths stay inside the tensors
        for offsets, lengths in (([-5, 10, 5, 10 ** 9, 7], [16, -3, 2 ** 31 - 1, 40]), ([0, 0, 0, 0, 0], [1, 1, 1, 1])):
            off, length = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (offsets, lengths))
            desc = dx.KvRows(off.data_ptr(), length.data_ptr(), rows.rows, 4, 40)
            dx.check(dxh.dxh_kvcache_write(c.desc, desc, dx.F32, R.heads(k), R.heads(v), stream()))
            dx.check(dxh.dxh_kvcache_read(c.desc, desc, dx.F32, R.heads(back[0]), R.heads(back[1]), stream()))
            torch.cuda.synchronize()


def test_without_table_or_offsets_strided_on_a_stream_and_recorded(dxh):
    """a cache without paging, the same number of rows a sequence, [heads, rows, dim] views, recorded into a graph whose lengths move on"""
    st, graph = C.c_void_p(), C.c_void_p()
    dx.check(dxh.dxh_stream_create(C.byref(st)))
    c = R.Cache("e4m3", 16, 3, 48, 4, 4, seed=7, paged=False)
    c.desc = c.upload()
    rows = R.Rows((2,) * 4, (3, 15, 16, 40), uniform=True)
    desc = rows.upload()
    base = torch.zeros(2, 3, 8, 48, device="cuda", dtype=torch.bfloat16)
    k, v = base[0].transpose(0, 1), base[1].transpose(0, 1)
    torch.cuda.synchronize()
    dx.check(dxh.dxh_graph_begin_capture(st))
    dx.check(dxh.dxh_kvcache_write(c.desc, desc, dx.BF16, R.heads(k), R.heads(v), st))
    dx.check(dxh.dxh_graph_end_capture(st, C.byref(graph)))
    for step in range(4):
        base.copy_(torch.randn(base.shape, device="cuda") * (1 + step))
        rows.lengths = [n + 2 * step for n in (3, 15, 16, 40)]
        rows.dev[1].copy_(torch.tensor(rows.lengths, dtype=torch.int32))
        torch.cuda.synchronize()
        dx.check(dxh.dxh_graph_launch(graph, st))
        dx.check(dxh.dxh_stream_sync(st))
        R.write(c, rows, k.float().cpu().numpy(), v.float().cpu().numpy())
        check_cache(c)
    dx.check(dxh.dxh_graph_destroy(graph))
    dx.check(dxh.dxh_stream_destroy(st))


def test_large_cache(dxh):
    """codes past 2^32 bytes: the last pages of a 5 GB cache of keys"""
    page, heads, dim = 128, 8, 256
    pages = 20000
    size = pages * heads * page * dim
    assert size > 2 ** 32
    k, v = (torch.zeros(size, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.ones(pages, heads, device="cuda") for _ in range(2))
    table = torch.tensor([[3, pages - 1], [pages - 2, 0]], dtype=torch.int32, device="cuda")
    length = torch.tensor([200, 100], dtype=torch.int32, device="cuda")
    cache = dx.KvCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(), pages, 2, page, heads, dim, dx.I8)
    x = torch.randn(200, heads, dim, device="cuda")
    rows = dx.KvRows(None, length.data_ptr(), 200, 2, 100)
    dx.check(dxh.dxh_kvcache_write(cache, rows, dx.F32, R.heads(x), R.heads(x), stream()))
    back = [torch.empty_like(x), torch.empty_like(x)]
    dx.check(dxh.dxh_kvcache_read(cache, rows, dx.F32, R.heads(back[0]), R.heads(back[1]), stream()))
    # a code is off by at most half a step of its page's scale, and the scales are max |x| / 127 of the page's rows — in page 3, where the first
    # sequence has 100 older tokens, at least the old scale of 1
    for b, scales in zip(back, (ks, vs)):
        for place, rows_of_page, least in ((3, slice(0, 28), 1.0), (pages - 1, slice(28, 100), 0.0), (pages - 2, slice(100, 200), 0.0)):
            top = x[rows_of_page].abs().amax((0, 2)) / 127
            assert torch.allclose(scales[place], top.clamp(min=least), rtol=1e-6)
            off = ((b - x)[rows_of_page].abs().amax((0, 2)) / scales[place]).max().item()
            assert off <= 0.501, (place, off)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("page,dim", [(16, 32), (64, 128)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_broken_scale_is_not_written_over(dxh, bad, page, dim, code):
    """older tokens whose page has a scale that is no finite number have no values: a new token in their page does not make them look as if they had, and the
    attention goes on giving NaN; a page that begins with the new rows gets a scale of its own"""
    c = R.Cache(code, page, 2, dim, 3, 2, seed=8)
    c.ks[c.page_of(0, 0), 1] = c.vs[c.page_of(1, 0), 0] = c.ks[c.page_of(2, 0), 0] = bad
    c.desc = c.upload()
    rows = R.Rows((1, 2, page), (page // 2, page - 1, page))  # the third sequence's page is new
    desc = rows.upload()
    g = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(rows.rows, 2, dim, generator=g, device="cuda") * 100 for _ in range(2))
    dx.check(dxh.dxh_kvcache_write(c.desc, desc, dx.F32, R.heads(k), R.heads(v), stream()))
    _, _, ks, vs = c.download()
    same = lambda x: x == bad or (np.isnan(bad) and np.isnan(x))  # noqa: E731
    assert same(ks[c.page_of(0, 0), 1]) and same(vs[c.page_of(1, 0), 0])
    assert np.isfinite(ks[c.page_of(0, 0), 0]) and np.isfinite(vs[c.page_of(0, 0)]).all() and np.isfinite(ks[c.page_of(2, 0)]).all() and np.isfinite(vs[c.page_of(2, 0)]).all()
    q, out, ws, need = torch.randn(rows.rows, 2, dim, generator=g, device="cuda"), torch.empty(rows.rows, 2, dim, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda"), C.c_size_t(0)
    dx.check(dxh.dxh_kvcache_attention_workspace_bytes(c.desc, desc, dx.F32, 2, C.byref(need)))
    assert need.value <= ws.numel()
    dx.check(dxh.dxh_kvcache_attention(c.desc, desc, dx.F32, 2, R.heads(q), R.heads(out), None, 0.1, 1, 0, ws.data_ptr(), ws.numel(), stream()))
    assert torch.isnan(out[0, 1]).all() and torch.isnan(out[1:3, 0]).all()
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[1:3, 1]).all() and torch.isfinite(out[3:]).all()
