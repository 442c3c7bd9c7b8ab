"""dxh_kvcache_attention against a 64-bit softmax over the tokens a row sees (tests/kv_reference.py, where the bars are derived)."""
import ctypes as C

import numpy as np
import pytest
import torch

from deepx_amd import lib as dx
from tests import kv_reference as R

pytestmark = pytest.mark.gpu


def stream():
    return torch.cuda.current_stream().cuda_stream


def call(L, cache, rows_desc, name, q, out, lse, scale, causal, window, st=None, ws=None):
    need = C.c_size_t(0)
    dx.check(L.dxh_kvcache_attention_workspace_bytes(cache, rows_desc, R.DT[name], q.shape[1], C.byref(need)), "query")
    if ws is None:
        ws = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")
    assert ws.numel() >= need.value
    dx.check(L.dxh_kvcache_attention(cache, rows_desc, R.DT[name], q.shape[1], R.heads(q), R.heads(out), lse.data_ptr() if lse is not None else None, scale, causal, window, ws.data_ptr(),
                                     need.value, stream() if st is None else st), "attention")
    return ws


def check(L, c, rows, name, q_heads, causal=1, window=0, scale=None, q=None, seed=0, size=1.0, far=0.0):
    scale = c.dim ** -0.5 if scale is None else scale
    if q is None:
        q = torch.randn(rows.rows, q_heads, c.dim, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * size
    q = q.to(R.TT[name])
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    ws = call(L, c.upload(), rows.upload(), name, q, out, lse, scale, causal, window)
    want = R.attention(c, rows, q.double().cpu().numpy(), scale, causal, window)
    got, got_lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert ws is not None
    for r in range(rows.rows):
        if r not in want:  # rows behind the last sequence or beyond max_rows
            assert (got[r] == 7.0).all() and (got_lse[r] == 7.0).all(), r
            continue
        bar, lse_bar = R.attention_bar(name, c, want[r], far)
        assert np.array_equal(np.isinf(got_lse[r]), np.isinf(want[r][1])), r
        err = np.abs(got[r] - want[r][0])
        worst = float((err / bar).max())
        assert worst <= 1, (r, worst)
        fine = np.isfinite(want[r][1])
        assert (np.abs(got_lse[r][fine] - want[r][1][fine]) <= lse_bar[fine]).all(), r
    return out


# code, page, key heads, query heads, dim, counts, lengths
CASES = [
    ("i8", 16, 1, 1, 64, (1,), (1,)), ("e4m3", 16, 2, 14, 64, (1, 1, 1), (1, 64, 65)), ("i8", 16, 2, 14, 64, (1,), (777,)), ("e4m3", 32, 1, 16, 128, (1, 1), (63, 500)),
    ("i8", 64, 1, 17, 128, (1, 1), (129, 1)), ("e4m3", 128, 3, 3, 80, (2, 5, 1), (2, 130, 255)), ("i8", 16, 2, 4, 16, (3, 0, 4), (30, 9, 4)), ("i8", 32, 1, 2, 96, (33, 7), (40, 200)),
    ("e4m3", 64, 2, 10, 256, (4, 1), (100, 321)), ("i8", 128, 1, 8, 192, (1, 9), (300, 9)), ("e4m3", 16, 1, 5, 48, (70, 1, 17), (70, 90, 100)), ("i8", 64, 4, 4, 32, (130, 65), (130, 150)),
    ("e4m3", 64, 1, 4, 128, (200,), (231,)), ("i8", 16, 1, 7, 64, (129,), (140,)),
]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_ragged(dxh, case, name):
    code, page, hk, hq, dim, counts, lengths = case
    c = R.Cache(code, page, hk, dim, len(counts), -(-max(lengths) // page), seed=dim + hq)
    check(dxh, c, R.Rows(counts, lengths, extra=1), name, hq)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("window", [0, 1, 2, 63, 64, 65, 200, 2 ** 40])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_masks(dxh, code, window, causal, name):
    """sliding windows with and without the causal limit over chunks of rows that begin inside and at the edges of tiles"""
    c = R.Cache(code, 16, 1, 64, 3, 20, seed=window % 97)
    check(dxh, c, R.Rows((70, 1, 33), (300, 257, 33)), name, 3, causal=causal, window=window)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_what_a_row_does_not_see_has_no_effect(dxh, code, name):
    """missing pages, rows without tokens, lengths of zero, past the table and negative, rows beyond max_rows; every code that no row sees is the
    worst there is (NaN in e4m3), every scale of a page that no row sees is NaN"""
    for rows in (R.Rows((5, 3, 40, 2, 1, 9), (90, 1, 20, 0, 16, 200), extra=2, max_rows=30), R.Rows((1, 1, 1, 1, 1, 1), (0, -5, 2 ** 31 - 1, 33, 17, 96))):
        c = R.Cache(code, 16, 2, 64, 6, 6, seed=3, missing=[(0, 1, -1), (1, 0, 1 << 30), (2, 5, -7), (4, 0, -1)])
        seen = np.zeros((c.pages, 16), bool)
        for b, r, t in rows.each():
            for j in range(0, min(t + 1, rows.lengths[b], 96) if t >= 0 else 0):
                if c.page_of(b, j // 16) >= 0:
                    seen[c.page_of(b, j // 16), j % 16] = True
        c.k[~np.broadcast_to(seen[:, None, :, None], c.k.shape)] = 127  # 0x7f: NaN in e4m3
        c.v[~np.broadcast_to(seen[:, None, None, :], c.v.shape)] = 127
        c.ks[~seen.any(1)] = np.nan
        c.vs[~seen.any(1)] = np.inf
        check(dxh, c, rows, name, 6)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_nan_of_a_later_token(dxh, name):
    """a NaN among the values (and, of another token, the keys) of a token: rows before it are as without it, rows that see it are NaN"""
    for kind in ("k", "v"):
        c = R.Cache("e4m3", 16, 1, 64, 1, 8, seed=4)
        rows = R.Rows((100,), (120,))
        q = torch.randn(100, 3, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
        clean = check(dxh, c, rows, name, 3, q=q)
        p, token = c.page_of(0, 70 // 16), 70 % 16
        if kind == "k":
            c.k[p, 0, token, 5] = 127
        else:
            c.v[p, 0, 5, token] = -1
        out = torch.full_like(clean, 7.0)
        call(dxh, c.upload(), rows.upload(), name, q.to(R.TT[name]), out, None, 0.125, 1, 0)
        sees = torch.arange(100) + 20 >= 70
        assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees][..., 5]).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_long_sequences_in_slices(dxh, code, name):
    """few rows over long ragged sequences: the tokens are cut into slices and joined; the same bits twice"""
    c = R.Cache(code, 64, 1, 64, 3, 80, seed=6)
    rows = R.Rows((1, 3, 2), (5000, 70, 2049))
    need = C.c_size_t(0)
    dx.check(dxh.dxh_kvcache_attention_workspace_bytes(c.upload(), rows.upload(), R.DT[name], 4, C.byref(need)))
    assert need.value > 0
    a = check(dxh, c, rows, name, 4)
    b = check(dxh, c, rows, name, 4)
    assert torch.equal(a, b)
    check(dxh, c, rows, name, 4, window=700)


@pytest.mark.parametrize("size", [0.0, 30.0, 3000.0])
def test_flat_and_peaked_scores(dxh, size):
    """all scores equal; scores so large that one token takes everything"""
    c = R.Cache("i8", 32, 1, 128, 2, 10, seed=8)
    check(dxh, c, R.Rows((3, 40), (300, 64)), "f32", 2, size=size)
    check(dxh, c, R.Rows((3, 40), (300, 64)), "bf16", 2, size=size, scale=-0.1)


def test_page_scales_of_very_different_size(dxh):
    c = R.Cache("i8", 16, 1, 64, 1, 40, seed=9)
    c.vs *= np.float32(10.0) ** np.random.default_rng(1).integers(-20, 20, c.vs.shape).astype(np.float32)
    for name in ("f32", "bf16"):
        check(dxh, c, R.Rows((40,), (600,)), name, 2)
    c.vs[:] = 0  # a cache of zeros
    check(dxh, c, R.Rows((1,), (600,)), "f32", 2)


def test_without_table_or_offsets_strided_and_shared_pages(dxh):
    c = R.Cache("i8", 16, 2, 64, 3, 5, seed=10, paged=False)
    check(dxh, c, R.Rows((4,) * 3, (5, 80, 33), uniform=True), "bf16", 4)
    # a prefix that two sequences share, and the same page twice in one
    c = R.Cache("e4m3", 16, 2, 64, 2, 5, seed=11)
    c.table[1, :3] = c.table[0, :3]
    c.table[0, 4] = c.table[0, 0]
    check(dxh, c, R.Rows((2, 3), (80, 70)), "f32", 4)
    # [heads, rows, dim] views in and out, no lse
    rows = R.Rows((20, 3), (30, 70))
    q = torch.randn(4, 23, 64, device="cuda").transpose(0, 1)
    want, out = torch.empty(23, 4, 64, device="cuda"), torch.empty(4, 23, 64, device="cuda").transpose(0, 1)
    call(dxh, c.upload(), rows.upload(), "f32", q.contiguous(), want, None, 0.125, 1, 0)
    call(dxh, c.upload(), rows.upload(), "f32", q, out, None, 0.125, 1, 0)
    assert torch.equal(out, want)


def test_recorded_and_replayed_as_sequences_grow(dxh):
    """one graph of a decode step, replayed while lengths and rows change under it, with eager calls between on another stream's workspace"""
    c = R.Cache("e4m3", 16, 1, 64, 2, 200, seed=12)
    rows = R.Rows((1, 1), (100, 2500))
    cache, desc = c.upload(), rows.upload()
    q = torch.randn(2, 7, 64, device="cuda").bfloat16()
    out, lse = torch.empty_like(q), torch.empty(2, 7, device="cuda")
    st, graph = C.c_void_p(), C.c_void_p()
    dx.check(dxh.dxh_stream_create(C.byref(st)))
    need = C.c_size_t(0)
    dx.check(dxh.dxh_kvcache_attention_workspace_bytes(cache, desc, dx.BF16, 7, C.byref(need)))
    ws = torch.empty(max(1, need.value), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    dx.check(dxh.dxh_graph_begin_capture(st))
    call(dxh, cache, desc, "bf16", q, out, lse, 0.125, 1, 0, st=st, ws=ws)
    dx.check(dxh.dxh_graph_end_capture(st, C.byref(graph)))
    for step in range(4):
        rows.dev[1].copy_(torch.tensor([100 + step * 300, 2500 + 64 * step], dtype=torch.int32))
        q.copy_(torch.randn(2, 7, 64, device="cuda"))
        eager, eager_lse = torch.empty_like(out), torch.empty_like(lse)
        call(dxh, cache, desc, "bf16", q, eager, eager_lse, 0.125, 1, 0)
        out.fill_(7.0)
        torch.cuda.synchronize()
        dx.check(dxh.dxh_graph_launch(graph, st))
        dx.check(dxh.dxh_stream_sync(st))
        assert torch.equal(out, eager) and torch.equal(lse, eager_lse)
    dx.check(dxh.dxh_graph_destroy(graph))
    dx.check(dxh.dxh_stream_destroy(st))


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_as_they_are_used_together(dxh, code):
    """a prompt and then tokens one by one: rotation, cache, attention, each step against the 64-bit attention over what the cache holds, and the
    attention over the cache against the attention over unquantised keys and values (off by what 8 bits cost: a code is off by half a step of
    max|x| / 127, or by 2^-4 of a value in e4m3)"""
    hq, hk, dim, page = 6, 2, 64, 16
    c = R.Cache(code, page, hk, dim, 2, 8, seed=13)
    cache = c.upload()
    g = torch.Generator(device="cuda").manual_seed(2)
    angle = torch.arange(128, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    wq, wk = torch.randn(dim, generator=g, device="cuda"), torch.randn(dim, generator=g, device="cuda")
    have = [0, 0]
    for counts in ((37, 80), (1, 1), (1, 1), (2, 0)):
        have = [a + b for a, b in zip(have, counts)]
        rows = R.Rows(counts, have)
        desc = rows.upload()
        pos = torch.tensor([t for _, _, t in rows.each()], dtype=torch.int32, device="cuda")
        qkv = torch.randn(rows.rows, (hq + 2 * hk) * dim, generator=g, device="cuda")
        q, k, v = (t.view(rows.rows, -1, dim) for t in qkv.split([hq * dim, hk * dim, hk * dim], 1))
        part = lambda x, w: dx.NormropePart(R.heads(x), R.heads(x), dx.Heads(), w.data_ptr(), None, x.shape[1], 1, dx.F32)  # noqa: E731
        rot = dx.Rotary(cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), 128, dim, 0, dx.I32)
        dx.check(dxh.dxh_normrope(dx.F32, (dx.NormropePart * 2)(part(q, wq), part(k, wk)), 2, rows.rows, dim, 1e-6, rot, stream()))
        dx.check(dxh.dxh_kvcache_write(cache, desc, dx.F32, R.heads(k), R.heads(v), stream()))
        out = torch.empty(rows.rows, hq, dim, device="cuda")
        call(dxh, cache, desc, "f32", q, out, None, dim ** -0.5, 1, 0)
        c.k, c.v, c.ks, c.vs = c.download()
        want = R.attention(c, rows, q.double().cpu().numpy(), dim ** -0.5, 1, 0)
        for r, entry in want.items():
            assert (np.abs(out[r].double().cpu().numpy() - entry[0]) <= R.attention_bar("f32", c, entry)[0]).all()
        back = [torch.empty_like(k), torch.empty_like(v)]
        dx.check(dxh.dxh_kvcache_read(cache, desc, dx.F32, R.heads(back[0]), R.heads(back[1]), stream()))
        for b, x in zip(back, (k, v)):
            # the page's scale is from the largest value ever in it: at most that of all rows so far (unit normal rows: below 6 here; keys times their weight)
            step = 6 * max(1.0, float(wk.abs().max())) * dim ** 0.5 / 127 / 2 if code == "i8" else 0
            bound = step if code == "i8" else x.abs() * 2 ** -4 + 6 * max(1.0, float(wk.abs().max())) * dim ** 0.5 / 448 * 2 ** -10
            assert ((b - x).abs() <= bound).all()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("counts,lengths", [((1,), (1300,)), ((2,), (128,)), ((1, 3), (5000, 200)), ((40,), (1300,)), ((300,), (2600,))], ids=str)
def test_value_scales_that_are_no_float_apart(dxh, counts, lengths, page, name):
    """page scales around 2^-91 and 2^55 in one sequence, in either order and in turn, over waves, tiles and slices: the tokens of both weigh the
    same in the sum of a row, although the ratio of their scales is less than any float; and a row that does not see the large ones has the small
    ones' values in full"""
    for order in ("small first", "large first", "in turn"):
        c = R.Cache("i8", page, 1, 64, len(counts), -(-max(lengths) // page), seed=14)
        for b, n in enumerate(lengths):
            for slot in range(c.per_seq):
                large = {"small first": slot * page >= n // 2, "large first": slot * page < n // 2, "in turn": slot % 2 == 1}[order]
                c.vs[c.page_of(b, slot)] *= np.float32(2.0 ** 60 if large else 2.0 ** -86)
        check(dxh, c, R.Rows(counts, lengths), name, 3, far=92)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("vs", [0.0, 2.0 ** -100, 2.0 ** 121])
def test_sums_at_the_ends_of_the_range(dxh, vs, rows, page):
    """a row's sum holds 1 / scale of every token: many tokens of the smallest scale that a cache can have, one of the largest"""
    for length in (1, 20000) if rows == 1 else (40, 9000):
        c = R.Cache("i8", page, 1, 64, 1, -(-length // page), seed=15)
        c.vs[:] = vs
        if vs <= 2.0 ** -100:
            c.v[:] = 0  # what has that scale: a page of zeros
        else:
            c.v[:] = np.clip(c.v, -32, 32)
        check(dxh, c, R.Rows((rows,), (length,)), "bf16", 1, far=121)
        check(dxh, c, R.Rows((rows,), (length,)), "f32", 1, size=0.0, far=121)


@pytest.mark.parametrize("name,code,page,dim", [("bf16", "i8", 64, 64), ("f16", "e4m3", 128, 128), ("f32", "i8", 16, 256), ("bf16", "e4m3", 32, 80), ("f32", "e4m3", 64, 128), ("bf16", "i8", 64, 256)])
def test_one_long_sequence_in_many_slices(dxh, name, code, page, dim):
    c = R.Cache(code, page, 1, dim, 1, -(-40000 // page), seed=16)
    rows = R.Rows((2,), (39990,))
    need = C.c_size_t(0)
    dx.check(dxh.dxh_kvcache_attention_workspace_bytes(c.upload(), rows.upload(), R.DT[name], 3, C.byref(need)))
    assert need.value > 16 * 2 * 3 * (dim + 2) * 4  # more than 16 slices
    a = check(dxh, c, rows, name, 3)
    assert torch.equal(a, check(dxh, c, rows, name, 3))
    check(dxh, c, rows, name, 3, window=30000)


@pytest.mark.parametrize("name,code,page,dim,counts,lengths", [("bf16", "i8", 16, 64, (400, 130), (700, 1500)), ("f16", "e4m3", 64, 128, (130, 300), (2000, 300)), ("f32", "e4m3", 16, 64, (200,), (1000,)),
                                                             ("bf16", "e4m3", 64, 256, (130,), (2200,)), ("f32", "i8", 32, 96, (150, 3), (300, 900)), ("bf16", "i8", 128, 192, (33,), (3000,))], ids=str)
def test_prompts_in_slices(dxh, name, code, page, dim, counts, lengths):
    c = R.Cache(code, page, 1, dim, len(counts), -(-max(lengths) // page), seed=17)
    rows = R.Rows(counts, lengths, extra=1)
    a = check(dxh, c, rows, name, 2)
    assert torch.equal(a, check(dxh, c, rows, name, 2))
    check(dxh, c, rows, name, 2, window=500)
    check(dxh, c, rows, name, 2, causal=0)
    # as many tiles of rows as leave some CUs idle, with more work than the kernel for few rows is given: slices of the other one
    rows.max_rows = 255 * 128 // 2 // len(counts)
    need = C.c_size_t(0)
    dx.check(dxh.dxh_kvcache_attention_workspace_bytes(c.upload(), rows.upload(), R.DT[name], 2, C.byref(need)))
    assert need.value > 0 or max(lengths) < 600 or dim > 128
    a = check(dxh, c, rows, name, 2)
    assert torch.equal(a, check(dxh, c, rows, name, 2))
    check(dxh, c, rows, name, 2, window=500)
    check(dxh, c, rows, name, 2, causal=0)


class LargeCache(R.Cache):
    """The same cache with its pages behind `gap` others in memory, past the reach of 32-bit offsets; what lies in those is whatever was there."""

    def upload(self):
        gap = (9 << 29) // (self.heads * self.page * self.dim)  # 4.5 GiB of keys
        self.dev = [torch.empty((gap + t.shape[0], *t.shape[1:]), dtype=torch.from_numpy(t).dtype, device="cuda") for t in (self.k, self.v, self.ks, self.vs)]
        for d, t in zip(self.dev, (self.k, self.v, self.ks, self.vs)):
            d[gap:] = torch.from_numpy(t).cuda()
        self.dev_table = torch.from_numpy(np.where((self.table >= 0) & (self.table < self.pages), self.table + gap, -1).astype(np.int32)).cuda()
        return dx.KvCache(*[t.data_ptr() for t in self.dev], self.dev_table.data_ptr(), gap + self.pages, self.per_seq, self.page, self.heads, self.dim, R.CODE[self.code])


@pytest.mark.parametrize("name,code,page,dim", [("bf16", "i8", 64, 128), ("f16", "e4m3", 128, 64), ("f32", "e4m3", 64, 64), ("bf16", "e4m3", 64, 256), ("bf16", "i8", 16, 64), ("f32", "i8", 128, 80)])
def test_a_cache_past_32_bit_offsets(dxh, name, code, page, dim):
    for counts, lengths in (((1, 1, 2, 1), (5000, 64, 700, 0)), ((50, 3), (90, 400))):
        c = LargeCache(code, page, 2, dim, len(counts), -(-max(lengths) // page), seed=18, missing=[(0, 0, -1)])
        check(dxh, c, R.Rows(counts, lengths), name, 4)
        check(dxh, c, many(counts, lengths), name, 4)


@pytest.mark.parametrize("page", [16, 64])
def test_many_short_sequences(dxh, page):
    """more workgroups than the card has places for"""
    lengths = [1 + 7 * i % 200 for i in range(300)]
    check(dxh, R.Cache("i8", page, 2, 64, 300, -(-200 // page), seed=19), R.Rows((1,) * 300, lengths), "bf16", 4)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("page,dim", [(64, 64), (64, 128), (64, 256), (16, 256), (64, 80), (128, 192), (32, 128), (128, 96)])
def test_unseen_tokens_have_no_effect_at_other_sizes(dxh, page, dim, name):
    """the worst codes and scales where no row sees them, over prompts, chunks and single rows, for pages that hold a tile and heads that leave
    registers empty or are shared by two workgroups"""
    per = -(-260 // page)
    for rows in (R.Rows((50, 70, 3, 0), (230, 70, 1, 5), extra=1), R.Rows((1, 2, 1, 1), (200, 260, 0, 2 ** 31 - 1))):
        c = R.Cache("e4m3", page, 1, dim, 4, per, seed=20, missing=[(0, 1, -1), (1, 0, 1 << 30), (3, per - 1, -7)])
        seen = np.zeros((c.pages, page), bool)
        for b, r, t in rows.each():
            for j in range(0, min(t + 1, rows.lengths[b], per * page) if t >= 0 else 0):
                if c.page_of(b, j // page) >= 0:
                    seen[c.page_of(b, j // page), j % page] = True
        c.k[~np.broadcast_to(seen[:, None, :, None], c.k.shape)] = 127
        c.v[~np.broadcast_to(seen[:, None, None, :], c.v.shape)] = -1
        c.ks[~seen.any(1)] = np.nan
        c.vs[~seen.any(1)] = -np.inf
        check(dxh, c, rows, name, 3)


@pytest.mark.parametrize("page,dim", [(64, 64), (64, 256), (16, 256), (128, 192), (64, 80)])
def test_a_nan_among_values_reaches_only_rows_that_see_it(dxh, page, dim):
    c = R.Cache("e4m3", page, 1, dim, 1, -(-300 // page), seed=21)
    rows = R.Rows((120,), (290,))
    q = torch.randn(120, 2, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    clean = check(dxh, c, rows, "bf16", 2, q=q)
    for d in (0, dim - 1):
        keep = c.v.copy()
        c.v[c.page_of(0, 200 // page), 0, d, 200 % page] = 127
        out = torch.full_like(clean, 7.0)
        call(dxh, c.upload(), rows.upload(), "bf16", q.bfloat16(), out, None, dim ** -0.5, 1, 0)
        sees = torch.arange(120) + 170 >= 200
        assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees][..., d]).all()
        c.v = keep


def few(counts, lengths, extra=0):
    return R.Rows(counts, lengths, extra=extra)


# The host chooses the kernel by the rows that a sequence can have; with room for this many it is the one for many rows, whatever there is.
def many(counts, lengths, extra=0):
    return R.Rows(counts, lengths, extra=extra, max_rows=1 << 15)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", CASES + [("i8", 64, 1, 3, 64, (130, 1), (200, 70)), ("e4m3", 32, 2, 2, 128, (129, 40), (129, 300)), ("i8", 128, 1, 2, 256, (100,), (300,)), ("e4m3", 16, 1, 2, 224, (40, 90), (50, 200)),
                                          ("i8", 64, 1, 2, 96, (70,), (190,)), ("e4m3", 32, 1, 1, 256, (33,), (100,))], ids=str)
def test_ragged_many(dxh, case, name):
    code, page, hk, hq, dim, counts, lengths = case
    c = R.Cache(code, page, hk, dim, len(counts), -(-max(lengths) // page), seed=dim + hq + 1)
    check(dxh, c, many(counts, lengths, extra=1), name, hq)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("window", [0, 1, 63, 64, 65, 200])
@pytest.mark.parametrize("code,page", [("i8", 16), ("e4m3", 64)])
def test_masks_many(dxh, code, page, window, causal, name):
    c = R.Cache(code, page, 1, 64, 3, -(-320 // page), seed=window % 97 + 1)
    check(dxh, c, many((70, 1, 33), (300, 257, 33)), name, 3, causal=causal, window=window)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 64), (64, 128), (64, 256), (16, 256), (64, 80), (128, 192), (32, 128), (128, 96)])
def test_unseen_tokens_many(dxh, page, dim, name):
    per = -(-260 // page)
    for rows in (many((50, 70, 3, 0), (230, 70, 1, 5), extra=1), many((1, 2, 1, 1), (200, 260, 0, 2 ** 31 - 1))):
        c = R.Cache("e4m3", page, 1, dim, 4, per, seed=22, missing=[(0, 1, -1), (1, 0, 1 << 30), (3, per - 1, -7)])
        seen = np.zeros((c.pages, page), bool)
        for b, r, t in rows.each():
            for j in range(0, min(t + 1, rows.lengths[b], per * page) if t >= 0 else 0):
                if c.page_of(b, j // page) >= 0:
                    seen[c.page_of(b, j // page), j % page] = True
        c.k[~np.broadcast_to(seen[:, None, :, None], c.k.shape)] = 127
        c.v[~np.broadcast_to(seen[:, None, None, :], c.v.shape)] = -1
        c.ks[~seen.any(1)] = np.nan
        c.vs[~seen.any(1)] = -np.inf
        check(dxh, c, rows, name, 3)


@pytest.mark.parametrize("page,dim", [(16, 64), (64, 64), (64, 256), (16, 256), (128, 192), (64, 80)])
def test_a_nan_among_values_many(dxh, page, dim):
    c = R.Cache("e4m3", page, 1, dim, 1, -(-300 // page), seed=23)
    rows = many((120,), (290,))
    q = torch.randn(120, 2, dim, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    clean = check(dxh, c, rows, "bf16", 2, q=q)
    for d in (0, dim - 1):
        keep = c.v.copy()
        c.v[c.page_of(0, 200 // page), 0, d, 200 % page] = 127
        out = torch.full_like(clean, 7.0)
        call(dxh, c.upload(), rows.upload(), "bf16", q.bfloat16(), out, None, dim ** -0.5, 1, 0)
        sees = torch.arange(120) + 170 >= 200
        assert torch.equal(out[~sees], clean[~sees]) and torch.isnan(out[sees][..., d]).all()
        c.v = keep


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("page", [16, 64])
def test_value_scales_many(dxh, page, name):
    """scales that are no float apart, and sums at the ends of their range"""
    for order in ("small first", "large first", "in turn"):
        c = R.Cache("i8", page, 1, 64, 1, -(-1300 // page), seed=24)
        for slot in range(c.per_seq):
            large = {"small first": slot * page >= 650, "large first": slot * page < 650, "in turn": slot % 2 == 1}[order]
            c.vs[c.page_of(0, slot)] *= np.float32(2.0 ** 60 if large else 2.0 ** -86)
        check(dxh, c, many((40,), (1300,)), name, 3, far=92)
    for vs in (0.0, 2.0 ** 121):
        c = R.Cache("i8", page, 1, 64, 1, -(-9000 // page), seed=25)
        c.vs[:] = vs
        c.v[:] = 0 if vs == 0 else np.clip(c.v, -32, 32)
        check(dxh, c, many((40,), (9000,)), name, 1, size=0.0, far=121)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("code,page", [("i8", 16), ("e4m3", 64)])
@pytest.mark.parametrize("room", [few, many], ids=["few", "many"])
def test_a_scale_that_is_not_finite(dxh, room, code, page, name):
    """a page whose key or value scale is an infinity or NaN, one token in it or all: rows that see it are NaN, whatever the sign of its products, the
    others are as without it; of two key heads only its own is touched"""
    for length, counts in ((page + 1, (3,)), (2 * page + 9, (page + 20,))):
        c = R.Cache(code, page, 2, 64, 1, 3, seed=26)
        rows = room(counts, (length,))
        q = torch.rand(rows.rows, 4, 64, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") + 0.5
        p = c.page_of(0, 1)
        sees = torch.arange(length - counts[0], length) >= page
        for sign in (1.0, -1.0):  # every product of the page's keys is of this sign
            c.k[p] = R.encode(sign * (np.abs(R.decode(c.k[p], code)) + 1), 1, code)
            clean = check(dxh, c, rows, name, 4, q=q)
            for scales in (c.ks, c.vs):
                keep = scales[p, 1]
                for bad in (np.inf, -np.inf, np.nan):
                    scales[p, 1] = bad
                    out = torch.full_like(clean, 7.0)
                    call(dxh, c.upload(), rows.upload(), name, q.to(R.TT[name]), out, None, 0.125, 1, 0)
                    assert torch.equal(out[~sees], clean[~sees]) and torch.equal(out[sees][:, :2], clean[sees][:, :2]), (length, sign, bad)
                    assert torch.isnan(out[sees][:, 2:]).all(), (length, sign, bad, scales is c.ks)
                scales[p, 1] = keep


class PoolCache(R.Cache):
    """The same cache at the start of a pool of `pool` bytes of keys: what a server allocates once."""
    pool = 600 << 20

    def upload(self):
        pages = self.pool // (self.heads * self.page * self.dim)
        self.dev = [torch.empty((pages, *t.shape[1:]), dtype=torch.from_numpy(t).dtype, device="cuda") for t in (self.k, self.v, self.ks, self.vs)]
        for d, t in zip(self.dev, (self.k, self.v, self.ks, self.vs)):
            d[:t.shape[0]] = torch.from_numpy(t).cuda()
        self.dev_table = torch.from_numpy(self.table).cuda()
        return dx.KvCache(*[t.data_ptr() for t in self.dev], self.dev_table.data_ptr(), pages, self.per_seq, self.page, self.heads, self.dim, R.CODE[self.code])


class WideCache(PoolCache):
    """The same with a table so wide that its sequences could hold more codes than the last-level cache: they are read past it where pages are of 64 tokens."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        self.table, self.per_seq = np.pad(self.table, ((0, 0), (0, 1200)), constant_values=-1), self.per_seq + 1200


@pytest.mark.parametrize("code,page,dim", [("i8", 64, 128), ("e4m3", 128, 64)])
def test_the_pool_around_a_cache_changes_no_bit(dxh, code, page, dim):
    """what serves a call goes by what its rows can read: the pages of their sequences, not the pool that those are taken from"""
    args = (code, page, 2, dim, 2, 24)
    rows = R.Rows((1, 2), (24 * page, 700))
    for name in ("f32", "bf16"):
        a, b = check(dxh, R.Cache(*args, seed=27), rows, name, 6), check(dxh, PoolCache(*args, seed=27), rows, name, 6)
        assert torch.equal(a, b), name


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("room", [few, many], ids=["few", "many"])
@pytest.mark.parametrize("code,page,dim,lengths", [("i8", 16, 64, (40,)), ("e4m3", 64, 128, (100, 3000)), ("i8", 128, 80, (9000,))], ids=str)
def test_the_largest_value_scales(dxh, code, page, dim, lengths, room, name):
    """scales up to the largest float under codes that keep the values finite: their reciprocals are less than any normal float"""
    c = R.Cache(code, page, 1, dim, len(lengths), -(-max(lengths) // page), seed=28)
    small = np.sign(R.decode(c.v, code)) / 4 * (4 if code == "i8" else 1)
    c.v = R.encode(small * (np.random.default_rng(3).random(small.shape) < 0.5), 1, code)
    for low, high in ((126.0, 127.9), (100.0, 127.9), (127.9, 127.9)):
        c.vs = np.float32(2.0) ** np.random.default_rng(4).uniform(low, high, c.vs.shape).astype(np.float32)
        check(dxh, c, room((2,) * len(lengths), lengths), name, 3, far=128)


def workgroups(L, c, rows, name, q_heads):
    """of the kernel for few rows: the sequences' 16-row tiles of every key head, each as many times as the workspace holds partial results for"""
    need = C.c_size_t(0)
    dx.check(L.dxh_kvcache_attention_workspace_bytes(c.upload(), rows.upload(), R.DT[name], q_heads, C.byref(need)))
    splits = max(1, round(need.value / (rows.rows * q_heads * (c.dim + 2) * 4)))
    return len(rows.counts) * c.heads * -(-rows.max_rows * q_heads // c.heads // 16) * splits


def ragged_batch(L, name, code, page, dim, hk, kind=R.Cache):
    """40 sequences of up to 1500 tokens, whose waves walk several tiles each: missing pages, windows that begin inside a tile, the worst codes and scales
    where no row sees them, a NaN among the values of a late token"""
    hq = 2 * hk
    per = -(-1500 // page)
    lengths = [1 + 487 * i % 1500 for i in range(38)] + [1500, 1490]
    rows = R.Rows([1 + i % 2 for i in range(38)] + [2, 1], lengths, extra=1)
    c = kind(code, page, hk, dim, 40, per, seed=29, missing=[(0, 0, -1), (3, 0, 1 << 30), (38, 3, -1), (38, per - 2, -9), (39, 1, 1 << 30)])
    assert (workgroups(L, c, rows, name, hq) > 256) == (hk > 1 or kind is WideCache)
    a = check(L, c, rows, name, hq)
    assert torch.equal(a, check(L, c, rows, name, hq))
    for window, causal in ((1000, 1), (333, 0)):
        check(L, c, rows, name, hq, window=window, causal=causal)
    seen = np.zeros((c.pages, page), bool)
    for b, r, t in rows.each():
        for slot in range(-(-(t + 1) // page) if t >= 0 else 0):
            if c.page_of(b, slot) >= 0:
                seen[c.page_of(b, slot), :min(page, t + 1 - slot * page)] = True
    c.k[~np.broadcast_to(seen[:, None, :, None], c.k.shape)] = 127  # NaN in e4m3
    c.v[~np.broadcast_to(seen[:, None, None, :], c.v.shape)] = 127
    c.ks[~seen.any(1)] = np.nan
    c.vs[~seen.any(1)] = np.inf
    assert torch.equal(a, check(L, c, rows, name, hq))
    if code == "e4m3":  # the last two tokens of the longest sequence: its first row sees one of them
        first = int(rows.offsets[38])
        c.v[c.page_of(38, 1498 // page), 0, 5, 1498 % page] = -1
        c.v[c.page_of(38, 1499 // page), hk - 1, 6, 1499 % page] = 127
        out = torch.full_like(a, 7.0)
        q = torch.randn(rows.rows, hq, dim, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda").to(R.TT[name])
        call(L, c.upload(), rows.upload(), name, q, out, None, dim ** -0.5, 1, 0)
        assert torch.isnan(out[first:first + 2, :2, 5]).all() and torch.isnan(out[first + 1, hq - 2:, 6]).all()
        same = torch.ones(rows.rows, hq, dtype=torch.bool, device="cuda")
        same[first:first + 2, :2] = False
        same[first + 1, hq - 2:] = False
        assert torch.equal(out[same], a[same])


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("code,page,dim", [("i8", 16, 64), ("e4m3", 16, 128), ("e4m3", 32, 80), ("i8", 32, 128), ("i8", 64, 128), ("e4m3", 64, 64), ("i8", 128, 80), ("e4m3", 128, 128), ("i8", 64, 256), ("e4m3", 16, 192)])
def test_batches_that_fill_the_card(dxh, code, page, dim, name):
    ragged_batch(dxh, name, code, page, dim, 4)  # more workgroups than CUs


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("code,page,dim", [("e4m3", 16, 64), ("i8", 32, 80), ("e4m3", 64, 128), ("e4m3", 128, 96), ("e4m3", 32, 128)])
def test_batches_that_leave_cus_idle(dxh, code, page, dim, name):
    ragged_batch(dxh, name, code, page, dim, 1)  # eight waves a workgroup, two tiles a wave in its slice


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("code,dim,hk", [("e4m3", 64, 4), ("i8", 128, 4), ("e4m3", 128, 1), ("e4m3", 80, 2), ("i8", 256, 2), ("e4m3", 192, 1)])
def test_batches_read_past_the_last_level_cache(dxh, code, dim, hk, name):
    c = WideCache(code, 64, hk, dim, 40, 24, seed=1)
    assert min(c.pool // (hk * 64 * dim), 40 * c.per_seq) * hk * 64 * dim * 2 > 340 << 20
    ragged_batch(dxh, name, code, 64, dim, hk, WideCache)


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("code,page,dim,counts,lengths", [("i8", 16, 64, (1,), (777,)), ("e4m3", 64, 128, (1, 4, 2), (3000, 500, 64)), ("i8", 128, 80, (4,), (9000,)), ("e4m3", 32, 256, (3, 1), (900, 70))], ids=str)
def test_probabilities_of_few_rows_keep_22_bits(dxh, code, page, dim, counts, lengths, name):
    """16-bit rows differ from the 64-bit value by what f32 rows may, and by one rounding of the result"""
    c = R.Cache(code, page, 2, dim, len(counts), -(-max(lengths) // page), seed=30)
    rows = R.Rows(counts, lengths)
    q = torch.randn(rows.rows, 6, dim, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(R.TT[name])
    out = torch.empty_like(q)
    call(dxh, c.upload(), rows.upload(), name, q, out, None, dim ** -0.5, 1, 0)
    for r, entry in R.attention(c, rows, q.double().cpu().numpy(), dim ** -0.5, 1, 0).items():
        bar = R.attention_bar("f32", c, entry)[0] + np.abs(entry[0]) * R.HALF_STEP[name] * (1 + 2 ** -8) + R.TINY[name]
        worst = float((np.abs(out[r].double().cpu().numpy() - entry[0]) / bar).max())
        assert worst <= 1, (r, worst)


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_what_eight_bits_cost(dxh, code):
    """A prompt and then tokens one by one, keys five times the size of the rest: what is read back against what was written, and the attention over the
    cache against the 64-bit attention over keys and values as they were.  With s a page's scale in the end:
      int8: a code is off by s / 2, and by as much again each time its page grew, at scales of at most s; an fp32 product by 2^-24 of 127 s;
      e4m3: by 2^-4 of the value and 2^-10 s (half its smallest step, 2^-9), each time relative to what the code was before;
      attention: scores off by e = scale sum |q| dk move weights by at most exp(2 e), values by dv: |out' - out| <= max dv + (exp(2 e) - 1) sum p |v|."""
    hq, hk, dim, page = 6, 2, 64, 16
    c = R.Cache(code, page, hk, dim, 2, 8, seed=31)
    cache = c.upload()
    g = torch.Generator(device="cuda").manual_seed(4)
    have, kept, writes = [0, 0], [[[], []], [[], []]], np.zeros((2, 8), int)
    for counts in ((37, 80), (1, 1), (1, 1), (2, 0), (1, 3)):
        have = [a + b for a, b in zip(have, counts)]
        rows = R.Rows(counts, have)
        desc = rows.upload()
        q, k, v = (torch.randn(rows.rows, h, dim, generator=g, device="cuda") * size for h, size in ((hq, 0.3), (hk, 5.0), (hk, 1.0)))
        dx.check(dxh.dxh_kvcache_write(cache, desc, dx.F32, R.heads(k), R.heads(v), stream()))
        out, back = torch.empty_like(q), [torch.empty_like(k), torch.empty_like(v)]
        call(dxh, cache, desc, "f32", q, out, None, dim ** -0.5, 1, 0)
        dx.check(dxh.dxh_kvcache_read(cache, desc, dx.F32, R.heads(back[0]), R.heads(back[1]), stream()))
        c.k, c.v, c.ks, c.vs = c.download()
        for b, r, t in rows.each():
            for i, x in enumerate((k, v)):
                kept[b][i].append(x[r].double().cpu().numpy())
        for b in range(2):
            for slot in {t // page for bb, _, t in rows.each() if bb == b}:
                writes[b, slot] += 1
        off = lambda x, s, n: (n * s / 2 + s * 127 * 2 ** -23 if code == "i8" else np.abs(x) * ((1 + 2 ** -4) ** n - 1) * (1 + 2 ** -20) + n * (s * 2 ** -10) * (1 + 2 ** -4) ** n)  # noqa: E731
        got = [t.double().cpu().numpy() for t in back]
        for b, r, t in rows.each():
            for i, scales in enumerate((c.ks, c.vs)):
                x, s = kept[b][i][t], scales[c.page_of(b, t // page)].astype(np.float64)[:, None]
                assert (np.abs(got[i][r] - x) <= off(x, s, 1)).all(), (b, t, i)
        for b, r, t in rows.each():
            K, V = (np.stack(kept[b][i][:t + 1]) for i in (0, 1))
            pages, n = [c.page_of(b, j // page) for j in range(t + 1)], np.array([writes[b, j // page] for j in range(t + 1)])[:, None, None]
            dk, dv = off(K, c.ks[pages].astype(np.float64)[..., None], n), off(V, c.vs[pages].astype(np.float64)[..., None], n)
            for h in range(hq):
                qq, kh = q[r, h].double().cpu().numpy(), h // (hq // hk)
                s = K[:, kh] @ qq * dim ** -0.5
                p = np.exp(s - s.max())
                p /= p.sum()
                e = (np.abs(qq) * np.broadcast_to(dk[:, kh], K[:, kh].shape)).sum(1).max() * dim ** -0.5
                bar = np.broadcast_to(dv[:, kh], V[:, kh].shape).max(0) + (np.exp(2 * e) - 1) * (p @ np.abs(V[:, kh])) + 1e-5
                err = np.abs(out[r, h].double().cpu().numpy() - p @ V[:, kh])
                assert (err <= bar).all(), (b, t, h, float((err / bar).max()))


@pytest.mark.parametrize("name,code,page,dim", [("bf16", "i8", 16, 64), ("f32", "e4m3", 64, 128), ("f16", "i8", 128, 80), ("bf16", "e4m3", 32, 256)])
def test_a_table_wider_than_its_sequences(dxh, name, code, page, dim):
    """a table of a context limit over short sequences: the calls are planned as if they were long, and slices without tokens take no part"""
    c = R.Cache(code, page, 1, dim, 3, -(-20000 // page), seed=32)
    c.table[:, -(-800 // page):] = [[-1], [1 << 30], [-7]]
    for counts, lengths in (((1, 1, 1), (777, 1, 0)), ((3, 8, 2), (700, 8, 65)), ((40, 1, 5), (90, 800, 5))):
        rows = R.Rows(counts, lengths)
        need = C.c_size_t(0)
        dx.check(dxh.dxh_kvcache_attention_workspace_bytes(c.upload(), rows.upload(), R.DT[name], 3, C.byref(need)))
        assert need.value >= 2 * rows.rows * 3 * (dim + 2) * 4
        a = check(dxh, c, rows, name, 3)
        assert torch.equal(a, check(dxh, c, rows, name, 3))
        check(dxh, c, rows, name, 3, window=50)
        check(dxh, c, many(counts, lengths), name, 3)
