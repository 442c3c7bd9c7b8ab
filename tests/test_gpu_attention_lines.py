"""The attention operators as deepxIR lines: a decoder layer's steps between the q / k / v products and the output product, line by line, as one
datagram, recorded into a graph, held, on side streams and over UDP — the same bits every way, and those of the C ABI (which has its own tests)."""
import numpy as np
import pytest
import torch

from deepx_amd import lib as dx
from tests import helpers as H
from tests import kv_reference as R
from tests.executor_client import InProc, UdpExecutor, read_tensor, write_tensor
from tests.test_gpu_batch import Host
from tests.test_gpu_executor import fetch, load

pytestmark = pytest.mark.gpu
HQ, HK, DIM, PAGE, PAGES, BATCH, PER_SEQ = 6, 2, 64, 16, 20, 2, 8


@pytest.fixture(autouse=True)
def _torch_owns_the_hip_runtime(dxh):
    yield


def layer_lines(tag, max_rows):
    cache = "listtensor<any>:[kc vc ks vs]"
    where = f"tensor<int32>:off{tag}, tensor<int32>:len{tag}, tensor<int32>:table, var<int32>:{max_rows}"
    return [f"normrope(listtensor<bfloat16>:[q{tag} k{tag}], listtensor<bfloat16>:[wq wk], tensor<float32>:cos, tensor<float32>:sin, tensor<int32>:pos{tag}, var<float32>:1e-6, var<bool>:false)->(listtensor<bfloat16>:[qr{tag} kr{tag}])",
            f"kvcachewrite(tensor<bfloat16>:kr{tag}, tensor<bfloat16>:v{tag}, {where}, var<string>:int8)->({cache})",
            f"kvcacheattention(tensor<bfloat16>:qr{tag}, {cache}, {where}, var<float32>:0.125, var<bool>:true, var<int32>:0, var<string>:int8)->(tensor<bfloat16>:o{tag}, tensor<float32>:lse{tag})",
            f"kvcacheread({cache}, {where}, var<string>:int8)->(tensor<bfloat16>:kb{tag}, tensor<bfloat16>:vb{tag})"]


class Steps:
    """a prompt and then two single tokens of two sequences: inputs and the lines of each step"""

    def __init__(self):
        rng = np.random.default_rng(5)
        n = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        angle = np.arange(128)[:, None] * 10000.0 ** (-np.arange(DIM // 2) / (DIM // 2))
        self.common = {"cos": (np.cos(angle).astype(np.float32), "float32"), "sin": (np.sin(angle).astype(np.float32), "float32"), "table": (rng.permutation(PAGES)[:BATCH * PER_SEQ].reshape(BATCH, PER_SEQ).astype(np.int32), "int32"),
                       "wq": (H.f32_to_bf16_bits(n(DIM)), "bfloat16"), "wk": (H.f32_to_bf16_bits(n(DIM)), "bfloat16")}
        self.steps, have = [], [0, 0]
        for tag, counts in enumerate(((37, 80), (1, 1), (1, 1))):
            have = [a + b for a, b in zip(have, counts)]
            rows = R.Rows(counts, have)
            t = {f"{name}{tag}": (H.f32_to_bf16_bits(n(rows.rows, heads, DIM)), "bfloat16") for name, heads in (("q", HQ), ("k", HK), ("v", HK))}
            t[f"off{tag}"], t[f"len{tag}"] = (rows.offsets, "int32"), (np.array(have, np.int32), "int32")
            t[f"pos{tag}"] = (np.array([p for _, _, p in rows.each()], np.int32), "int32")
            out = [(f"qr{tag}", [rows.rows, HQ, DIM], "bfloat16"), (f"kr{tag}", [rows.rows, HK, DIM], "bfloat16"), (f"o{tag}", [rows.rows, HQ, DIM], "bfloat16"), (f"lse{tag}", [rows.rows, HQ], "float32"),
                   (f"kb{tag}", [rows.rows, HK, DIM], "bfloat16"), (f"vb{tag}", [rows.rows, HK, DIM], "bfloat16")]
            self.steps.append((rows, t, out, layer_lines(tag, max(counts))))
        self.cache = [("kc", [PAGES, HK, PAGE, DIM], "int8"), ("vc", [PAGES, HK, DIM, PAGE], "int8"), ("ks", [PAGES, HK], "float32"), ("vs", [PAGES, HK], "float32")]

    def names(self):
        return [o[0] for _, _, out, _ in self.steps for o in out] + [c[0] for c in self.cache]

    def new(self, name, shape, dt):
        return f"newtensor(vector<int32>:[{' '.join(str(d) for d in shape)}])->(tensor<{dt}>:{name})"


def through_the_abi(L, S):
    """the same steps through the C ABI on torch tensors"""
    dev = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a).view(np.int16) if dt == "bfloat16" else a).cuda().view(torch.bfloat16 if dt == "bfloat16" else torch.float32 if dt == "float32" else torch.int32)  # noqa: E731
    g = {k: dev(*v) for k, v in S.common.items()}
    kinds = {"int8": torch.int8, "float32": torch.float32, "bfloat16": torch.bfloat16}
    res = {name: torch.zeros(shape, dtype=kinds[dt], device="cuda") for name, shape, dt in S.cache}
    st = torch.cuda.current_stream().cuda_stream
    for tag, (rows, t, out, _) in enumerate(S.steps):
        g.update({k: dev(*v) for k, v in t.items()})
        res.update({name: torch.zeros(shape, dtype=kinds[dt], device="cuda") for name, shape, dt in out})
        cache = dx.KvCache(res["kc"].data_ptr(), res["vc"].data_ptr(), res["ks"].data_ptr(), res["vs"].data_ptr(), g["table"].data_ptr(), PAGES, PER_SEQ, PAGE, HK, DIM, dx.I8)
        desc = dx.KvRows(g[f"off{tag}"].data_ptr(), g[f"len{tag}"].data_ptr(), rows.rows, BATCH, rows.max_rows)
        part = lambda x, y, w: dx.NormropePart(R.heads(g[f"{x}{tag}"]), R.heads(res[f"{y}{tag}"]), dx.Heads(), g[w].data_ptr(), None, g[f"{x}{tag}"].shape[1], 1, dx.BF16)  # noqa: E731, B023
        rot = dx.Rotary(g["cos"].data_ptr(), g["sin"].data_ptr(), g[f"pos{tag}"].data_ptr(), 128, DIM, 0, dx.I32)
        dx.check(L.dxh_normrope(dx.BF16, (dx.NormropePart * 2)(part("q", "qr", "wq"), part("k", "kr", "wk")), 2, rows.rows, DIM, 1e-6, rot, st))
        dx.check(L.dxh_kvcache_write(cache, desc, dx.BF16, R.heads(res[f"kr{tag}"]), R.heads(g[f"v{tag}"]), st))
        ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
        dx.check(L.dxh_kvcache_attention(cache, desc, dx.BF16, HQ, R.heads(res[f"qr{tag}"]), R.heads(res[f"o{tag}"]), res[f"lse{tag}"].data_ptr(), 0.125, 1, 0, ws.data_ptr(), ws.numel(), st))
        dx.check(L.dxh_kvcache_read(cache, desc, dx.BF16, R.heads(res[f"kb{tag}"]), R.heads(res[f"vb{tag}"]), st))
    return {k: res[k].cpu().view(torch.int16 if res[k].dtype == torch.bfloat16 else res[k].dtype).numpy() for k in S.names()}


@pytest.fixture(scope="module")
def steps():
    return Steps()


@pytest.fixture(scope="module")
def want(dxh, steps):
    return through_the_abi(dxh, steps)


def same(got, want):
    for name, w in want.items():
        g = got[name]
        assert np.array_equal(g.reshape(-1).view(np.int8), w.reshape(-1).view(np.int8)), name


@pytest.mark.parametrize("mode", ["line by line", "datagram", "deferred", "streams", "driver storage"])
def test_every_way_gives_the_bits_of_the_abi(steps, want, tmp_path, mode):
    ex = InProc()
    try:
        ex.set_pool(mode != "driver storage")
        h = Host(ex, tmp_path)
        if mode == "deferred":
            ex.set_defer(True)
        if mode == "streams":
            ex.set_streams(3)
        for name, (arr, dt) in steps.common.items():
            h.put(name, arr, dt)
        for c in steps.cache:
            h.run(steps.new(*c))
        for rows, t, out, lines in steps.steps:
            for name, (arr, dt) in t.items():
                h.put(name, arr, dt)
            lines = [steps.new(*o) for o in out] + lines
            if mode == "datagram":
                assert all(" ok//" in r for r in ex.execute_batch([f"{x} // id={i + 1}" for i, x in enumerate(lines)]))
            else:
                for x in lines:
                    h.run(x)
        ex.flush()
        same({n: h.get(n) for n in steps.names()}, want)
    finally:
        ex.set_pool(True)
        ex.close()


def test_recorded_into_a_graph_and_replayed(steps, want, tmp_path):
    """the prompt's lines as a datagram, recorded on its second arrival; a write that is repeated changes nothing, and each replay comes after a new prompt
    in the same tensors and eager work of the same executor between"""
    ex = InProc()
    try:
        ex.set_graphs(True)
        h = Host(ex, tmp_path)
        rows, t, out, lines = steps.steps[0]
        for name, (arr, dt) in {**steps.common, **t}.items():
            h.put(name, arr, dt)
        for c in steps.cache + out:
            h.run(steps.new(*c))
        rng = np.random.default_rng(9)
        for turn in range(5):
            size = 1.0 + turn
            if turn:  # loadtensordata keeps the tensors where they are
                for name in ("q0", "k0", "v0"):
                    p = str(tmp_path / f"{name}_{turn}")
                    write_tensor(p, H.f32_to_bf16_bits(rng.standard_normal(t[name][0].shape).astype(np.float32) * size), "bfloat16")
                    h.run(f"loadtensordata(var<string>:{p}.data)->(tensor<bfloat16>:{name})")
            assert all(" ok//" in r for r in ex.execute_batch([f"{x} // id={i + 1}" for i, x in enumerate(lines)]))
            graph = {n: h.get(n) for n in [o[0] for o in out] + [c[0] for c in steps.cache]}
            for x in lines:
                h.run(x)
            same({n: h.get(n) for n in graph}, graph)
            if turn == 0:
                same({n: graph[n] for n in ("qr0", "kr0", "o0", "lse0", "kb0", "vb0")}, {n: want[n] for n in ("qr0", "kr0", "o0", "lse0", "kb0", "vb0")})
        assert ex.stats()["replays"] >= 3
    finally:
        ex.close()


def test_gradients_and_rope_over_udp(dxh, tmp_path):
    srv = UdpExecutor()
    try:
        rng = np.random.default_rng(3)
        rows, h, dim = 33, 3, 32
        x, dy, w = (rng.standard_normal(s).astype(np.float32) for s in ((rows, h, dim), (rows, h, dim), (dim,)))
        a = rng.uniform(0, 6, (50, dim // 2))
        cos, sin, pos = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32), rng.integers(0, 50, rows)
        for name, arr, dt in (("x", x, "float32"), ("dy", dy, "float32"), ("w", w, "float32"), ("cos", cos, "float32"), ("sin", sin, "float32"), ("pos", pos, "int64")):
            load(srv, tmp_path, name, arr, dt)
        for name, shape in (("dx", "[33 3 32]"), ("dw", "[32]"), ("y", "[33 3 32]"), ("n", "[33 3 32]")):
            srv.must("newtensor", [f"vector<int32>:{shape}"], [f"tensor<float32>:{name}"], author="")
        tables = ["tensor<float32>:cos", "tensor<float32>:sin", "tensor<int64>:pos"]
        srv.must("normropebackward", ["listtensor<float32>:[x]", "listtensor<float32>:[dy]", "listtensor<float32>:[w]", *tables, "var<float32>:1e-6", "var<bool>:true"], ["listtensor<float32>:[dx]", "listtensor<float32>:[dw]"])
        srv.must("rope", ["listtensor<float32>:[x]", *tables, "var<bool>:false"], ["listtensor<float32>:[y]"])
        srv.must("normrope", ["listtensor<float32>:[x]", "listtensor<float32>:[w]", *tables, "var<float32>:1e-6", "var<bool>:true"], ["listtensor<float32>:[n]"])
        t = {k: torch.from_numpy(v).cuda() for k, v in (("x", x), ("dy", dy), ("w", w), ("cos", cos), ("sin", sin), ("pos", pos))}
        got = {k: torch.empty(rows, h, dim, device="cuda") for k in ("dx", "y", "n")}
        got["dw"] = torch.empty(dim, device="cuda")
        st, ws = torch.cuda.current_stream().cuda_stream, torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
        rot = lambda inter: dx.Rotary(t["cos"].data_ptr(), t["sin"].data_ptr(), t["pos"].data_ptr(), 50, dim, inter, dx.I64)  # noqa: E731
        one = lambda *p: (dx.NormropePart * 1)(dx.NormropePart(*p))  # noqa: E731
        dx.check(dxh.dxh_normrope_backward(dx.F32, one(R.heads(t["x"]), R.heads(t["dy"]), R.heads(got["dx"]), t["w"].data_ptr(), got["dw"].data_ptr(), h, 1, dx.F32), 1, rows, dim, 1e-6, rot(1), ws.data_ptr(), ws.numel(), st))
        dx.check(dxh.dxh_normrope(dx.F32, one(R.heads(t["x"]), R.heads(got["y"]), dx.Heads(), None, None, h, 0, 0), 1, rows, dim, 0.0, rot(0), st))
        dx.check(dxh.dxh_normrope(dx.F32, one(R.heads(t["x"]), R.heads(got["n"]), dx.Heads(), t["w"].data_ptr(), None, h, 1, dx.F32), 1, rows, dim, 1e-6, rot(1), st))
        for name, g in got.items():
            assert np.array_equal(fetch(srv, tmp_path, name)[0].view(np.int32), g.cpu().numpy().view(np.int32)), name
    finally:
        srv.close()


def test_lines_that_are_refused(tmp_path):
    """wrong ranks, dtypes, lists and sizes are error replies, and the executor goes on"""
    ex = InProc()
    try:
        h = Host(ex, tmp_path)
        for name, shape, dt in (("q", [4, 6, 64], "float32"), ("k", [4, 2, 64], "float32"), ("v", [4, 2, 64], "float32"), ("flat", [4, 64], "float32"), ("h16", [4, 2, 64], "float16"), ("w", [64], "float32"), ("w2", [32], "float32"),
                                ("cos", [8, 32], "float32"), ("sin", [8, 32], "float32"), ("pos", [4], "int32"), ("pos3", [3], "int32"), ("kc", [4, 2, 16, 64], "int8"), ("vc", [4, 2, 64, 16], "int8"), ("ks", [4, 2], "float32"),
                                ("vs", [4, 2], "float32"), ("off", [3], "int32"), ("len", [2], "int32"), ("table", [2, 2], "int32"), ("o", [4, 6, 64], "float32")):
            h.run(f"newtensor(vector<int32>:[{' '.join(map(str, shape))}])->(tensor<{dt}>:{name})")

        def refused(line, why):
            r = ex.execute(line)
            assert " error//" in r and why in r, r

        tab = "tensor<float32>:cos, tensor<float32>:sin, tensor<int32>:pos, "
        nr = lambda xs, ws, ys, tab=tab: f"normrope(listtensor<any>:[{xs}], listtensor<any>:[{ws}], {tab}var<float32>:1e-6, var<bool>:false)->(listtensor<any>:[{ys}])"  # noqa: E731
        refused(nr("flat", "w", "flat"), "must be a [rows, heads, dim]")
        refused(nr("q k", "w", "q k"), "as many of each list")
        refused(nr("q", "w2", "q"), "a weight must hold")
        refused(nr("k", "w", "q"), "must have one dtype and shape")
        refused(nr("k h16", "w w", "k h16"), "agree in dtype")
        refused(nr("k v", "w w", "v k"), "normrope")
        refused(nr("k", "w", "nothere"), "tensor not found")
        refused(nr("k", "w", "k", tab.replace(":pos", ":pos3")), "one entry a row")
        refused(nr("k", "w", "k", tab.replace(":sin", ":w")), "sin must be")
        where = "tensor<int32>:off, tensor<int32>:len, tensor<int32>:table, var<int32>:2, "
        wr = lambda k="k", v="v", where=where, code="int8", cache="kc vc ks vs": f"kvcachewrite(tensor<any>:{k}, tensor<any>:{v}, {where}var<string>:{code})->(listtensor<any>:[{cache}])"  # noqa: E731
        refused(wr(code="int4"), "code must be")
        refused(wr(cache="kc vc ks"), "a cache is four tensors")
        refused(wr(cache="vc kc ks vs"), "rows must have the cache's 2 heads and head size 16")
        refused(wr(cache="q vc ks vs"), "cached keys must be int8")
        refused(wr(k="q", v="q"), "rows must have the cache's")
        refused(wr(k="h16"), "Type mismatch")
        refused(wr(where=where.replace(":off", ":len")), "offsets must hold")
        refused(wr(where=where.replace(":table", ":off")), "the page table must be")
        at = lambda q="q", o="o", window="0", causal="true": f"kvcacheattention(tensor<any>:{q}, listtensor<any>:[kc vc ks vs], {where}var<float32>:0.1, var<bool>:{causal}, var<int32>:{window}, var<string>:int8)->(tensor<any>:{o})"  # noqa: E731
        refused(at(o="q"), "in place")
        refused(at(o="k"), "shape mismatch")
        refused(at(window="-1"), "kvcacheattention")
        refused(at(causal="maybe"), "Invalid bool")
        refused(f"kvcacheread(listtensor<any>:[kc vc ks vs], {where}var<string>:int8)->(tensor<any>:k, tensor<any>:k)", "kvcacheread")
        h.run(wr())
        h.run(at())
        assert not h.get("o").any()  # no sequence has rows: offsets are zeros
    finally:
        ex.close()


def test_results_that_are_other_inputs_are_refused(tmp_path):
    """a line whose result is also its weight, another part's, a gradient's other result or a scale of the cache"""
    ex = InProc()
    try:
        h = Host(ex, tmp_path)
        for name, shape, dt in (("x", [1, 1, 64], "float32"), ("x2", [1, 1, 64], "float32"), ("w", [1, 1, 64], "float32"), ("w2", [64], "float32"), ("g", [1, 1, 64], "float32"), ("y", [1, 1, 64], "float32"),
                                ("cos", [8, 32], "float32"), ("sin", [8, 32], "float32"), ("pos", [1], "int32"), ("q", [4, 2, 64], "float32"), ("o", [4, 2, 64], "float32"), ("kc", [4, 2, 16, 64], "int8"),
                                ("vc", [4, 2, 64, 16], "int8"), ("ks", [4, 2], "float32"), ("vs", [4, 2], "float32"), ("off", [3], "int32"), ("len", [2], "int32"), ("table", [2, 2], "int32")):
            h.run(f"newtensor(vector<int32>:[{' '.join(map(str, shape))}])->(tensor<{dt}>:{name})")
        tab = "tensor<float32>:cos, tensor<float32>:sin, tensor<int32>:pos, var<float32>:1e-6, var<bool>:false"
        nr = lambda xs, ws, ys: f"normrope(listtensor<any>:[{xs}], listtensor<any>:[{ws}], {tab})->(listtensor<any>:[{ys}])"  # noqa: E731
        back = lambda dxs, dws: f"normropebackward(listtensor<any>:[x], listtensor<any>:[g], listtensor<any>:[w], {tab})->(listtensor<any>:[{dxs}], listtensor<any>:[{dws}])"  # noqa: E731
        at = lambda lse: ("kvcacheattention(tensor<any>:q, listtensor<any>:[kc vc ks vs], tensor<int32>:off, tensor<int32>:len, tensor<int32>:table, var<int32>:2, var<float32>:0.1, var<bool>:true, var<int32>:0, "  # noqa: E731
                          f"var<string>:int8)->(tensor<any>:o, tensor<float32>:{lse})")
        for line in (nr("x", "w", "w"), nr("x x2", "w w2", "y w"), back("w", "w2"), back("y", "y"), at("ks"), at("vs")):
            assert " error//" in ex.execute(line), line
        h.run(nr("x x2", "w w2", "x y"))
        h.run(back("g", "w2"))
    finally:
        ex.close()
