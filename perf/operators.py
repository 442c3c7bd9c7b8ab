"""The attention operators over an 8-bit cache, as they are measured: cases, inputs, plain forms, values in 64 bits.

Operators:
  normrope            RMS norm of every query and key head and the position rotation, one pass over a row's heads
  normrope_backward   its gradients: inputs and both weights
  kvcache_write       new keys and values into a paged cache of 8-bit codes with one scale for each (page, head)
  kvcache_read        the codes of a sequence's last tokens back as values
  kvcache_attention   attention of a ragged batch of rows over that cache, from one row a sequence to whole prompts

Packed rows: the rows of sequence b are offsets[b] .. offsets[b+1]-1 of a [rows, heads, dim] tensor and are the last tokens of the
lengths[b] that the sequence has in the cache.  Codes: int8, or float8 e4m3.  Keys lie [page, head, token, dim], values
[page, head, dim, token].
"""
import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CODES = {"int8": torch.int8, "float8e4m3": torch.float8_e4m3fn}
CODE_MAX = {"int8": 127.0, "float8e4m3": 448.0}
CODE_INV = {"int8": 0.007874015718698502, "float8e4m3": 0.0022321429569274187}  # 1/127 and 1/448 in 32 bits
SCALE_MIN = 2.0 ** -100
FLT_MAX = 3.4028234663852886e38
EPS = 1e-6


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of eight sequences of the 14 + 2 heads of 64 that make the 896 wide rows of the decoder block
        {"name": "normrope decode", "op": "normrope", "dtype": "bfloat16", "rows": 8, "q_heads": 14, "kv_heads": 2, "dim": 64, "rotary": 64, "interleaved": False, "table": 4096},
        # the prompts of a batch, rows 4096 wide
        {"name": "normrope prompts", "op": "normrope", "dtype": "bfloat16", "rows": 16384, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "table": 32768},
        # a training step of the small block in 32 bits, half of each head rotated in neighbouring pairs
        {"name": "normrope backward small", "op": "normrope_backward", "dtype": "float32", "rows": 2047, "q_heads": 14, "kv_heads": 2, "dim": 64, "rotary": 32, "interleaved": True, "table": 2048},
        # a training step's sequences, rows 4096 wide
        {"name": "normrope backward large", "op": "normrope_backward", "dtype": "bfloat16", "rows": 8192, "q_heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128, "interleaved": False, "table": 8192},
        # one new token of each of 64 sequences: most pages hold older tokens whose scale may have to grow
        {"name": "write decode", "op": "kvcache_write", "dtype": "bfloat16", "code": "float8e4m3", "batch": 64, "len_min": 1, "len_max": 4096, "new_max": 1, "kv_heads": 8, "dim": 128, "page": 16},
        # whole ragged prompts in 32 bits
        {"name": "write prompts", "op": "kvcache_write", "dtype": "float32", "code": "int8", "batch": 32, "len_min": 333, "len_max": 2048, "new_max": 2048, "kv_heads": 2, "dim": 64, "page": 64},
        # a few sequences moved out of the cache
        {"name": "read few", "op": "kvcache_read", "dtype": "float32", "code": "int8", "batch": 5, "len_min": 17, "len_max": 777, "new_max": 777, "kv_heads": 2, "dim": 64, "page": 16},
        # a whole cache read back
        {"name": "read all", "op": "kvcache_read", "dtype": "bfloat16", "code": "float8e4m3", "batch": 16, "len_min": 6000, "len_max": 8192, "new_max": 8192, "kv_heads": 8, "dim": 128, "page": 64},
        # one user, one token: latency
        {"name": "attention one", "op": "kvcache_attention", "dtype": "bfloat16", "code": "int8", "batch": 1, "len_min": 777, "len_max": 777, "new_max": 1, "q_heads": 14, "kv_heads": 2, "dim": 64, "page": 16, "causal": True, "window": 0},
        # a serving batch, one token each, ragged lengths
        {"name": "attention batch", "op": "kvcache_attention", "dtype": "bfloat16", "code": "float8e4m3", "batch": 64, "len_min": 1024, "len_max": 16384, "new_max": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0},
        # one long sequence, four tokens checked at once
        {"name": "attention long", "op": "kvcache_attention", "dtype": "float16", "code": "int8", "batch": 1, "len_min": 131071, "len_max": 131071, "new_max": 4, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "causal": True, "window": 0},
        # prompts of up to 4096 tokens, causal
        {"name": "attention prompts", "op": "kvcache_attention", "dtype": "bfloat16", "code": "float8e4m3", "batch": 4, "len_min": 3333, "len_max": 4096, "new_max": 4096, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "causal": True, "window": 0},
    ]


def draw(rng):
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    op = rng.choice(["normrope", "normrope_backward", "kvcache_write", "kvcache_read", "kvcache_attention", "kvcache_attention"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    q_heads = kv_heads * rng.choice([1, 2, 4, 5, 7])
    if op.startswith("normrope"):
        most = 16384 * 40 * 128 if op == "normrope" else 8192 * 40 * 128
        size = 2 if dtype == "float32" else 1
        rows = min(log(1, 16384), most // ((q_heads + kv_heads) * dim * size))
        return {"op": op, "dtype": dtype, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotary": rng.choice([dim, dim, dim // 2]), "interleaved": rng.random() < 0.3, "table": 32768}
    case = {"op": op, "dtype": dtype, "code": rng.choice(["int8", "float8e4m3"]), "kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 32, 64, 128])}
    if op == "kvcache_attention":
        kind = rng.choice(["decode", "few", "prompt"])
        if kind == "prompt":
            longest = log(32, 2048)
            batch, new = max(1, min(8, 4096 // longest)), longest
        else:
            longest = log(16, 65536)
            batch, new = max(1, min(log(1, 64), (1 << 18) // longest)), 1 if kind == "decode" else rng.choice([2, 3, 5, 8])
        return {**case, "batch": batch, "len_min": max(1, int(longest * rng.random())), "len_max": longest, "new_max": min(new, longest), "q_heads": q_heads,
                "causal": rng.random() < 0.8, "window": rng.choice([0, 0, 0, log(16, 4096)])}
    longest = log(16, 8192)
    batch = max(1, min(log(1, 64), (1 << 16) // longest))
    return {**case, "batch": batch, "len_min": max(1, int(longest * rng.random())), "len_max": longest, "new_max": rng.choice([1, min(longest, 77), longest])}


def lengths_of(case):
    """Each sequence's tokens in the cache and its new rows: spread evenly over the case's range, the longest first."""
    n, lo, hi = case["batch"], case["len_min"], case["len_max"]
    lengths = [hi if b == 0 else lo + int((hi - lo + 1) * (b * 0.6180339887498949 % 1.0)) for b in range(n)]
    return lengths, [min(case["new_max"], length) for length in lengths]


def work(case):
    e = 4 if case["dtype"] == "float32" else 2
    if case["op"].startswith("normrope"):
        n = case["rows"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        back = case["op"] != "normrope"
        table = 2 * 4 * min(case["rows"], case["table"]) * (case["rotary"] // 2)
        return {"bytes": (3 if back else 2) * n * e + table, "flops": (18 if back else 10) * n}
    lengths, news = lengths_of(case)
    head = case["kv_heads"] * case["dim"]
    if case["op"] == "kvcache_write" or case["op"] == "kvcache_read":
        return {"bytes": 2 * sum(news) * head * (e + 1), "flops": 4 * sum(news) * head}
    seen = pairs = 0
    for length, new in zip(lengths, news):
        window = case["window"] or length
        first = max(0, length - new - window + 1) if case["window"] else 0
        seen += length - first
        for i in {0, new - 1} if new > 1 else {0}:
            p = length - new + i
            visible = (p + 1 if case["causal"] else length) - max(0, p - window + 1)
            pairs += visible * new / (2 if new > 1 else 1)
    return {"bytes": 2 * seen * head + 2 * sum(news) * case["q_heads"] * case["dim"] * e, "flops": 4 * pairs * case["q_heads"] * case["dim"]}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    s = dict(case)
    dim, hk = case["dim"], case["kv_heads"]
    if case["op"].startswith("normrope"):
        rows, hq, rd = case["rows"], case["q_heads"], case["rotary"]
        # the rows of one product q | k | v, as it leaves them: query and key heads are views of it
        qkv = (normal(rows, (hq + 2 * hk) * dim) * 1.5).to(dtype)
        s["q"], s["k"] = qkv[:, :hq * dim].view(rows, hq, dim), qkv[:, hq * dim:(hq + hk) * dim].view(rows, hk, dim)
        s["wq"], s["wk"] = (1 + 0.2 * normal(dim)).to(dtype), (1 + 0.2 * normal(dim)).to(dtype)
        angle = torch.arange(case["table"], device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(rd // 2, device=dev, dtype=torch.float64) * 2 / rd)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["positions"] = torch.randint(0, case["table"], (rows,), generator=g, device=dev, dtype=torch.int32)
        s["q_out"], s["k_out"] = torch.empty(rows, hq, dim, device=dev, dtype=dtype), torch.empty(rows, hk, dim, device=dev, dtype=dtype)
        if case["op"] == "normrope_backward":
            s["dq"], s["dk"] = normal(rows, hq, dim).to(dtype), normal(rows, hk, dim).to(dtype)
            s["dwq"], s["dwk"] = torch.empty(dim, device=dev), torch.empty(dim, device=dev)
            s["scratch"] = torch.empty(4 << 20, device=dev, dtype=torch.uint8)
        return s
    batch, page, code = case["batch"], case["page"], case["code"]
    lengths, news = lengths_of(case)
    per_seq = -(-max(lengths) // page)
    used = [-(-n // page) for n in lengths]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((batch, per_seq), -1, device=dev, dtype=torch.int32)
    at = 0
    for b in range(batch):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
    s["table"], s["pages"], s["per_seq"] = table, pages, per_seq
    s["host_lengths"], s["host_news"] = lengths, news
    s["lengths"] = torch.tensor(lengths, device=dev, dtype=torch.int32)
    s["offsets"] = torch.tensor([sum(news[:b]) for b in range(batch + 1)], device=dev, dtype=torch.int32)
    s["rows"], s["max_rows"] = sum(news), max(news)
    # what the cache holds: normal values, each page and head with a scale of its own
    spread = 32.0 if code == "int8" else 100.0
    codes = lambda *shape: (normal(*shape) * spread).round_().clamp_(-CODE_MAX[code], CODE_MAX[code]).to(CODES[code])  # noqa: E731
    s["kc"], s["vc"] = codes(pages, hk, page, dim), codes(pages, hk, dim, page)
    s["ks"], s["vs"] = ((0.5 + torch.rand(pages, hk, generator=g, device=dev)) / spread for _ in range(2))
    if case["op"] == "kvcache_attention":
        s["q"] = normal(s["rows"], case["q_heads"], dim).to(dtype)
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = dim ** -0.5
        s["scratch"] = torch.empty(256 << 20, device=dev, dtype=torch.uint8)
    else:
        s["k"], s["v"] = normal(s["rows"], hk, dim).to(dtype), normal(s["rows"], hk, dim).to(dtype)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return OWN[s["op"]](s)
    return PLAIN[s["op"]](s)


def _rotate(n, cos, sin, rd, interleaved, back):
    """`n` [rows, heads, dim] in 32 bits, rotated by cos / sin [rows, 1, rd/2], or back."""
    if back:
        sin = -sin
    head, rest = n[..., :rd], n[..., rd:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = head[..., :rd // 2], head[..., rd // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def plain_normrope(s):
    p = s["positions"].long()
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]

    def one(x, w):
        x = x.float()
        n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
        return _rotate(n, cos, sin, s["rotary"], s["interleaved"], False).to(s["q"].dtype)

    return {"q": one(s["q"], s["wq"]), "k": one(s["k"], s["wk"])}


def plain_normrope_backward(s):
    p = s["positions"].long()
    cos, sin = s["cos"][p][:, None], s["sin"][p][:, None]

    def one(x, dy, w):
        x = x.float()
        g = _rotate(dy.float(), cos, sin, s["rotary"], s["interleaved"], True)
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        h = g * w.float()
        dx = r * h - x * (r * r * r * (h * x).mean(-1, keepdim=True))
        return dx.to(s["q"].dtype), (g * x * r).sum((0, 1))

    dq, dwq = one(s["q"], s["dq"], s["wq"])
    dk, dwk = one(s["k"], s["dk"], s["wk"])
    return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _rows_of(s):
    """Sequence and position of each packed row."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["offsets"][1:].long(), row, right=True)
    return seq, s["lengths"].long()[seq] - (s["offsets"].long()[seq + 1] - row)


def _encode(x, inv, code):
    x = (x * inv).clamp(-CODE_MAX[code], CODE_MAX[code])
    return (x.round() if code == "int8" else x).to(CODES[code])


def plain_write(s):
    page, code = s["page"], s["code"]
    seq, pos = _rows_of(s)
    slot = pos // page
    place = s["table"].long()[seq, slot]
    # a page that the first new row starts inside of holds older tokens; every other touched page starts new
    first = (s["lengths"] - (s["offsets"][1:] - s["offsets"][:-1])).long()
    border = s["table"].long().gather(1, (first // page)[:, None])[:, 0]
    old = torch.zeros(s["pages"], dtype=torch.long, device="cuda")
    old[border] = first % page

    def one(x, codes, scales, across):
        x = x.float()
        a = x.abs().amax(-1).clamp(max=FLT_MAX)
        top = torch.zeros_like(scales).scatter_reduce(0, place[:, None].expand_as(a), a, "amax")
        touched = torch.zeros(s["pages"], dtype=torch.bool, device="cuda")
        touched[place] = True
        new = (top * CODE_INV[code]).clamp(min=SCALE_MIN)
        kept = (old > 0)[:, None]
        new = torch.where(kept, torch.maximum(new, scales), new)
        new = torch.where(touched[:, None], new, scales)
        factor = (scales * (1 / new))[border][:, :, None, None]
        older = (torch.arange(page, device="cuda") < (first % page)[:, None])[:, None]
        older = (older[..., None, :] if across else older[..., None]) & (new > scales)[border][:, :, None, None]
        before = codes[border].float()
        codes[border] = torch.where(older, _encode(before, factor, code).float(), before).to(CODES[code])
        fresh = _encode(x, (1 / new)[place][..., None], code)
        raw, bits = codes.view(torch.int8), fresh.view(torch.int8)
        if across:
            raw[place, :, :, pos % page] = bits
        else:
            raw[place, :, pos % page] = bits
        scales.copy_(new)

    one(s["k"], s["kc"], s["ks"], False)
    one(s["v"], s["vc"], s["vs"], True)
    return {"k": s["kc"], "v": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}


def plain_read(s):
    page = s["page"]
    seq, pos = _rows_of(s)
    place = s["table"].long()[seq, pos // page]
    k = s["kc"].view(torch.int8)[place, :, pos % page].view(CODES[s["code"]]).float() * s["ks"][place][..., None]
    v = s["vc"].view(torch.int8)[place, :, :, pos % page].view(CODES[s["code"]]).float() * s["vs"][place][..., None]
    return {"k": k.to(s["k"].dtype), "v": v.to(s["v"].dtype)}


def plain_attention(s):
    batch, hk, dim, page = s["batch"], s["kv_heads"], s["dim"], s["page"]
    group, most, total = s["q_heads"] // hk, s["max_rows"], s["per_seq"] * page
    t = s["table"].long().clamp(min=0)
    k = (s["kc"].view(torch.int8)[t].view(CODES[s["code"]]).float() * s["ks"][t][..., None, None]).permute(0, 2, 1, 3, 4).reshape(batch, hk, total, dim)
    v = (s["vc"].view(torch.int8)[t].view(CODES[s["code"]]).float() * s["vs"][t][..., None, None]).permute(0, 2, 1, 4, 3).reshape(batch, hk, total, dim)
    seq, pos = _rows_of(s)
    at = torch.arange(s["rows"], device="cuda") - s["offsets"].long()[seq]
    q = torch.zeros(batch, most, hk, group, dim, device="cuda")
    q[seq, at] = s["q"].float().view(-1, hk, group, dim)
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).reshape(batch, hk, group * most, dim), k.transpose(-1, -2)).view(batch, hk, group, most, total)
    token = torch.arange(total, device="cuda")
    position = torch.full((batch, most), -1, device="cuda", dtype=torch.long)
    position[seq, at] = pos
    seen = (token < s["lengths"][:, None, None]) & (position[..., None] >= 0)
    if s["causal"]:
        seen = seen & (token <= position[..., None])
    if s["window"]:
        seen = seen & (token > position[..., None] - s["window"])
    score = (score * s["scale"]).masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == float("-inf"), 0.0, top)).exp_()
    total_p = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(batch, hk, group * most, total), v).view(batch, hk, group, most, dim)
    out = out / torch.where(total_p == 0, 1.0, total_p)
    return out.permute(0, 3, 1, 2, 4)[seq, at].reshape(s["q"].shape).to(s["q"].dtype)


PLAIN = {"normrope": plain_normrope, "normrope_backward": plain_normrope_backward, "kvcache_write": plain_write, "kvcache_read": plain_read, "kvcache_attention": plain_attention}


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _heads(dx, t):
    return dx.Heads(t.data_ptr(), t.stride(0), t.stride(1))


def _rotary(dx, s):
    return dx.Rotary(s["cos"].data_ptr(), s["sin"].data_ptr(), s["positions"].data_ptr(), s["table"], s["rotary"], int(s["interleaved"]), dx.I32)


def own_normrope(s):
    from deepx_amd import lib as dx
    dt = {"float32": dx.F32, "float16": dx.F16, "bfloat16": dx.BF16}[s["dtype"]]
    part = lambda x, y, w: dx.NormropePart(_heads(dx, s[x]), _heads(dx, s[y]), dx.Heads(), s[w].data_ptr(), None, s[x].shape[1], 1, dt)  # noqa: E731
    parts = (dx.NormropePart * 2)(part("q", "q_out", "wq"), part("k", "k_out", "wk"))
    dx.check(dx.load().dxh_normrope(dt, parts, 2, s["rows"], s["dim"], EPS, _rotary(dx, s), _stream()), "normrope")
    return {"q": s["q_out"], "k": s["k_out"]}


def own_normrope_backward(s):
    from deepx_amd import lib as dx
    dt = {"float32": dx.F32, "float16": dx.F16, "bfloat16": dx.BF16}[s["dtype"]]
    part = lambda x, dy, out, w, dw: dx.NormropePart(_heads(dx, s[x]), _heads(dx, s[dy]), _heads(dx, s[out]), s[w].data_ptr(), s[dw].data_ptr(), s[x].shape[1], 1, dt)  # noqa: E731
    parts = (dx.NormropePart * 2)(part("q", "dq", "q_out", "wq", "dwq"), part("k", "dk", "k_out", "wk", "dwk"))
    dx.check(dx.load().dxh_normrope_backward(dt, parts, 2, s["rows"], s["dim"], EPS, _rotary(dx, s), s["scratch"].data_ptr(), s["scratch"].numel(), _stream()), "normrope_backward")
    return {"dq": s["q_out"], "dk": s["k_out"], "dwq": s["dwq"], "dwk": s["dwk"]}


def _cache(dx, s):
    return (dx.KvCache(s["kc"].data_ptr(), s["vc"].data_ptr(), s["ks"].data_ptr(), s["vs"].data_ptr(), s["table"].data_ptr(), s["pages"], s["per_seq"], s["page"], s["kv_heads"], s["dim"],
                       dx.I8 if s["code"] == "int8" else dx.F8E4M3),
            dx.KvRows(s["offsets"].data_ptr(), s["lengths"].data_ptr(), s["rows"], s["batch"], s["max_rows"]))


def own_write(s):
    from deepx_amd import lib as dx
    dt = {"float32": dx.F32, "float16": dx.F16, "bfloat16": dx.BF16}[s["dtype"]]
    cache, rows = _cache(dx, s)
    dx.check(dx.load().dxh_kvcache_write(cache, rows, dt, _heads(dx, s["k"]), _heads(dx, s["v"]), _stream()), "kvcache_write")
    return {"k": s["kc"], "v": s["vc"], "k_scale": s["ks"], "v_scale": s["vs"]}


def own_read(s):
    from deepx_amd import lib as dx
    dt = {"float32": dx.F32, "float16": dx.F16, "bfloat16": dx.BF16}[s["dtype"]]
    cache, rows = _cache(dx, s)
    k, v = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    dx.check(dx.load().dxh_kvcache_read(cache, rows, dt, _heads(dx, k), _heads(dx, v), _stream()), "kvcache_read")
    return {"k": k, "v": v}


def own_attention(s):
    from deepx_amd import lib as dx
    dt = {"float32": dx.F32, "float16": dx.F16, "bfloat16": dx.BF16}[s["dtype"]]
    cache, rows = _cache(dx, s)
    dx.check(dx.load().dxh_kvcache_attention(cache, rows, dt, s["q_heads"], _heads(dx, s["q"]), _heads(dx, s["out"]), None, s["scale"], int(s["causal"]), s["window"],
                                             s["scratch"].data_ptr(), s["scratch"].numel(), _stream()), "kvcache_attention")
    return s["out"]


OWN = {"normrope": own_normrope, "normrope_backward": own_normrope_backward, "kvcache_write": own_write, "kvcache_read": own_read, "kvcache_attention": own_attention}


# ---- the definition in 64 bits, sequence by sequence -----------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op, dim = case["op"], case["dim"]
    if op.startswith("normrope"):
        half = case["rotary"] // 2
        lo = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        hi = lo + (1 if case["interleaved"] else half)
        c, z = (s[name].double()[s["positions"].long()].unsqueeze(1) for name in ("cos", "sin"))

        def forward(x, w):
            x = x.double()
            y = x / (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
            a, b = y[..., lo], y[..., hi]
            y[..., lo], y[..., hi] = a * c - b * z, a * z + b * c
            return y

        if op == "normrope":
            return {"q": forward(s["q"], s["wq"]), "k": forward(s["k"], s["wk"])}

        def backward(x, dy, w):
            x, g = x.double(), dy.double().clone()
            a, b = g[..., lo], g[..., hi]
            g[..., lo], g[..., hi] = a * c + b * z, b * c - a * z
            norm = (x.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt()
            unit = x / norm
            inner = (g * w.double() * unit).sum(-1, keepdim=True) / dim
            return (g * w.double() - unit * inner) / norm, (g * unit).flatten(0, 1).sum(0)

        dq, dwq = backward(s["q"], s["dq"], s["wq"])
        dk, dwk = backward(s["k"], s["dk"], s["wk"])
        return {"dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    page, hk = case["page"], case["kv_heads"]
    kc, vc, ks, vs = s["kc"].double(), s["vc"].double(), s["ks"].double(), s["vs"].double()
    starts = s["offsets"].tolist()
    tables = s["table"].tolist()
    if op == "kvcache_write":
        # codes as the numbers they stand for before rounding to 8 bits; whole numbers have no such value
        for b, (length, new) in enumerate(zip(s["host_lengths"], s["host_news"])):
            begin = length - new
            for slot in range(begin // page, (length - 1) // page + 1):
                p, t0, t1 = tables[b][slot], max(begin, slot * page), min(length, slot * page + page)
                kept = t0 - slot * page
                rows = slice(starts[b] + t0 - begin, starts[b] + t1 - begin)
                for x, codes, scales, across in ((s["k"], kc, ks, False), (s["v"], vc, vs, True)):
                    x = x[rows].double().transpose(0, 1)  # [heads, tokens, dim]
                    scale = (x.abs().amax((1, 2)) / CODE_MAX[case["code"]]).clamp(min=SCALE_MIN)
                    view = codes[p].transpose(1, 2) if across else codes[p]
                    if kept:
                        scale = torch.maximum(scale, scales[p])
                        view[:, :kept] *= (scales[p] / scale)[:, None, None]
                    view[:, kept:kept + t1 - t0] = x / scale[:, None, None]
                    scales[p] = scale
        whole = case["code"] == "int8"
        return {"k": None if whole else kc, "v": None if whole else vc, "k_scale": ks, "v_scale": vs}
    outs, more = [], []
    for b, (length, new) in enumerate(zip(s["host_lengths"], s["host_news"])):
        mine = torch.tensor(tables[b][:-(-length // page)], device="cuda")
        k = (kc[mine] * ks[mine][:, :, None, None]).transpose(0, 1).reshape(hk, -1, dim)[:, :length]
        v = (vc[mine] * vs[mine][:, :, None, None]).permute(1, 0, 3, 2).reshape(hk, -1, dim)[:, :length]
        if op == "kvcache_read":
            outs.append(k[:, length - new:].transpose(0, 1))
            more.append(v[:, length - new:].transpose(0, 1))
            continue
        q = s["q"][starts[b]:starts[b] + new].double()
        out = torch.zeros(new, case["q_heads"], dim, device="cuda", dtype=torch.float64)
        row, token = torch.arange(length - new, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
        hidden = (token > row) if case["causal"] else torch.zeros(new, length, device="cuda", dtype=torch.bool)
        if case["window"]:
            hidden = hidden | (token <= row - case["window"])
        for h in range(case["q_heads"]):
            one = h * hk // case["q_heads"]
            score = (q[:, h] @ k[one].t().contiguous() * dim ** -0.5).masked_fill(hidden, float("-inf"))
            out[:, h] = torch.softmax(score, -1) @ v[one]
        outs.append(out)
    if op == "kvcache_read":
        return {"k": torch.cat(outs), "v": torch.cat(more)}
    return torch.cat(outs)
