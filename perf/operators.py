"""The decoder-side operators as a user's program calls them, beside their plain forms, over the sizes they serve.

Four operators: `matvec` (few rows of activations times int4 group-64 weights), `kv4` (new tokens into a paged 4-bit
K/V cache, and rows of it back), `decode` (attention of the newest tokens over that cache) and `cross` (attention to
another sequence's states). A case is one call with its sizes; `run` is one pass of it.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

GROUP = 64  # values that share one f16 scale


def listed():
    return [
        # a k or v projection of one token: 4.9 MB of weights, where the call's latency counts
        {"name": "matvec token kv", "op": "matvec", "m": 1, "n": 1536, "k": 6144, "dtype": "bf16", "bias": True},
        # an MLP's up projection of one token
        {"name": "matvec token mlp", "op": "matvec", "m": 1, "n": 16384, "k": 6144, "dtype": "bf16", "bias": False},
        # the MLP's down projection of eight sequences' tokens
        {"name": "matvec batch mlp", "op": "matvec", "m": 8, "n": 6144, "k": 16384, "dtype": "bf16", "bias": False},
        # odd sizes in f32
        {"name": "matvec f32 odd", "op": "matvec", "m": 3, "n": 5003, "k": 2496, "dtype": "f32", "bias": True},
        # one token of each of 16 sequences into the cache
        {"name": "kv4 token", "op": "kv4", "batch": 16, "tokens": 1, "longest": 4000, "shortest": 0, "kv_heads": 12,
         "dim": 128, "page": 64, "dtype": "bf16"},
        # two prompts of ragged offsets into the cache, and back for their attention
        {"name": "kv4 prompt", "op": "kv4", "batch": 2, "tokens": 4099, "longest": 1000, "shortest": 0, "kv_heads": 12,
         "dim": 128, "page": 64, "dtype": "bf16"},
        # one sequence early in its text
        {"name": "decode one short", "op": "decode", "batch": 1, "tokens": 1, "longest": 517, "shortest": 517,
         "heads": 48, "kv_heads": 12, "dim": 128, "page": 64, "dtype": "bf16"},
        # a batch of ragged sequences
        {"name": "decode batch", "op": "decode", "batch": 16, "tokens": 1, "longest": 16384, "shortest": 3001,
         "heads": 48, "kv_heads": 12, "dim": 128, "page": 64, "dtype": "bf16"},
        # a few tokens at once (drafted ones to be checked), f32, small pages, narrow heads
        {"name": "decode drafted f32", "op": "decode", "batch": 3, "tokens": 5, "longest": 3333, "shortest": 1,
         "heads": 16, "kv_heads": 8, "dim": 64, "page": 16, "dtype": "f32"},
        # image tokens of two images to their text states, the second text shorter
        {"name": "cross image to text", "op": "cross", "batch": 2, "tq": 4096, "tk": 512, "longest": 512,
         "shortest": 333, "heads": 24, "kv_heads": 24, "dim": 128, "mask": False, "dtype": "bf16"},
        # one token of each of 8 sequences to an image's states
        {"name": "cross token to image", "op": "cross", "batch": 8, "tq": 1, "tk": 4096, "longest": 4096,
         "shortest": 4096, "heads": 48, "kv_heads": 12, "dim": 128, "mask": False, "dtype": "bf16"},
        # f32 states of odd lengths with holes in the mask
        {"name": "cross f32 masked", "op": "cross", "batch": 2, "tq": 300, "tk": 203, "longest": 203, "shortest": 77,
         "heads": 16, "kv_heads": 8, "dim": 64, "mask": True, "dtype": "f32"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["matvec", "matvec", "kv4", "decode", "decode", "cross", "cross"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "matvec":
        while True:
            m, n, k = rng.randint(1, 16), _log_int(rng, 200, 32768), GROUP * _log_int(rng, 8, 256)
            if n * k <= 6144 * 16384:
                return {"op": op, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5}
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    page = rng.choice([16, 32, 64, 128])
    if op == "kv4":
        batch = rng.randint(1, 16)
        return {"op": op, "batch": batch, "tokens": _log_int(rng, 1, 8192 // batch), "longest": rng.randint(0, 4000),
                "shortest": 0, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": "bf16"}
    if op == "decode":
        batch = rng.randint(1, 16)
        tokens = rng.choice([1, 1, 1, 2, 3, 5, 8])
        longest = _log_int(rng, 16, 131072 // (batch * tokens))
        return {"op": op, "batch": batch, "tokens": tokens, "longest": longest,
                "shortest": rng.randint(0, longest), "heads": kv_heads * rng.choice([1, 2, 4, 8]),
                "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    heads = kv_heads * rng.choice([1, 2, 4])
    batch, tk = rng.randint(1, 8), _log_int(rng, 1, 4096)
    most = 8192 * 400 * 24 if dtype == "bf16" else 1024 * 512 * 24  # query rows x keys
    rows = min(most // tk, (8192 if dtype == "bf16" else 4096) * 24)
    tq = min(rng.choice([1, _log_int(rng, 1, 4096)]), max(1, rows // (batch * heads)))
    return {"op": op, "batch": batch, "tq": tq, "tk": tk, "longest": tk, "shortest": rng.randint(1, tk),
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "mask": rng.random() < 0.5, "dtype": dtype}


# ---------------- inputs ----------------
def _quantise(x):
    """Rows [..., d] as symmetric int4 in groups of 64: codes in -8..7 (f32) and f16 scales [..., d / 64]."""
    g = x.float().unflatten(-1, (-1, GROUP))
    scale = (g.abs().amax(-1) / 7.0).clamp(max=65504.0).to(torch.float16)
    s = scale.float().unsqueeze(-1)
    codes = torch.where(s > 0, (g / s).round().clamp(-8, 7), torch.zeros_like(g))
    return codes.flatten(-2), scale


def _pack(codes):
    """Two codes to a byte, the lower value in the low half."""
    c = codes.to(torch.int16) & 15
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)


def _lengths(case):
    """Tokens that each sequence holds already, from the longest to the shortest."""
    b, lo, hi = case["batch"], case["shortest"], case["longest"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def _cache(case, lengths, filled, gen, dev):
    """A paged 4-bit cache with room for `filled[b]` tokens of each sequence, its pages in random order."""
    batch, kvh, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    used = [-(-f // page) for f in filled]
    max_pages = max(1, max(used))
    pages = batch * max_pages
    c = {"page_table": torch.randperm(pages, generator=gen, device=dev).to(torch.int32).view(batch, max_pages),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev), "pages": pages, "max_pages": max_pages}
    for name in ("k", "v"):
        x = torch.randn(pages, kvh, page, dim, generator=gen, device=dev, dtype=torch.bfloat16)
        codes, scale = _quantise(x)
        del x
        c[name], c[name + "_scale"] = _pack(codes), scale
        del codes
    return c


def prepare(case, seed):
    dev = torch.device("cuda")
    if own:
        _graph()
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dt)

    s = {"case": case}
    if case["op"] == "matvec":
        m, n, k = case["m"], case["n"], case["k"]
        codes, s["scale"] = _quantise(torch.randn(n, k, generator=gen, device=dev) * 0.02)
        s["w"] = _pack(codes)
        s["x"] = randn(m, k)
        s["bias"] = torch.randn(n, generator=gen, device=dev) if case["bias"] else None
        s["y"] = torch.empty(m, n, device=dev, dtype=dt)
    elif case["op"] == "kv4":
        lengths, t = _lengths(case), case["tokens"]
        s["cache"] = _cache(case, lengths, [x + t for x in lengths], gen, dev)
        shape = (case["batch"], t, case["kv_heads"], case["dim"])
        s["k"], s["v"] = randn(*shape), randn(*shape)
        s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    elif case["op"] == "decode":
        lengths, t = _lengths(case), case["tokens"]
        s["cache"] = _cache(case, lengths, [x + t for x in lengths], gen, dev)
        s["q"] = randn(case["batch"], t, case["heads"], case["dim"], std=2.0)
        s["out"] = torch.empty_like(s["q"])
    else:
        b, tq, tk, h, kvh, d = (case[x] for x in ("batch", "tq", "tk", "heads", "kv_heads", "dim"))
        s["q"], s["k"], s["v"] = randn(b, tq, h, d, std=2.0), randn(b, tk, kvh, d), randn(b, tk, kvh, d)
        s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        s["mask"] = (torch.rand(b, tk, generator=gen, device=dev) < 0.8).to(torch.uint8) if case["mask"] else None
        s["out"] = torch.empty_like(s["q"])
    if own:
        s["calls"] = _calls(case, s)
    return s


# ---------------- the framework's calls ----------------
_kept = {}


def _graph():
    """The package and one graph of it on a stream of its own, which torch's work shares."""
    if not _kept:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "web-engine_b200")
        spec = importlib.util.spec_from_file_location("web_engine_b200", os.path.join(root, "__init__.py"),
                                                      submodule_search_locations=[root])
        we = sys.modules["web_engine_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(we)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        _kept["we"], _kept["graph"] = we, we.Graph(torch.cuda.current_device())
        _kept["graph"].set_stream(stream.cuda_stream)
        _kept["stream"] = stream
    return _kept["we"], _kept["graph"]


def _calls(case, s):
    """The prepared calls that a decoding loop keeps: its buffers stay in place from token to token."""
    we, g = _graph()
    dt = case["dtype"]
    if case["op"] == "matvec":
        return [we.kernels.matvec_call(g, s["x"], s["w"], s["y"], case["m"], case["n"], case["k"],
                                       group_scale=s["scale"], x_dtype=dt, y_dtype=dt, bias=s["bias"])]
    if case["op"] == "cross":
        return [we.kernels.cross_attention_call(g, s["q"], s["k"], s["v"], s["out"], case["batch"], case["tq"],
                                                case["tk"], case["heads"], case["kv_heads"], case["dim"],
                                                key_lengths=s["lengths"], key_mask=s["mask"], dtype=dt,
                                                out_dtype=dt)]
    c = s["cache"]
    cache = we.kv4.Cache(c["k"], c["v"], c["k_scale"], c["v_scale"], c["page_table"], c["lengths"], c["pages"],
                         c["max_pages"], case["batch"], case["kv_heads"], case["page"], case["dim"])
    if case["op"] == "kv4":
        return [we.kv4.append_call(g, cache, s["k"], s["v"], case["tokens"], dtype=dt),
                we.kv4.unpack_call(g, cache, s["k_back"], s["v_back"], case["tokens"], dtype=dt)]
    return [we.kv4.attention_call(g, cache, s["q"], s["out"], case["tokens"], case["heads"], dtype=dt, out_dtype=dt)]


def run(s):
    case = s["case"]
    if own:
        for call in s["calls"]:
            call()
        if case["op"] == "matvec":
            return s["y"]
        return {"k": s["k_back"], "v": s["v_back"]} if case["op"] == "kv4" else s["out"]
    return _PLAIN[case["op"]](case, s)


# ---------------- the plain forms ----------------
def _values(packed, scale):
    """What packed rows stand for, in f32."""
    low, high = (packed & 15).to(torch.int8), (packed >> 4).to(torch.int8)
    q = torch.stack((low, high), -1).flatten(-2)
    q = torch.where(q > 7, q - 16, q).float()
    return (q.unflatten(-1, (-1, GROUP)) * scale.float().unsqueeze(-1)).flatten(-2)


def _plain_matvec(case, s):
    y = s["x"].float() @ _values(s["w"], s["scale"]).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_kv4(case, s):
    back = {}
    for name in ("k", "v"):
        codes, scale = _quantise(s[name])
        values = (codes.unflatten(-1, (-1, GROUP)) * scale.float().unsqueeze(-1)).flatten(-2)
        back[name] = values.to(s[name].dtype)
    return back


def _paged(rows, table):
    """[pages, kv_heads, page, x] by each sequence's pages: [batch, kv_heads, tokens, x]."""
    return rows[table.long()].transpose(1, 2).flatten(2, 3)


def _softmax(scores, seen):
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


def _grouped(q, kv_heads):
    """[batch, t, heads, dim] as [batch, kv_heads, group * t, dim]."""
    b, t, h, d = q.shape
    return q.view(b, t, kv_heads, h // kv_heads, d).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)


def _ungrouped(o, t):
    b, kvh, rows, d = o.shape
    return o.view(b, kvh, rows // t, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, -1, d)


def _plain_decode(case, s):
    c, t, kvh = s["cache"], case["tokens"], case["kv_heads"]
    k = _values(_paged(c["k"], c["page_table"]), _paged(c["k_scale"], c["page_table"]))
    scores = _grouped(s["q"].float(), kvh) @ k.transpose(-1, -2) / math.sqrt(case["dim"])
    at = c["lengths"].long().view(-1, 1) + torch.arange(t, device=k.device)  # each query's own position
    at = at.repeat(1, case["heads"] // kvh).view(case["batch"], 1, -1, 1)
    p = _softmax(scores, torch.arange(k.shape[2], device=k.device) <= at)
    v = _values(_paged(c["v"], c["page_table"]), _paged(c["v_scale"], c["page_table"]))
    return _ungrouped(p @ v, t).to(s["q"].dtype)


def _plain_cross(case, s):
    k, v = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    scores = _grouped(s["q"].float(), case["kv_heads"]) @ k.transpose(-1, -2) / math.sqrt(case["dim"])
    seen = torch.arange(case["tk"], device=k.device) < s["lengths"].view(-1, 1)
    if s["mask"] is not None:
        seen = seen & (s["mask"] != 0)
    p = _softmax(scores, seen.view(case["batch"], 1, 1, -1))
    return _ungrouped(p @ v, case["tq"]).to(s["q"].dtype)


_PLAIN = {"matvec": _plain_matvec, "kv4": _plain_kv4, "decode": _plain_decode, "cross": _plain_cross}


# ---------------- what a pass cannot do without ----------------
def work(case):
    e = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "matvec":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k // 2 + n * (k // GROUP) * 2 + (m * k + m * n) * e + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    d, kvh = case["dim"], case["kv_heads"]
    row = d // 2 + d // GROUP * 2
    if case["op"] == "kv4":
        rows = case["batch"] * case["tokens"] * kvh * 2
        return {"bytes": 2 * rows * (d * e + row), "flops": 4 * rows * d}
    if case["op"] == "decode":
        t = case["tokens"]
        keys = sum(x + t for x in _lengths(case))
        pairs = sum(x + i + 1 for x in _lengths(case) for i in range(t))
        return {"bytes": keys * kvh * row * 2 + 2 * case["batch"] * t * case["heads"] * d * e,
                "flops": 4 * pairs * case["heads"] * d}
    keys = sum(_lengths(case))
    return {"bytes": (2 * keys * kvh + 2 * case["batch"] * case["tq"] * case["heads"]) * d * e,
            "flops": 4 * keys * case["tq"] * case["heads"] * d}


# ---------------- the definitions in 64 bits ----------------
def _codes64(packed):
    """[..., d / 2] bytes as d two's complement values, the low half of a byte first."""
    b = packed.to(torch.int64)
    nib = torch.empty(*b.shape[:-1], b.shape[-1] * 2, dtype=torch.int64, device=b.device)
    nib[..., 0::2], nib[..., 1::2] = b % 16, b // 16
    return ((nib + 8) % 16 - 8).double()


def _attend64(q, k, v, last):
    """One head's rows: q [t, d], k, v [keys, d]; row i sees the first last[i] keys (or those marked, for a mask)."""
    sc = torch.einsum("td,kd->tk", q, k) * q.shape[-1] ** -0.5
    sc = sc.masked_fill(~last, -math.inf)
    p = torch.softmax(sc, -1)
    return torch.einsum("tk,kd->td", torch.nan_to_num(p), v)


def exact(case, seed):
    s = prepare(case, seed)
    dev = "cuda"
    if case["op"] == "matvec":
        w = _codes64(s["w"]) * s["scale"].double().repeat_interleave(GROUP, -1)
        y = torch.einsum("mk,nk->mn", s["x"].double(), w)
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "kv4":
        back = {}
        for name in ("k", "v"):
            x = s[name].double()
            top = x.abs().view(*x.shape[:-1], -1, GROUP).max(-1).values
            sc = (top / 7).clamp(max=65504).half().double().repeat_interleave(GROUP, -1)
            q = torch.round(x / sc.clamp(min=1e-30)).clamp(-8, 7)
            back[name] = torch.where(sc > 0, q * sc, torch.zeros_like(q))
        return back
    kvh, d, group = case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(*s["out"].shape, dtype=torch.float64, device=dev)
    if case["op"] == "decode":
        c, t = s["cache"], case["tokens"]
        for b, have in enumerate(_lengths(case)):
            n = have + t
            ids = c["page_table"][b].long()
            seen = torch.arange(n, device=dev)[None, :] <= torch.arange(have, n, device=dev)[:, None]
            for j in range(kvh):
                k, v = ((_codes64(c[x][ids, j]) * c[x + "_scale"][ids, j].double().repeat_interleave(GROUP, -1))
                        .reshape(-1, d)[:n] for x in ("k", "v"))
                for h in range(j * group, (j + 1) * group):
                    out[b, :, h] = _attend64(s["q"][b, :, h].double(), k, v, seen)
        return out
    for b, n in enumerate(_lengths(case)):
        seen = torch.arange(case["tk"], device=dev) < n
        if s["mask"] is not None:
            seen = seen & s["mask"][b].bool()
        for h in range(case["heads"]):
            out[b, :, h] = _attend64(s["q"][b, :, h].double(), s["k"][b, :, h // group].double(),
                                     s["v"][b, :, h // group].double(), seen.expand(case["tq"], -1))
    return out
