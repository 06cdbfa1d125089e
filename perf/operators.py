"""The operators between two fused launches of a layer, as cases that can be timed and compared.

``norm``    ``rmsnorm_int8``: residual add + RMSNorm over packed rows, 8-bit integers and a scale
            for each token out (the operand of the next projection).
``linear``  ``linear_int8``: the projection itself, 8-bit integers with a scale for each token and
            each output channel.
``append``  ``rope_append``: the projection's Q rotated, its new K rotated and V, put into the pages
            that the paged layer reads.

With ``own`` false ``run`` computes the same from elementary torch operations in 32 bits (angles in
64).  Sizes are this repository's benchmark configurations (``megaattention_b200/workloads.py``,
``perf/cases.py``) and generic serving shapes.
"""
import math

import torch

own = False

D = 128
PAGE = 128
EPS = 1e-6
THETA = 10000.0

_SWEEP = [7500, 4100, 3300, 2600, 2000, 1500, 1000, 600]
# a prefix-cached batch: short new turns behind conversations of a few thousand tokens
_TURNS_Q = [17, 256, 45, 130, 300, 64, 1, 97, 211, 33, 150, 80]
_TURNS_K = [2065, 3300, 801, 1154, 4396, 640, 1537, 5217, 1235, 2800, 150, 3152]


def _norm(name, tokens, hidden, residual):
    return {"name": name, "op": "norm", "tokens": tokens, "hidden": hidden, "residual": residual}


def _linear(name, tokens, inner, width, bias=False, out="bf16"):
    return {"name": name, "op": "linear", "tokens": tokens, "inner": inner, "width": width,
            "bias": bias, "out": out}


def _append(name, q, k, heads, kv_heads, fused):
    """``fused``: q, k and v are views of one projection's output, not tensors of their own."""
    return {"name": name, "op": "append", "q": ",".join(map(str, q)), "k": ",".join(map(str, k)),
            "heads": heads, "kv_heads": kv_heads, "fused": fused}


def listed():
    return [
        # a decode step of eight sequences: the norm before a projection
        _norm("norm_decode", 8, 4096, True),
        # the first norm of a model over a ragged prefill batch: no residual yet
        _norm("norm_first", 13400, 4096, False),
        # the largest prefill batch of the wide model
        _norm("norm_wide", 22600, 16384, True),
        # one token through the QKV projection of the whole 64-head model
        _linear("linear_token", 1, 4096, 10240),
        # a decode step of 48 sequences, one rank of the wide model
        _linear("linear_decode", 48, 16384, 2304),
        # the new turns of a dozen conversations, one rank's QKV projection
        _linear("linear_turns", sum(_TURNS_Q), 4096, 1280),
        # odd sizes throughout, bias, 32-bit result (a small model's scores)
        _linear("linear_odd", 777, 1000, 1001, True, "f32"),
        # a ragged prefill batch, QKV of the whole model, with bias
        _linear("linear_prefill", 13400, 4096, 10240, True),
        # the largest: a prefill batch into four times the model's width
        _linear("linear_large", 22600, 4096, 16384),
        # a decode step: one token for each of 64 conversations
        _append("append_tokens", [1] * 64, [97 + 251 * i for i in range(64)], 8, 1, True),
        # new turns of a dozen conversations in one step
        _append("append_turns", _TURNS_Q, _TURNS_K, 16, 2, True),
        # the largest: complete prompts of the whole 64-head model, q, k and v of their own
        _append("append_whole", _SWEEP, _SWEEP, 64, 8, False),
    ]


def _lens(case):
    return [int(x) for x in case["q"].split(",")], [int(x) for x in case["k"].split(",")]


def work(case):
    """Every input read once, every output written once."""
    if case["op"] == "norm":
        n = case["tokens"] * case["hidden"]
        per = 2 + 1 + (4 if case["residual"] else 0)
        return {"bytes": float(per * n + 4 * case["tokens"] + 2 * case["hidden"]), "flops": 6.0 * n}
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["width"]
        size = 2 if case["out"] == "bf16" else 4
        return {"bytes": float(m * k + n * k + size * m * n + 4 * (m + n) + (2 * n if case["bias"] else 0)),
                "flops": 2.0 * m * k * n}
    q, k = _lens(case)
    t, h, hkv = sum(q), case["heads"], case["kv_heads"]
    table = len(k) * max(-(-n // PAGE) for n in k)
    return {"bytes": 2.0 * t * D * (2 * h + 4 * hkv) + 4.0 * (table + 2 * len(q) + 1) + 256.0,
            "flops": 6.0 * t * D * (h + hkv)}


def draw(rng):
    """One more case of these ranges: 1 to 24000 tokens, hidden sizes to 16384, odd ones among them,
    never more work than the largest listed case of the same operator."""
    def log(lo, hi):
        return math.exp(rng.uniform(math.log(lo), math.log(hi)))

    while True:
        op = rng.choice(["norm", "linear", "append"])
        if op == "norm":
            c = _norm("", round(log(1, 24000)), 8 * round(log(64, 16384) / 8), rng.random() < 0.7)
        elif op == "linear":
            k, n = round(log(64, 16384)), round(log(64, 32768))
            if rng.random() < 0.5:
                k, n = max(64, k // 128 * 128), max(64, n // 64 * 64)
            c = _linear("", round(log(1, 24000)), k, n, rng.random() < 0.4,
                        rng.choice(["bf16", "bf16", "bf16", "f32"]))
        else:
            heads, kv = rng.choice([(8, 1), (8, 8), (16, 2), (16, 1), (4, 1), (7, 1), (6, 2), (12, 12),
                                    (32, 4), (64, 8)])
            n = round(log(1, 200))
            if rng.random() < 0.4:
                q = [1] * n
            else:
                tokens = log(n, 24000)
                share = [rng.uniform(0.2, 1.0) ** 2 for _ in range(n)]
                q = [max(1, round(tokens * s / sum(share))) for s in share]
            longest = log(1, 16000) if rng.random() < 0.7 else 0.0
            k = [a + round(longest * rng.random()) for a in q]
            if sum(k) > 400000:
                continue
            c = _append("", q, k, heads, kv, rng.random() < 0.7)
        del c["name"]
        most = [work(x) for x in listed() if x["op"] == op]
        w = work(c)
        if w["flops"] <= max(m["flops"] for m in most) and w["bytes"] <= max(m["bytes"] for m in most):
            return c


def _eight_bits(x):
    """Rows of 8-bit integers and their scales; the rows start 16 bytes apart, as the framework has them."""
    rows, n = x.shape
    top = x.abs().amax(-1, keepdim=True).clamp_min(1e-20)
    q = torch.zeros(rows, -(-n // 16) * 16, dtype=torch.int8, device=x.device)
    q[:, :n] = torch.round(x * (127.0 / top)).to(torch.int8)
    return q[:, :n], (top / 127.0).reshape(-1).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))

    def randn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, generator=g, device=dev, dtype=dtype)

    s = {"op": case["op"]}
    if case["op"] == "norm":
        t, n = case["tokens"], case["hidden"]
        # channels of a trained model differ in size; the residual stream is larger than what is added
        channel = torch.exp(0.5 * randn(n, dtype=torch.float32)).to(torch.bfloat16)
        s["x"] = randn(t, n).mul_(channel)
        s["residual"] = randn(t, n).mul_(3.0 * channel) if case["residual"] else None
        s["weight"] = 1.0 + 0.1 * randn(n)
    elif case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["width"]
        s["x"], s["x_scale"] = _eight_bits(randn(m, k, dtype=torch.float32))
        s["weight"], s["weight_scale"] = _eight_bits(randn(n, k, dtype=torch.float32).mul_(k ** -0.5))
        s["bias"] = 0.5 * randn(n) if case["bias"] else None
        s["dtype"] = torch.bfloat16 if case["out"] == "bf16" else torch.float32
    else:
        q, k = _lens(case)
        t, h, hkv = sum(q), case["heads"], case["kv_heads"]
        if case["fused"]:
            qkv = randn(t, (h + 2 * hkv) * D)
            s["q"] = qkv[:, :h * D].unflatten(1, (h, D))
            s["k"] = qkv[:, h * D:(h + hkv) * D].unflatten(1, (hkv, D))
            s["v"] = qkv[:, (h + hkv) * D:].unflatten(1, (hkv, D))
        else:
            s["q"], s["k"], s["v"] = randn(t, h, D), randn(t, hkv, D), randn(t, hkv, D)
        need = [-(-n // PAGE) for n in k]
        pages = sum(need) + 8
        order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
        table = torch.zeros(len(k), max(need), dtype=torch.int32, device=dev)
        n = torch.tensor(need, device=dev)
        col = torch.arange(max(need), device=dev)
        table[col < n[:, None]] = order[:sum(need)]
        s["page_table"] = table
        s["k_cache"], s["v_cache"] = randn(pages, PAGE, hkv, D), randn(pages, PAGE, hkv, D)
        s["cache_seqlens"] = torch.tensor(k, dtype=torch.int32, device=dev)
        cu = torch.zeros(len(q) + 1, dtype=torch.int32)
        cu[1:] = torch.tensor(q).cumsum(0)
        s["cu_seqlens_q"] = cu.to(dev)
        s["inv_freq"] = 1.0 / (THETA ** (torch.arange(0, D, 2, dtype=torch.float32, device=dev) / D))
    return s


def _plain_norm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (h.float() + s["residual"].float()).to(torch.bfloat16)
    x = h.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    top = y.abs().amax(-1, keepdim=True)
    q = torch.round(y * (127.0 / top))
    scale = top / 127.0
    out = {"values": (q * scale).to(torch.bfloat16), "scale": scale.reshape(-1)}
    if s["residual"] is not None:
        out["residual"] = h
    return out


def _plain_linear(s):
    y = (s["x"].float() @ s["weight"].float().T) * s["x_scale"][:, None] * s["weight_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


def _rotate(x, c, s):
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def _places(s, tokens):
    """Position, page and row in the page of each of the tokens."""
    cu = s["cu_seqlens_q"].long()
    t = torch.arange(tokens, device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    p = s["cache_seqlens"].long()[b] - (cu[b + 1] - t)
    return p, s["page_table"][b, p // PAGE].long(), p % PAGE


def _plain_append(s):
    p, page, row = _places(s, s["q"].shape[0])
    angle = p.double()[:, None, None] * s["inv_freq"].double()
    c, sn = angle.cos().float(), angle.sin().float()
    q = _rotate(s["q"].float(), c, sn).to(torch.bfloat16)
    s["k_cache"][page, row] = _rotate(s["k"].float(), c, sn).to(torch.bfloat16)
    s["v_cache"][page, row] = s["v"]
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def run(s):
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "append": _plain_append}[s["op"]](s)
    from megaattention_b200 import runtime
    if s["op"] == "norm":
        got = runtime.rmsnorm_int8(s["x"], s["weight"], EPS, residual=s["residual"])
        # (8-bit values are returned as what they stand for)
        out = {"values": runtime.dequantize_int8(got[0], got[1]), "scale": got[1]}
        if s["residual"] is not None:
            out["residual"] = got[2]
        return out
    if s["op"] == "linear":
        return runtime.linear_int8(s["x"], s["x_scale"], s["weight"], s["weight_scale"], bias=s["bias"],
                                   out_dtype=s["dtype"])
    q = runtime.rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["page_table"],
                            s["cache_seqlens"], s["cu_seqlens_q"], inv_freq=s["inv_freq"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def exact(case, seed):
    """What ``run`` returns, in float64 from the definition.  The residual stream is held in 16 bits by
    definition, and the 8-bit values are whole multiples of their scale."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        values, scales, stream = [], [], []
        w = s["weight"].double()
        for a in range(0, case["tokens"], 2048):
            h = s["x"][a:a + 2048].double()
            if case["residual"]:
                h = (h + s["residual"][a:a + 2048].double()).to(torch.bfloat16)
                stream.append(h)
                h = h.double()
            y = h * w / torch.sqrt(h.square().sum(-1, keepdim=True) / case["hidden"] + EPS)
            step = y.abs().max(-1, keepdim=True).values / 127.0
            values.append(torch.round(y / step) * step)
            scales.append(step.squeeze(-1))
        out = {"values": torch.cat(values), "scale": torch.cat(scales)}
        if case["residual"]:
            out["residual"] = torch.cat(stream).double()
        return out
    if case["op"] == "linear":
        w = s["weight"].double() * s["weight_scale"].double()[:, None]
        b = s["bias"].double() if case["bias"] else 0.0
        return torch.cat([(s["x"][a:a + 4096].double() * s["x_scale"][a:a + 4096].double()[:, None]) @ w.T + b
                          for a in range(0, case["tokens"], 4096)])
    lens_q, lens_k = _lens(case)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    q = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    table = s["page_table"].tolist()
    a = 0
    freq = s["inv_freq"].double()
    for i, (n, m) in enumerate(zip(lens_q, lens_k)):
        pos = torch.arange(m - n, m, dtype=torch.float64, device=q.device)
        turn = torch.polar(torch.ones(n, D // 2, dtype=torch.float64, device=q.device), pos[:, None] * freq)

        def turned(x):
            z = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * turn[:, None]
            return torch.cat([z.real, z.imag], -1)

        q[a:a + n] = turned(s["q"][a:a + n])
        k, v = turned(s["k"][a:a + n]), s["v"][a:a + n].double()
        at = m - n
        while at < m:
            stop = min(m, (at // PAGE + 1) * PAGE)
            page, lo = table[i][at // PAGE], at % PAGE
            k_cache[page, lo:lo + stop - at] = k[at - (m - n):stop - (m - n)]
            v_cache[page, lo:lo + stop - at] = v[at - (m - n):stop - (m - n)]
            at = stop
        a += n
    return {"q": q, "k_cache": k_cache, "v_cache": v_cache}
