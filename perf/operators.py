"""The decoder-side operators of this library: what is measured, in plain form and through qik.

Four operators that a transformer server runs together around the FP8 linears:

* ``norm``    residual addition + RMS norm with an e4m3 output (``qik.rms_norm``);
* ``rotary``  rotary positions on q and k, the rotated k and v stored in a paged cache (``qik.rotary``);
* ``pages``   copies between pages of a paged cache: the moves of a fork or a compaction (``qik.paged_kv``);
* ``attn``    attention of new tokens over a paged cache: one token, a chunk or a whole prompt
              per sequence, causal or not, with an optional window and sinks (``qik.paged_attention``).

``run`` computes them with elementary torch operations in 32 bits (rotary angles in 64) when
``own`` is false, and through the library when it is true.  ``exact`` is the definition in 64
bits, written apart.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_PKG = Path(__file__).resolve().parent.parent / "qwen-image-kernel_b200"
_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEV = "cuda"


def _qik(module):
    if str(_PKG) not in sys.path:
        sys.path.insert(0, str(_PKG))
    import importlib
    return importlib.import_module("qik." + module)


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # one sequence decoding its next token, early in an answer: latency
        {"name": "attn_decode_one", "op": "attn", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "batch": 1, "new_lo": 1, "new_hi": 1, "ctx_lo": 300, "ctx_hi": 300, "causal": True, "window": 0, "sinks": 0,
         "mix": 1},
        # a full decode batch whose sequences have very different lengths: bandwidth
        {"name": "attn_decode_batch", "op": "attn", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "batch": 64, "new_lo": 1, "new_hi": 1, "ctx_lo": 500, "ctx_hi": 12000, "causal": True, "window": 0, "sinks": 0,
         "mix": 2},
        # chunked prefill: a few hundred new tokens each over contexts already in the cache
        {"name": "attn_chunks", "op": "attn", "dtype": "bf16", "heads": 28, "kv_heads": 4, "dim": 128, "page": 32,
         "batch": 5, "new_lo": 200, "new_hi": 700, "ctx_lo": 1500, "ctx_hi": 9000, "causal": True, "window": 0,
         "sinks": 0, "mix": 3},
        # a whole long prompt at once, every head with its own keys (this library's 24 heads of 128)
        {"name": "attn_prompt", "op": "attn", "dtype": "bf16", "heads": 24, "kv_heads": 24, "dim": 128, "page": 128,
         "batch": 1, "new_lo": 8001, "new_hi": 8001, "ctx_lo": 0, "ctx_hi": 0, "causal": True, "window": 0, "sinks": 0,
         "mix": 4},
        # drafted tokens being verified under a sliding window with four sink tokens, long contexts
        {"name": "attn_window_sinks", "op": "attn", "dtype": "fp16", "heads": 16, "kv_heads": 2, "dim": 64, "page": 16,
         "batch": 24, "new_lo": 1, "new_hi": 7, "ctx_lo": 3000, "ctx_hi": 30000, "causal": True, "window": 1024,
         "sinks": 4, "mix": 5},
        # the rows of a small decode step, for the next FP8 linear: latency
        {"name": "norm_rows_3", "op": "norm", "dtype": "bf16", "rows": 3, "cols": 4096, "scales": "tensor"},
        # the rows of a prefill step, for the next FP8 linear
        {"name": "norm_rows_8192", "op": "norm", "dtype": "bf16", "rows": 8192, "cols": 5120, "scales": "tensor"},
        # one scale per token, an odd row count
        {"name": "norm_row_scales", "op": "norm", "dtype": "fp16", "rows": 1001, "cols": 3584, "scales": "row"},
        # a decode step's q / k / v: rotation in halves, stored to scattered slots
        {"name": "rotary_decode", "op": "rotary", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "page": 16,
         "tokens": 48, "rot": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "far": 30000},
        # a prompt's q / k / v: interleaved pairs, half of each head, far positions under a scaled table
        {"name": "rotary_prompt", "op": "rotary", "dtype": "bf16", "heads": 24, "kv_heads": 24, "dim": 128, "page": 64,
         "tokens": 8111, "rot": 64, "interleaved": True, "scaling": "yarn", "factor": 4.0, "far": 120000},
        # forks of seven sequences: each child's own copy of a partly filled last page, all layers
        {"name": "pages_fork", "op": "pages", "dtype": "bf16", "layers": 32, "kv_heads": 8, "dim": 128, "page": 32,
         "pool": 64, "moves": 7, "whole": False},
        # a compaction: whole pages moved down into the holes that freed sequences left
        {"name": "pages_compact", "op": "pages", "dtype": "bf16", "layers": 12, "kv_heads": 8, "dim": 128, "page": 64,
         "pool": 1200, "moves": 500, "whole": True},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(("attn", "attn", "attn", "norm", "rotary", "pages"))
    dtype = rng.choice(("bf16", "fp16"))
    if op == "norm":
        return {"op": op, "dtype": dtype, "rows": _log(rng, 1, 8192), "cols": 8 * _log(rng, 8, 640),
                "scales": rng.choice(("tensor", "row"))}
    if op == "rotary":
        dim = rng.choice((64, 128))
        kv = rng.choice((1, 2, 4, 8, 24))
        return {"op": op, "dtype": dtype, "heads": kv * (rng.choice((1, 2, 3, 4, 7, 8)) if kv <= 4 else 1),
                "kv_heads": kv, "dim": dim, "page": rng.choice((16, 32, 64, 128)), "tokens": _log(rng, 1, 8000),
                "rot": rng.choice((dim, dim // 2, 3 * dim // 4, 16)), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(("none", "linear", "ntk", "yarn", "bands")), "factor": rng.choice((1.5, 4.0, 8.0)),
                "far": _log(rng, 10000, 130000)}
    if op == "pages":
        pool = _log(rng, 12, 1200)
        return {"op": op, "dtype": dtype, "layers": rng.randint(1, 12), "kv_heads": rng.choice((1, 2, 4, 8)),
                "dim": rng.choice((64, 128)), "page": rng.choice((16, 32, 64)), "pool": pool,
                "moves": _log(rng, 1, pool // 2 - 1), "whole": rng.random() < 0.5}
    kv = rng.choice((1, 2, 4, 8, 24))
    case = {"op": op, "dtype": dtype, "heads": kv * rng.choice((1, 2, 3, 4, 5, 7, 8) if kv <= 4 else (1, 2, 4) if kv == 8 else (1,)),
            "kv_heads": kv, "dim": rng.choice((64, 128, 128)), "page": rng.choice((16, 32, 64, 128))}
    kind = rng.choice(("decode", "draft", "chunk", "prompt"))
    if kind == "decode":
        batch, hi = _log(rng, 1, 64), 1
        ctx = _log(rng, 16, 100000 // batch)
    elif kind == "draft":
        batch, hi = _log(rng, 1, 32), rng.randint(2, 40)
        ctx = _log(rng, 16, 50000 // batch)
    elif kind == "chunk":
        batch, hi = _log(rng, 1, 4), _log(rng, 40, 500)
        ctx = _log(rng, 16, 6000)
    else:
        batch, hi = _log(rng, 1, 3), _log(rng, 100, 2000)
        ctx = 0
    case |= {"batch": batch, "new_lo": 1 if kind == "draft" else hi if kind == "decode" else max(1, hi // 3), "new_hi": hi,
             "ctx_lo": ctx // 5, "ctx_hi": ctx, "causal": kind == "decode" or rng.random() < 0.8, "window": 0, "sinks": 0,
             "mix": rng.randint(1, 10 ** 6)}
    if case["causal"] and rng.random() < 0.4:
        case |= {"window": _log(rng, 16, 4000), "sinks": rng.choice((0, 1, 4, 37))}
    return case


def _lengths(c):
    """(new tokens, cache lengths with them) of each sequence, from the case alone."""
    r = random.Random(c["mix"])
    new = [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]
    return new, [n + r.randint(c["ctx_lo"], c["ctx_hi"]) for n in new]


def _seen(c, new, kv):
    """(pairs of query and key that are computed, distinct keys that are read) of one sequence."""
    pairs = low = 0
    for j in range(new):
        limit = kv - new + j if c["causal"] else kv - 1
        first = max(0, limit - c["window"] + 1) if c["window"] else 0
        pairs += limit + 1 - first + min(c["sinks"], first)
        low = first if j == 0 else min(low, first)
    return pairs, kv - low + min(c["sinks"], low)


def work(c):
    if c["op"] == "norm":
        # x, residual, weight in; the sum, the codes and the scales out
        n = c["rows"] * c["cols"]
        return {"bytes": n * (2 + 2 + 2 + 1) + 2 * c["cols"] + 4 * (c["rows"] if c["scales"] == "row" else 1),
                "flops": 5 * n}
    if c["op"] == "rotary":
        # q, k, v and each token's angles in; q, k and v out
        h = c["heads"] + 2 * c["kv_heads"]
        return {"bytes": c["tokens"] * (2 * h * c["dim"] * 2 + c["rot"] * 4 + 16),
                "flops": c["tokens"] * 3 * (c["heads"] + c["kv_heads"]) * c["rot"]}
    if c["op"] == "pages":
        tokens = sum(t for _, _, t in _moves(c))
        return {"bytes": 2 * 2 * tokens * c["layers"] * c["kv_heads"] * c["dim"] * 2, "flops": 0}
    new, kv = _lengths(c)
    seen = [_seen(c, n, m) for n, m in zip(new, kv)]
    return {"bytes": 2 * c["dim"] * (2 * c["heads"] * sum(new) + 2 * c["kv_heads"] * sum(k for _, k in seen)),
            "flops": 4 * c["dim"] * c["heads"] * sum(p for p, _ in seen)}


def _moves(c):
    """(from, to, tokens) of each copied page, from the case alone: distinct pages, none both read and written."""
    r = random.Random(c["pool"] * 1009 + c["moves"])
    ids = r.sample(range(c["pool"]), 2 * c["moves"])
    return [(ids[i], ids[c["moves"] + i], c["page"] if c["whole"] else r.randint(1, c["page"])) for i in range(c["moves"])]


# ------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    c = case
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DTYPE[c["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=_DEV, dtype=torch.float32).mul_(std).to(dt)

    s = {"case": c}
    if c["op"] == "norm":
        # a residual stream that has grown over the layers, some columns far larger than the rest
        columns = torch.exp(0.8 * torch.randn(c["cols"], generator=g, device=_DEV))
        s["x"] = normal(c["rows"], c["cols"])
        s["residual"] = (torch.randn(c["rows"], c["cols"], generator=g, device=_DEV) * columns * 4).to(dt)
        s["weight"] = (1 + 0.2 * torch.randn(c["cols"], generator=g, device=_DEV)).to(dt)
        s["eps"] = 1e-6
        return s
    if c["op"] == "rotary":
        # views of one fused projection's output, as the QKV linear leaves it
        T, H, K, D, page = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
        qkv = normal(T, (H + 2 * K) * D)
        s["q"] = qkv[:, :H * D].unflatten(1, (H, D))
        s["k"] = qkv[:, H * D:(H + K) * D].unflatten(1, (K, D))
        s["v"] = qkv[:, (H + K) * D:].unflatten(1, (K, D))
        pages = -(-T // page) + 7
        s["k_pages"], s["v_pages"] = normal(pages, K, page, D), normal(pages, K, page, D)
        # decode steps scatter over many sequences' pages; a prompt's tokens follow one another in theirs
        if T <= 256:
            s["slots"] = torch.randperm(pages * page, generator=g, device=_DEV)[:T]
            s["positions"] = torch.randint(0, c["far"], (T,), generator=g, device=_DEV)
        else:
            order = torch.randperm(pages, generator=g, device=_DEV)
            t = torch.arange(T, device=_DEV)
            s["slots"] = order[t // page] * page + t % page
            first = torch.randint(0, max(1, c["far"] - T), (1,), generator=g, device=_DEV)
            s["positions"] = first + t
        # the table of cosines and sines that a server makes once and keeps
        if own:
            s["table"] = _qik("rotary").rotary_table(c["rot"], c["far"], base=10000.0, scaling=c["scaling"],
                                                     factor=c["factor"], original_positions=4096, device=_DEV)
        else:
            freq, gain = _frequencies(c)
            angle = torch.arange(c["far"], device=_DEV, dtype=torch.float64)[:, None] * freq
            s["table"] = ((gain * angle.cos()).float(), (gain * angle.sin()).float())
        return s
    if c["op"] == "pages":
        shape = (c["layers"], c["pool"], c["kv_heads"], c["page"], c["dim"])
        s["k_pages"], s["v_pages"] = (torch.empty(shape, dtype=dt, device=_DEV).normal_(generator=g) for _ in range(2))
        s["moves"] = _moves(c)
        return s
    new, kv = _lengths(c)
    H, K, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    s["q"] = normal(sum(new), H, D)
    width = max(-(-n // page) for n in kv)
    pages = sum(-(-n // page) for n in kv) + 3
    s["k_pages"] = torch.empty(pages, K, page, D, dtype=dt, device=_DEV).normal_(generator=g)
    s["v_pages"] = torch.empty(pages, K, page, D, dtype=dt, device=_DEV).normal_(generator=g)
    order = torch.randperm(pages, generator=g, device=_DEV).to(torch.int32).cpu()
    table = torch.zeros(len(kv), width, dtype=torch.int32)
    at = 0
    for i, n in enumerate(kv):
        m = -(-n // page)
        table[i, :m] = order[at:at + m]
        at += m
    s["page_table"] = table.to(_DEV)
    s["seq_lens"] = torch.tensor(kv, dtype=torch.int32, device=_DEV)
    s["query_starts"] = torch.tensor([0] + new, dtype=torch.int32).cumsum(0).to(torch.int32).to(_DEV)
    s["max_new"], s["max_kv"] = max(new), max(kv)
    return s


def _frequencies(c):
    """Rotary frequencies (64 bits) of a case's scaling, and the factor on its cosines and sines."""
    rot, base, factor, original = c["rot"], 10000.0, c["factor"], 4096
    i = torch.arange(rot // 2, device=_DEV, dtype=torch.float64)
    plain = base ** (-2 * i / rot)
    if c["scaling"] == "linear":
        return plain / factor, 1.0
    if c["scaling"] == "ntk":
        return (base * factor ** (rot / max(1, rot - 2))) ** (-2 * i / rot), 1.0
    if c["scaling"] == "yarn":
        # dimensions that turn over 32 times in the original length stay, under one turn they are divided
        at = [rot * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(0, math.floor(at[0])), min(rot - 1, math.ceil(at[1]))
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        return plain / factor * ramp + plain * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if c["scaling"] == "bands":
        # wavelengths under a quarter of the original length stay, over the whole of it they are divided
        turns = original * plain / (2 * math.pi)
        mix = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return plain / factor * (1 - mix) + plain * mix, 1.0
    return plain, 1.0


# ------------------------------------------------------------------------------ one pass
def run(state):
    s = state
    c = s["case"]
    if own:
        return _run_own(s, c)
    return {"norm": _norm, "rotary": _rotary, "pages": _pages, "attn": _attn}[c["op"]](s, c)


def _run_own(s, c):
    if c["op"] == "norm":
        f = _fn(s, "rms_norm", "fused_add_rms_norm_e4m3")
        return f(s["x"], s["residual"], s["weight"], s["eps"], scales=c["scales"])
    if c["op"] == "rotary":
        f = _fn(s, "rotary", "rotary_store")
        q = f(s["q"], s["k"], s["v"], s["positions"], s["table"], s["slots"], s["k_pages"], s["v_pages"],
              interleaved=c["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    if c["op"] == "pages":
        _fn(s, "paged_kv", "copy_pages")(s["k_pages"], s["v_pages"], s["moves"])
        return s["k_pages"], s["v_pages"]
    f = _fn(s, "paged_attention", "paged_attention")
    return f(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["seq_lens"], s["query_starts"], s["max_new"],
             max_kv=s["max_kv"], causal=c["causal"], window=c["window"], sinks=c["sinks"])


def _fn(s, module, name):
    """The library's function, as a program that has imported it holds it."""
    f = s.get("fn")
    if f is None:
        f = s["fn"] = getattr(_qik(module), name)
    return f


def _norm(s, c):
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + s["eps"]) * s["weight"].float()
    top = y.abs().amax(1) if c["scales"] == "row" else y.abs().amax().reshape(1)
    scale = (top / 448).clamp_min(1e-12)
    codes = (y / (scale[:, None] if c["scales"] == "row" else scale)).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes, scale, h.to(s["x"].dtype)


def _rotary(s, c):
    cos, sin = (t[s["positions"]][:, None] for t in s["table"])

    def turn(x):
        x = x.float()
        y = x.clone()
        a, b = (slice(0, c["rot"], 2), slice(1, c["rot"], 2)) if c["interleaved"] else \
            (slice(0, c["rot"] // 2), slice(c["rot"] // 2, c["rot"]))
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., b] * cos + x[..., a] * sin
        return y.to(s["q"].dtype)

    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_pages"][page, :, at] = turn(s["k"])
    s["v_pages"][page, :, at] = s["v"]
    return turn(s["q"]), s["k_pages"], s["v_pages"]


def _pages(s, c):
    a, b, t = torch.tensor(s["moves"], device=_DEV).unbind(1)
    filled = (torch.arange(c["page"], device=_DEV) < t[:, None])[None, :, None, :, None]
    for_k, for_v = (torch.where(filled, p[:, a], p[:, b]) for p in (s["k_pages"], s["v_pages"]))
    s["k_pages"][:, b] = for_k
    s["v_pages"][:, b] = for_v
    return s["k_pages"], s["v_pages"]


def _attn(s, c):
    H, K, D = c["heads"], c["kv_heads"], c["dim"]
    G, n, B, T = H // K, s["max_new"], c["batch"], s["q"].shape[0]
    new = (s["query_starts"][1:] - s["query_starts"][:-1]).long()
    kv = s["seq_lens"].long()
    keys, values = (p[s["page_table"].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :s["max_kv"]].float()
                    for p in (s["k_pages"], s["v_pages"]))                                    # [B, K, S, D]
    row = (s["query_starts"][:-1].long()[:, None] + torch.arange(n, device=_DEV)).clamp_max(T - 1)
    q = s["q"][row].float().reshape(B, n, K, G, D).permute(0, 2, 3, 1, 4).reshape(B, K, G * n, D)
    j = torch.arange(s["max_kv"], device=_DEV)
    limit = (kv - new)[:, None] + torch.arange(n, device=_DEV) if c["causal"] else (kv - 1)[:, None].expand(B, n)
    seen = (j <= limit[..., None]) & (j < kv[:, None, None])
    if c["window"]:
        seen &= (j > limit[..., None] - c["window"]) | (j < c["sinks"])                       # [B, n, S]
    score = ((q @ keys.transpose(2, 3)) * D ** -0.5).view(B, K, G, n, -1)
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    score.sub_(score.amax(-1, keepdim=True).clamp_min(-3e38)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(B, K, G * n, -1) @ values).view(B, K, G, n, D) / torch.where(total == 0, 1.0, total)
    # back to one row for each new token
    seq = torch.repeat_interleave(torch.arange(B, device=_DEV), new, output_size=T)
    at = torch.arange(T, device=_DEV) - s["query_starts"].long()[seq]
    return out.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[seq, at].to(s["q"].dtype)


# ------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        rms = ((h * h).sum(1) / c["cols"] + s["eps"]).sqrt()
        y = h / rms[:, None] * s["weight"].double()
        if c["scales"] == "row":
            scale = torch.clamp(y.abs().max(1).values / 448, min=1e-12)
            return _e4m3(y / scale[:, None]), scale, h
        scale = torch.clamp(y.abs().max() / 448, min=1e-12).reshape(1)
        return _e4m3(y / scale), scale, h
    if c["op"] == "rotary":
        freq, gain = _frequencies(c)
        angle = s["positions"].double()[:, None] * freq
        # each pair of a head is a complex number, turned by its angle
        turn = torch.polar(torch.full_like(angle, gain), angle)[:, None]

        def turned(x):
            x = x.double()
            head, rest = x[..., :c["rot"]], x[..., c["rot"]:]
            if c["interleaved"]:
                z = torch.view_as_complex(head.unflatten(-1, (-1, 2)).contiguous()) * turn
                return torch.cat((torch.view_as_real(z).flatten(-2), rest), -1)
            z = torch.complex(*head.chunk(2, -1)) * turn
            return torch.cat((z.real, z.imag, rest), -1)

        k, v = s["k_pages"].double(), s["v_pages"].double()
        # a slot is page * size + place in it
        k = k.transpose(1, 2).flatten(0, 1).index_copy(0, s["slots"], turned(s["k"])).unflatten(0, (-1, c["page"])).transpose(1, 2)
        v = v.transpose(1, 2).flatten(0, 1).index_copy(0, s["slots"], s["v"].double()).unflatten(0, (-1, c["page"])).transpose(1, 2)
        return turned(s["q"]), k, v
    if c["op"] == "pages":
        for pool in (s["k_pages"], s["v_pages"]):
            for a, b, t in s["moves"]:
                pool[:, b, :, :t] = pool[:, a, :, :t]
        return s["k_pages"].double(), s["v_pages"].double()
    G, out = c["heads"] // c["kv_heads"], []
    for i, (new, kv) in enumerate(zip(*_lengths(c))):
        at = int(s["query_starts"][i])
        t = torch.arange(kv, device=_DEV)
        page = s["page_table"][i].long()[t // c["page"]]
        p = torch.arange(kv - new, kv, device=_DEV)[:, None] if c["causal"] else torch.full((new, 1), kv - 1, device=_DEV)
        hidden = t > p
        if c["window"]:
            hidden |= (t <= p - c["window"]) & (t >= c["sinks"])
        rows = []
        for h in range(c["heads"]):
            q = s["q"][at:at + new, h].double()
            k, v = (x[page, h // G, t % c["page"]].double() for x in (s["k_pages"], s["v_pages"]))
            a = torch.softmax((q @ k.T / math.sqrt(c["dim"])).masked_fill(hidden, -math.inf), 1)
            rows.append(torch.nan_to_num(a) @ v)
        out.append(torch.stack(rows, 1))
    return torch.cat(out)


def _e4m3(x):
    """The nearest value of 8-bit floating point with 4 exponent and 3 mantissa bits, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)
