"""Cases and plain forms of the 8-bit K/V cache operators and of attention over key spans.

Operators:
  append   `ops.rope_kv_append_q8` followed by `ops.kv_read_q8` of the slots it wrote: rope a chunk's q and k, write k
           and v into their cache slots as 8-bit magnitudes with one power-of-two exponent per (token, head), and read
           them back, as a stream does that looks at what its cache holds of the new frame
  read     `ops.kv_read_q8`: a range of the 8-bit cache as bf16
  attn     `ops.attn_kvcache_q8`: the chunk's queries over the 8-bit cache
  spans    `ops.attn_spans`: attention in which query i attends keys begin[i] .. end[i] - 1 only

The format: for x in one head vector (128 values), e = max(floor(log2(max |x|)) - 6, -126), magnitude
m = min(rint(|x| / 2^e), 127), sign beside it; the value that is held is sign * m * 2^e.  A vector with a value that is
not finite is held as NaN.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda"
D = 128
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one small frame of one stream, two heads: latency
        dict(name="append_tiny", op="append", dtype="bf16", rows=1, heads=2, grid="1x6x8", cache=336),
        # the streaming configuration: 480x832 video, two latent frames per chunk, two denoise levels, 12 heads
        dict(name="append_1p3b", op="append", dtype="bf16", rows=2, heads=12, grid="2x30x52", cache=32760),
        # four denoise levels of the 40-head model
        dict(name="append_14b", op="append", dtype="bf16", rows=4, heads=40, grid="2x30x52", cache=9360),
        # fp32 run with an odd grid and head count
        dict(name="append_fp32_odd", op="append", dtype="fp32", rows=3, heads=5, grid="3x17x29", cache=5000),
        # the three sink frames that the adaptive test compares with a new frame
        dict(name="read_sink", op="read", rows=1, heads=12, cache=9360, tokens=4680),
        # a whole cache back to bf16
        dict(name="read_window", op="read", rows=2, heads=12, cache=32760, tokens=32760),
        # one query token per row over ragged cache lengths, one of them empty
        dict(name="attn_one_token", op="attn", rows=4, heads=12, queries=1, cache=32760, lens="32760,20001,1,0"),
        # a chunk of odd size over partly filled caches
        dict(name="attn_odd", op="attn", rows=3, heads=5, queries=1479, cache=9000, lens="8999,4111,130"),
        # the streaming configuration's chunk over the full window
        dict(name="attn_1p3b", op="attn", rows=2, heads=12, queries=3120, cache=32760, lens="32760,32760"),
        # a clip of nine frames without a cache: every three-frame block sees itself and what came before
        dict(name="spans_clip", op="spans", rows=1, heads=12, queries=14040, keys=14040, mask="blocks", blocks="4680,4680,4680"),
        # text cross-attention with prompts of different lengths, one of them empty
        dict(name="spans_text", op="spans", rows=4, heads=12, queries=3120, keys=512, mask="lens", lens="512,77,226,0"),
        # small clips packed into one row, each attending itself only
        dict(name="spans_packed", op="spans", rows=1, heads=3, queries=1001, keys=1001, mask="docs", blocks="300,1,444,77,179"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _pieces(rng, total):
    sizes = []
    while total > 0:
        n = min(total, _log(rng, 1, total + 1))
        sizes.append(n)
        total -= n
    rng.shuffle(sizes)
    return ",".join(str(s) for s in sizes)


def draw(rng):
    op = rng.choice(("append", "read", "attn", "attn", "spans", "spans"))
    rows, heads = rng.randint(1, 4), rng.randint(1, 16)
    if op == "append":
        f, h, w = rng.randint(1, 3), _log(rng, 1, 30), _log(rng, 1, 52)
        n = f * h * w
        return dict(op=op, dtype=rng.choice(("bf16", "bf16", "fp32")), rows=rows, heads=heads, grid="%dx%dx%d" % (f, h, w),
                    cache=n + _log(rng, 1, 8000))
    cache = _log(rng, 1, 32760)
    if op == "read":
        return dict(op=op, rows=rng.randint(1, 2), heads=rng.randint(1, 12), cache=cache, tokens=max(1, cache - _log(rng, 1, cache + 1)))
    queries = _log(rng, 1, 3120)
    if op == "attn":
        lens = [rng.choice((cache, rng.randint(0, cache), _log(rng, 1, cache + 1) - 1)) for _ in range(rows)]
        return dict(op=op, rows=rows, heads=rng.randint(1, 6), queries=queries, cache=cache, lens=",".join(map(str, lens)))
    mask = rng.choice(("blocks", "lens", "docs", "free"))
    heads = rng.randint(1, 6)
    if mask in ("blocks", "docs"):
        n = _log(rng, 1, 8000)
        return dict(op=op, rows=rng.randint(1, 2), heads=heads, queries=n, keys=n, mask=mask, blocks=_pieces(rng, n))
    keys = _log(rng, 1, 8000)
    if mask == "lens":
        return dict(op=op, rows=rows, heads=heads, queries=queries, keys=keys, mask=mask,
                    lens=",".join(str(rng.randint(0, keys)) for _ in range(rows)))
    return dict(op=op, rows=rows, heads=heads, queries=queries, keys=keys, mask=mask, span_seed=rng.randint(0, 1 << 20))


def _ints(text):
    return [int(t) for t in text.split(",")]


def _spans(case):
    """begin, end: int64 arrays [rows, queries]."""
    rows, n, keys = case["rows"], case["queries"], case["keys"]
    if case["mask"] == "lens":
        end = np.repeat(np.array(_ints(case["lens"]))[:, None], n, 1)
        return np.zeros_like(end), end
    if case["mask"] == "free":                     # any begin and end, a tenth of the rows empty
        r = np.random.RandomState(case["span_seed"])
        a, b = r.randint(0, keys + 1, (rows, n)), r.randint(0, keys + 1, (rows, n))
        begin, end = np.minimum(a, b), np.maximum(a, b)
        end[r.rand(rows, n) < 0.1] = 0
        return begin, end
    sizes = np.array(_ints(case["blocks"]))
    ends = np.repeat(np.cumsum(sizes), sizes)[None].repeat(rows, 0)
    return (np.zeros_like(ends) if case["mask"] == "blocks" else ends - np.repeat(sizes, sizes)[None]), ends


def work(case):
    rows, heads, op = case["rows"], case["heads"], case["op"]
    if op == "append":
        vecs = rows * heads * int(np.prod([int(t) for t in case["grid"].split("x")]))
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": vecs * (D * size * 4 + 2 * (D + 1) + 2 * (D + 1) + 2 * D * 2), "flops": vecs * D * 10}
    if op == "read":
        return {"bytes": rows * heads * case["tokens"] * 2 * (D + 1 + 2 * D), "flops": rows * heads * case["tokens"] * D * 2}
    n = case["queries"]
    if op == "attn":
        lens = _ints(case["lens"])
        return {"bytes": rows * n * heads * D * 4 + sum(lens) * heads * 2 * (D + 1), "flops": 4 * D * heads * n * sum(lens)}
    begin, end = _spans(case)
    return {"bytes": rows * (n + case["keys"]) * heads * D * 4 + rows * n * 8,
            "flops": 4 * D * heads * int(np.maximum(end - begin, 0).sum())}


# ------------------------------------------------------------------------------------------------ inputs
def _quantise(x):
    """Magnitudes with signs (uint8, sign in the top bit) and exponents (int8) of head vectors of finite values."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    e = (torch.frexp(top).exponent - 1 - 6).clamp_min(-126)
    e = torch.where(top > 0, e, torch.full_like(e, -126))
    m = torch.round(x.abs() * torch.exp2(-e.double())).clamp_max(127)
    return (m + 128 * (x < 0)).to(torch.uint8), e.squeeze(-1).to(torch.int8)


def _rope_table(positions=1024):
    """[positions, 64, 2] cos and sin: 22 columns for time, 21 each for height and width."""
    def unit(dim):
        inv = 1.0 / torch.pow(10000.0, torch.arange(0, dim, 2, dtype=torch.float64, device=DEVICE) / dim)
        a = torch.arange(positions, dtype=torch.float64, device=DEVICE)[:, None] * inv
        return torch.stack((a.cos(), a.sin()), -1)
    return torch.cat([unit(44), unit(42), unit(42)], 1).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)  # noqa: E731
    rows, heads, op = case["rows"], case["heads"], case["op"]
    s = {"case": case}
    if op == "append":
        grid = [int(t) for t in case["grid"].split("x")]
        n, cache = int(np.prod(grid)), case["cache"]
        r = np.random.RandomState(int(seed) % (1 << 31))
        s["q"], s["k"], s["v"] = (rnd(rows, n, 3, heads, D) * torch.exp(rnd(1, 1, 3, heads, D))).to(TYPES[case["dtype"]]).unbind(2)
        s["grid"], s["table"] = grid, _rope_table()
        s["frames"] = [int(t) for t in r.randint(0, 1024 - grid[0] + 1, rows)]
        s["slots"] = [int(t) for t in r.randint(0, cache - n + 1, rows)]
        for name in ("k", "v"):
            s[name + "_cache"] = torch.zeros(rows, cache, heads, D, dtype=torch.uint8, device=DEVICE)
            s[name + "_exp"] = torch.zeros(rows, cache, heads, dtype=torch.int8, device=DEVICE)
        return s
    if op in ("read", "attn"):
        cache = case["cache"]
        s["k_cache"], s["k_exp"] = _quantise(rnd(rows, cache, heads, D) * torch.exp(0.5 * rnd(1, 1, heads, D)))
        s["v_cache"], s["v_exp"] = _quantise(rnd(rows, cache, heads, D) * torch.exp(rnd(rows, cache, heads, 1)))
        if op == "read":
            s["begin"] = [cache - case["tokens"]] * rows
        else:
            s["q"] = rnd(rows, case["queries"], heads, D).to(torch.bfloat16)
            s["lens"] = _ints(case["lens"])
        return s
    s["q"], s["k"], s["v"] = (rnd(rows, m, heads, D).to(torch.bfloat16) for m in (case["queries"], case["keys"], case["keys"]))
    s["begin"], s["end"] = (torch.from_numpy(t.astype(np.int32)).to(DEVICE) for t in _spans(case))
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _value(held, exp):
    """What 8-bit magnitudes and exponents stand for, fp32."""
    m = (held & 127).float() * torch.exp2(exp.float())[..., None]
    return torch.where(held >= 128, -m, m)


def _slots(t, begin, n):
    at = torch.tensor(begin, device=t.device)[:, None] + torch.arange(n, device=t.device)
    return t[torch.arange(t.shape[0], device=t.device)[:, None], at]


def _rotate(x, cs):
    a, b, c, d = x[..., 0::2].double(), x[..., 1::2].double(), cs[..., 0], cs[..., 1]
    return torch.stack((a * c - b * d, a * d + b * c), -1).flatten(-2)


def _plain_append(s):
    f, h, w = s["grid"]
    t = torch.arange(f * h * w, device=DEVICE)
    frame = torch.tensor(s["frames"], device=DEVICE)[:, None] + t // (h * w)
    table = s["table"]
    cs = torch.cat((table[frame, :22], table[(t // w) % h, 22:43].expand(len(s["frames"]), -1, -1, -1),
                    table[t % w, 43:].expand(len(s["frames"]), -1, -1, -1)), 2)[:, :, None]
    held_k, exp_k = _quantise(_rotate(s["k"], cs))
    held_v, exp_v = _quantise(s["v"])
    at = torch.tensor(s["slots"], device=DEVICE)[:, None] + t
    row = torch.arange(len(s["slots"]), device=DEVICE)[:, None]
    for name, held, exp in (("k", held_k, exp_k), ("v", held_v, exp_v)):
        s[name + "_cache"][row, at], s[name + "_exp"][row, at] = held, exp
    return {"q": _rotate(s["q"], cs).to(s["q"].dtype), "k": _value(held_k, exp_k).to(torch.bfloat16),
            "v": _value(held_v, exp_v).to(torch.bfloat16)}


def _plain_attention(q, k, v, mask):
    """q [B, N, H, D], k and v [B, S, H, D] in fp32; mask [B, N or 1, S]; rows without a key give zeros."""
    scores = torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(D))
    scores = scores.masked_fill(~mask[:, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2)) / torch.where(total > 0, total, torch.ones_like(total))
    return out.transpose(1, 2).to(torch.bfloat16)


def run(s):
    op = s["case"]["op"]
    if own:
        from streamdiffusionv2_b200 import ops
        if op == "append":
            q = ops.rope_kv_append_q8(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["table"],
                                      s["grid"], s["frames"], s["slots"])
            k, v = ops.kv_read_q8(s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["slots"], s["q"].shape[1])
            return {"q": q, "k": k, "v": v}
        if op == "read":
            k, v = ops.kv_read_q8(s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["begin"], s["case"]["tokens"])
            return {"k": k, "v": v}
        if op == "attn":
            return {"out": ops.attn_kvcache_q8(s["q"], s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["lens"])}
        return {"out": ops.attn_spans(s["q"], s["k"], s["v"], s["begin"], s["end"])}
    if op == "append":
        return _plain_append(s)
    if op == "read":
        n = s["case"]["tokens"]
        return {c: _value(_slots(s[c + "_cache"], s["begin"], n), _slots(s[c + "_exp"], s["begin"], n)).to(torch.bfloat16)
                for c in ("k", "v")}
    if op == "attn":
        mask = torch.arange(s["case"]["cache"], device=DEVICE) < torch.tensor(s["lens"], device=DEVICE)[:, None, None]
        return {"out": _plain_attention(s["q"].float(), _value(s["k_cache"], s["k_exp"]), _value(s["v_cache"], s["v_exp"]), mask)}
    key = torch.arange(s["case"]["keys"], device=DEVICE)
    mask = (key >= s["begin"][..., None]) & (key < s["end"][..., None])
    return {"out": _plain_attention(s["q"].float(), s["k"].float(), s["v"].float(), mask)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _held64(x):
    """The values that the format holds of head vectors x, from its definition."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    exp = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    exp = torch.where(torch.exp2(exp) > top, exp - 1, exp)
    exp = torch.where(torch.exp2(exp + 1) <= top, exp + 1, exp)
    step = torch.exp2((exp - 6).clamp_min(-126))
    return (x / step).round().clamp(-127, 127) * step


def exact(case, seed):
    s = prepare(case, seed)
    op, heads, rows = case["op"], case["heads"], case["rows"]
    if op == "append":
        f, h, w = s["grid"]
        inv = [10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEVICE) / d) for d in (44, 42, 42)]
        ar = lambda n: torch.arange(n, dtype=torch.float64, device=DEVICE)  # noqa: E731
        out = {"q": [], "k": [], "v": []}
        for b in range(rows):
            angle = torch.cat([((ar(f) + s["frames"][b])[:, None, None, None] * inv[0]).expand(f, h, w, 22),
                               (ar(h)[None, :, None, None] * inv[1]).expand(f, h, w, 21),
                               (ar(w)[None, None, :, None] * inv[2]).expand(f, h, w, 21)], -1).reshape(f * h * w, 1, 64)
            turn = torch.polar(torch.ones_like(angle), angle)
            turned = [torch.view_as_real(torch.view_as_complex(s[c][b].double().unflatten(-1, (64, 2)).contiguous()) * turn).flatten(-2)
                      for c in ("q", "k")]
            out["q"].append(turned[0])
            out["k"].append(_held64(turned[1]))
            out["v"].append(_held64(s["v"][b]))
        return {c: torch.stack(t) for c, t in out.items()}
    held = lambda c: torch.where(s[c + "_cache"] > 127, 128.0 - s[c + "_cache"].double(), s[c + "_cache"].double()) \
        * torch.pow(2.0, s[c + "_exp"].double())[..., None]  # noqa: E731
    if op == "read":
        return {c: held(c)[:, case["cache"] - case["tokens"]:] for c in ("k", "v")}
    k, v = (held("k"), held("v")) if op == "attn" else (s["k"].double(), s["v"].double())
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    for b in range(rows):
        if op == "attn":
            n = s["lens"][b]
            inside = torch.ones(1, n, dtype=torch.bool, device=DEVICE)
        else:
            n = case["keys"]
            at = torch.arange(n, device=DEVICE)
            inside = (at >= s["begin"][b][:, None]) & (at < s["end"][b][:, None])
        some = inside.any(-1, keepdim=True)
        for hd in range(heads):
            if n == 0:
                continue
            z = (s["q"][b, :, hd].double() @ k[b, :n, hd].T) / math.sqrt(D)
            z = torch.where(inside, z, torch.full_like(z, -math.inf))
            z = torch.where(some, torch.exp(z - torch.logsumexp(torch.where(some, z, torch.zeros_like(z)), -1, keepdim=True)), torch.zeros_like(z))
            out[b, :, hd] = z @ v[b, :n, hd]
    return {"out": out}
