"""Plain 64-bit statements of the 8-bit cache format and of attention over key spans, for the tests."""
import math

import torch

NOT_FINITE = -128


def quantise(x64: torch.Tensor):
    """(bytes uint8, exponents int8) of head vectors x64 [..., 128] in float64."""
    top = x64.abs().amax(-1)
    bad = ~(top < 2.0 ** 128)                              # infinite, NaN, or beyond fp32
    e = torch.full(top.shape, -126, dtype=torch.int64)
    some = (top > 0) & ~bad
    e[some] = torch.frexp(top[some])[1].long() - 1 - 6     # top = m * 2^x with m in [0.5, 1)
    e = e.clamp_min(-126)
    m = torch.round(torch.ldexp(x64.abs(), -e.unsqueeze(-1).expand_as(x64))).clamp_max(127)
    m = torch.where(bad.unsqueeze(-1), torch.zeros_like(m), m)
    held = m.to(torch.int64) + 128 * torch.signbit(x64) * ~bad.unsqueeze(-1)
    e = torch.where(bad, torch.full_like(e, NOT_FINITE), e)
    return held.to(torch.uint8), e.to(torch.int8)


def values(held: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """What bytes and exponents stand for, float64."""
    h = held.long()
    v = torch.ldexp((h & 127).double(), exps.long().unsqueeze(-1).expand_as(h)) * torch.where(h > 127, -1.0, 1.0)
    return torch.where((exps == NOT_FINITE).unsqueeze(-1), torch.full_like(v, math.nan), v)


def rope64(x: torch.Tensor, table: torch.Tensor, grid, start_frames) -> torch.Tensor:
    """x [B, N, H, 128] rotated in float64 with separately rounded products; table [rows, 64, 2] float64."""
    f, h, w = grid
    t = torch.arange(f * h * w)
    out = []
    for b, s in enumerate(start_frames):
        cs = torch.cat((table[s + t // (h * w), :22], table[(t // w) % h, 22:43], table[t % w, 43:]), 1)[:, None]
        re, im, c, d = x[b, ..., 0::2].double(), x[b, ..., 1::2].double(), cs[..., 0], cs[..., 1]
        out.append(torch.stack((re * c - im * d, re * d + im * c), -1).flatten(-2))
    return torch.stack(out)


def span_attention(q, k, v, begin, end, scale=None):
    """(out, weight) in float64 for q [B, N, H, D], k / v [B, S, H, D]: out = softmax over begin <= j < end, 0 where a span
    is empty; weight = softmax . |v|, what a relative error of the softmax weights multiplies.  Keys outside a span do not
    enter, whatever they hold."""
    B, n, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(B, n, H, D, dtype=torch.float64, device=q.device)
    weight = torch.zeros_like(out)
    key = torch.arange(k.shape[1], device=q.device)
    for b in range(B):
        inside = (key >= begin[b].to(q.device)[:, None]) & (key < end[b].to(q.device)[:, None])
        used = inside.any(0)
        some = inside[:, used].any(1)
        if not bool(some.any()):
            continue
        for h in range(H):
            kk, vv = k[b, used, h].double(), v[b, used, h].double()
            s = (q[b, some, h].double() @ kk.T) * scale
            s = s.masked_fill(~inside[some][:, used], -math.inf)
            p = torch.softmax(s, -1)
            out[b, some, h] = p @ vv
            weight[b, some, h] = p @ vv.abs()
    return out, weight


def check_attention(got: torch.Tensor, ref: torch.Tensor, weight: torch.Tensor, keys: int, what="") -> None:
    """|got - ref| <= half a bf16 step of the result (2^-8 |ref|), plus the softmax weights' own rounding to bf16
    (2^-8 of softmax . |v|), plus fp32 sums over the keys (keys * 2^-24 of it) and fp32 scores: a dot product of 128
    terms and its scaling are off by at most 129 * 2^-24 of the sum of magnitudes; for the tests' q, k of unit variance
    that sum times the scale stays under 64, so e^score is off by under 2^-10 of itself."""
    got, ref, weight = got.double().cpu(), ref.cpu(), weight.cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), (what, "finite values differ")
    fine = torch.isfinite(ref)
    allowed = 2.0 ** -8 * ref.abs() + (2.0 ** -8 + keys * 2.0 ** -24 + 2.0 ** -10) * weight + 2.0 ** -133
    over = (got - ref).abs() - allowed
    assert bool((over[fine] <= 0).all()), (what, "over by", over[fine].max().item(), "error", (got - ref).abs()[fine].max().item())
