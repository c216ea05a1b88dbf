"""The 8-bit K/V cache (append, read back, attention) and attention over key spans against 64-bit statements of them."""
import pytest
import torch

import q8_reference as ref
from oracle import causal_attention_oracle as orc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ops():
    from streamdiffusionv2_b200 import ops
    return ops


def _table():
    return torch.view_as_real(orc.rope_table(128)).contiguous()


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def _garbage_cache(rows, tokens, heads, seed=99):
    g = torch.Generator().manual_seed(seed)
    c = {n: torch.randint(0, 256, (rows, tokens, heads, 128), generator=g, dtype=torch.uint8) for n in ("k", "v")}
    c.update({n: torch.randint(-128, 128, (rows, tokens, heads), generator=g, dtype=torch.int8) for n in ("k_exp", "v_exp")})
    return c


def _cuda(c):
    return {n: t.to(DEV) for n, t in c.items()}


def _append(c, q, k, v, grid, frames, slots, **kw):
    return _ops().rope_kv_append_q8(q, k, v, c["k"], c["v"], c["k_exp"], c["v_exp"], _table().to(DEV), grid, frames, slots, **kw)


def _expected(c, k, v, grid, frames, slots):
    want = {n: t.clone() for n, t in c.items()}
    held = {"k": ref.quantise(ref.rope64(k, _table(), grid, frames)), "v": ref.quantise(v.double())}
    n = k.shape[1]
    for name, (m, e) in held.items():
        for b, s in enumerate(slots):
            want[name][b, s:s + n], want[name + "_exp"][b, s:s + n] = m[b], e[b]
    return want


def _same_cache(got, want):
    for name in want:
        assert torch.equal(got[name].cpu(), want[name]), name


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,heads,grid,frames,slots,cache", [
    (1, 1, (1, 1, 1), [0], [0], 1),                       # one token, one head, a cache of one
    (1, 2, (1, 6, 8), [1023], [7], 60),                   # last frame of the table
    (2, 5, (2, 3, 7), [0, 400], [0, 58], 100),            # odd head count; second row ends at the cache's end
    (3, 12, (1, 5, 9), [5, 6, 7], [1, 2, 3], 64),
    (2, 40, (1, 2, 3), [9, 2], [10, 0], 16),
])
def test_append_writes_the_format_bit_for_bit(dtype, rows, heads, grid, frames, slots, cache):
    """Bytes and exponents of the slots, and nothing outside them; q as rope_kv_append ropes it."""
    ops = _ops()
    n = grid[0] * grid[1] * grid[2]
    x = (_randn(3, rows, n, 3, heads, 128) * torch.exp(3 * _randn(4, rows, n, 3, heads, 1))).to(dtype)
    q, k, v = x.unbind(2)                                  # slices of one fused projection
    c = _garbage_cache(rows, cache, heads)
    want = _expected(c, k, v, grid, frames, slots)
    got = _cuda(c)
    qd, kd, vd = x.to(DEV).unbind(2)
    q_out = _append(got, qd, kd, vd, grid, frames, slots)
    _same_cache(got, want)
    kc, vc = (torch.zeros(rows, cache, heads, 128, dtype=dtype, device=DEV) for _ in range(2))
    assert torch.equal(q_out, ops.rope_kv_append(qd, kd, vd, kc, vc, _table().to(DEV), grid, frames, slots))
    ops.read_status(torch.device(DEV))


@pytest.mark.parametrize("grid", [(3, 1, 1), (2, 5, 1), (1, 7, 1), (2, 1, 6), (3, 4, 1)])
def test_appends_of_grids_one_token_wide_or_high(grid):
    """Frames, rows and columns of one: the 8-bit append against its statement, and the plain append's keys and queries
    against the 64-bit rope rounded once."""
    n = grid[0] * grid[1] * grid[2]
    q, k, v = (_randn(s, 2, n, 3, 128) for s in (1, 2, 3))
    c = _garbage_cache(2, n + 9, 3)
    want = _expected(c, k, v, grid, [5, 100], [4, 0])
    d = _cuda(c)
    q_out = _append(d, q.to(DEV), k.to(DEV), v.to(DEV), grid, [5, 100], [4, 0])
    _same_cache(d, want)
    kc = torch.zeros(2, n, 3, 128, device=DEV)
    vc = torch.zeros_like(kc)
    q_plain = _ops().rope_kv_append(q.to(DEV), k.to(DEV), v.to(DEV), kc, vc, _table().to(DEV), grid, [5, 100], [0, 0])
    assert torch.equal(kc.cpu(), ref.rope64(k, _table(), grid, [5, 100]).float()) and torch.equal(vc.cpu(), v)
    assert torch.equal(q_out, q_plain) and torch.equal(q_out.cpu(), ref.rope64(q, _table(), grid, [5, 100]).float())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_special_values(dtype):
    """Zeros, subnormals, the largest finite values, infinities and NaN, values on rounding ties and above 127.5 steps."""
    x = _randn(1, 1, 16, 3, 2, 128)
    x[0, 0] = 0.0
    x[0, 1] *= 2.0 ** -130
    x[0, 2] = torch.finfo(dtype).max
    x[0, 3, :, 0, 5], x[0, 4, :, 1, 127], x[0, 5, :, 0, 0] = float("inf"), float("nan"), float("-inf")
    x[0, 6] = torch.arange(-64, 64).float() + 0.5          # ties at a step of 1
    x[0, 6, ..., 0] = 127.9                                # above 127.5 steps
    x[0, 7, ..., ::2] = 0.0
    x[0, 8] *= 2.0 ** 120
    x[0, 9] = -0.0
    x[0, 10] = 2.0 ** -126
    x[0, 11] = 2.0 ** torch.arange(-64, 64).float()
    x = x.to(dtype)
    q, k, v = x.unbind(2)
    grid, frames, slots = (1, 4, 4), [3], [2]
    c = _garbage_cache(1, 20, 2)
    want = _expected(c, k, v, grid, frames, slots)
    got = _cuda(c)
    qd, kd, vd = x.to(DEV).unbind(2)
    _append(got, qd, kd, vd, grid, frames, slots)
    _same_cache(got, want)


def test_append_strided_caches_indices_and_device_parameters():
    """Caches and exponents as slices of larger tensors with their heads apart; parameters by value and from the device."""
    ops = _ops()
    rows, heads, grid, n, cache = 2, 3, (2, 2, 5), 20, 50
    q, k, v = (_randn(s, rows, n, heads, 128).to(torch.bfloat16) for s in (1, 2, 3))
    frames, slots = [4, 900], [30, 1]
    qd, kd, vd = (t.to(DEV) for t in (q, k, v))
    c = _garbage_cache(rows, cache, heads)
    want = _expected(c, k, v, grid, frames, slots)
    for indirect in (False, True):
        big = {n_: torch.zeros((rows, cache + 3, 2 * heads) + t.shape[3:], dtype=t.dtype, device=DEV) for n_, t in c.items()}
        got = {n_: big[n_][:, 1:cache + 1, ::2] for n_ in c}
        for n_ in c:
            got[n_].copy_(c[n_])
        idx = [torch.zeros(rows, dtype=torch.int64, device=DEV) for _ in range(2)]
        kw = {"index_tensors": tuple(idx)}
        if indirect:
            kw["step_params"] = torch.tensor([frames, slots, [77, 78], [20, 21]], device=DEV)
            _append(got, qd, kd, vd, grid, [0, 0], [0, 0], **kw)
        else:
            _append(got, qd, kd, vd, grid, frames, slots, index_values=([77, 78], [20, 21]), **kw)
        _same_cache(got, want)
        assert idx[0].tolist() == [77, 78] and idx[1].tolist() == [20, 21]
        for n_ in c:                                       # the neighbours stay as they were
            assert not bool(big[n_][:, :, 1::2].any()) and not bool(big[n_][:, 0].any()) and not bool(big[n_][:, -2:].any())
    ops.read_status(torch.device(DEV))


def test_append_refuses_bad_device_parameters_and_writes_nothing():
    from streamdiffusionv2_b200 import _native as N
    ops = _ops()
    q = _randn(1, 2, 6, 2, 128).to(torch.bfloat16).to(DEV)
    for params in ([[0, 0], [0, 5], [1, 1], [1, 1]], [[0, 0], [0, -1], [1, 1], [1, 1]], [[0, 1023], [0, 0], [1, 1], [1, 1]]):
        c = _garbage_cache(2, 10, 2)
        got = _cuda(c)
        idx = tuple(torch.zeros(2, dtype=torch.int64, device=DEV) for _ in range(2))
        _append(got, q, q.clone(), q.clone(), (2, 1, 3), [0, 0], [0, 0], index_tensors=idx,
                step_params=torch.tensor(params, device=DEV))
        with pytest.raises(N.NativeError):
            ops.read_status(torch.device(DEV))
        _same_cache(got, c)
        assert idx[0].tolist() == [0, 0]


# ------------------------------------------------------------------------------------------------ read back
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,heads,cache,begin,tokens", [
    (1, 1, 1, [0], 1), (2, 3, 40, [5, 39], 1), (2, 12, 77, [0, 0], 77), (3, 40, 33, [1, 2, 30], 3), (1, 64, 9, [2], 7),
])
def test_read_back_is_exact(dtype, rows, heads, cache, begin, tokens):
    c = _garbage_cache(rows, cache, heads)
    for n in ("k_exp", "v_exp"):
        c[n] = torch.where(c[n] > -127, c[n].clamp_max(121), torch.full_like(c[n], -128))
    got = _ops().kv_read_q8(*(t.to(DEV) for t in (c["k"], c["v"], c["k_exp"], c["v_exp"])), begin, tokens, dtype=dtype)
    for name, g in zip(("k", "v"), got):
        want = torch.stack([ref.values(c[name][b, s:s + tokens], c[name + "_exp"][b, s:s + tokens]) for b, s in enumerate(begin)])
        assert g.dtype == dtype and torch.equal(torch.isnan(g.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(g.double().cpu()), torch.nan_to_num(want)), name


def test_read_back_of_broadcast_rows_into_strided_tensors():
    ops = _ops()
    c = _garbage_cache(1, 20, 2)
    for n in ("k_exp", "v_exp"):
        c[n] = c[n].clamp(-126, 121)
    d = _cuda(c)
    wide = [t.expand(3, *t.shape[1:]) for t in (d["k"], d["v"], d["k_exp"], d["v_exp"])]
    buf = torch.zeros(3, 8, 4, 128, dtype=torch.bfloat16, device=DEV)
    k, v = ops.kv_read_q8(*wide, [3, 0, 12], 8, out=(buf[:, :, ::2], buf[:, :, 1::2]))
    for b, s in enumerate([3, 0, 12]):
        assert torch.equal(k[b].double().cpu(), ref.values(c["k"][0, s:s + 8], c["k_exp"][0, s:s + 8]))
        assert torch.equal(v[b].double().cpu(), ref.values(c["v"][0, s:s + 8], c["v_exp"][0, s:s + 8]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_read_back_into_tensors_aligned_to_16_bytes_only(dtype):
    ops = _ops()
    c = _garbage_cache(2, 30, 3)
    for n in ("k_exp", "v_exp"):
        c[n] = c[n].clamp(-126, 121)
    d = _cuda(c)
    pad = 128 // torch.finfo(dtype).bits                  # elements in 16 bytes
    flat = torch.zeros(2 * 2 * 30 * (3 * 128 + pad) + pad, dtype=dtype, device=DEV)
    out = [flat[pad + i * 30 * 2 * (3 * 128 + pad):].as_strided((2, 30, 3, 128), (30 * (384 + pad), 384 + pad, 128, 1)) for i in range(2)]
    assert out[0].data_ptr() % 32 == 16
    k, v = ops.kv_read_q8(d["k"], d["v"], d["k_exp"], d["v_exp"], [0, 0], 30, dtype=dtype, out=out)
    assert torch.equal(k.double().cpu(), ref.values(c["k"], c["k_exp"])) and torch.equal(v.double().cpu(), ref.values(c["v"], c["v_exp"]))


# ------------------------------------------------------------------------------------------------ attention, 8 bits
def _held_cache(rows, tokens, heads, seed, spread=0.0):
    """A cache that holds unit-variance K and V whose head vectors' scales differ by factors of e^spread."""
    c = {}
    for i, n in enumerate(("k", "v")):
        x = _randn(seed + i, rows, tokens, heads, 128)
        if n == "v" and spread:
            x = x * torch.exp(spread * _randn(seed + 7, rows, tokens, heads, 1))
        c[n], c[n + "_exp"] = ref.quantise(x.double())
    return c


def _check_q8(c, q, lens, out, scale=None):
    k, v = (ref.values(c[n], c[n + "_exp"]) for n in ("k", "v"))
    end = torch.tensor(lens)[:, None].expand(-1, q.shape[1])
    want, weight = ref.span_attention(q.to(DEV), k.to(DEV), v.to(DEV), torch.zeros_like(end), end, scale)
    ref.check_attention(out, want, weight, k.shape[1], lens)


@pytest.mark.parametrize("queries,heads,cache,lens", [
    (1, 1, 1, [1]), (1, 2, 130, [130, 0]), (1, 12, 5000, [5000, 4999, 1, 0]), (2, 3, 300, [129]), (16, 2, 2000, [1999, 1]),
    (17, 2, 300, [299, 16]), (32, 3, 3111, [3111, 64, 15]), (33, 1, 200, [200]), (5, 70, 400, [400, 399, 17, 0, 128]),
    (48, 2, 700, [127, 128, 129]), (100, 2, 300, [300]), (128, 1, 128, [128]), (129, 1, 256, [255]), (256, 2, 1000, [1000, 517]),
    (257, 1, 640, [640]), (300, 3, 1100, [1000, 0, 1100, 3]), (1479, 5, 2100, [2047, 2048]), (3120, 2, 4680, [4680]),
    (700, 40, 600, [600, 385]),                            # more tiles than multiprocessors: whole tiles and a split tail
    (300, 20, 9000, [9000, 700, 64, 8999, 0]),             # whole tiles, tail tiles of different rows and part counts
])
def test_q8_attention(queries, heads, cache, lens):
    ops = _ops()
    c = _held_cache(len(lens), cache, heads, 11, spread=1.0)
    q = _randn(5, len(lens), queries, heads, 128).to(torch.bfloat16)
    d = _cuda(c)
    out = ops.attn_kvcache_q8(q.to(DEV), d["k"], d["v"], d["k_exp"], d["v_exp"], lens)
    _check_q8(c, q, lens, out)
    ops.read_status(torch.device(DEV))


def test_q8_attention_ignores_what_lies_behind_the_length():
    """Uninitialised slots: any bytes, exponents that read as NaN."""
    ops = _ops()
    lens = [1, 200, 333]
    c = _held_cache(3, 512, 2, 3)
    junk = _garbage_cache(3, 512, 2)
    for b, n in enumerate(lens):
        for name in c:
            c[name][b, n:] = junk[name][b, n:]
        c["v_exp"][b, n:n + 3] = -128
        c["k_exp"][b, n] = -128
    q = _randn(5, 3, 140, 2, 128).to(torch.bfloat16)
    d = _cuda(c)
    out = ops.attn_kvcache_q8(q.to(DEV), d["k"], d["v"], d["k_exp"], d["v_exp"], lens)
    assert bool(torch.isfinite(out).all())
    _check_q8(c, q, lens, out)


@pytest.mark.parametrize("queries", [1, 32, 33, 900])
def test_q8_attention_ignores_junk_behind_the_length_and_in_scratch(queries):
    """As above for few queries and for many, whose bf16 scratch takes over memory that was full of NaN."""
    ops = _ops()
    lens = [1, 0, 500, 333]
    c = _held_cache(4, 512, 2, 4)
    junk = _garbage_cache(4, 512, 2)
    for b, n in enumerate(lens):
        for name in c:
            c[name][b, n:] = junk[name][b, n:]
        c["v_exp"][b, n:] = -128
        c["k_exp"][b, n:] = -128
    q = _randn(5, 4, queries, 2, 128).to(torch.bfloat16)
    d, qd = _cuda(c), q.to(DEV)
    dirt = [torch.full((n >> 2,), float("nan"), device=DEV) for n in (4 << 20, 2 << 20, 1 << 20, 512 << 10) for _ in range(4)]
    del dirt
    out = ops.attn_kvcache_q8(qd, d["k"], d["v"], d["k_exp"], d["v_exp"], lens)
    assert bool(torch.isfinite(out).all()) and not out[1].any()
    _check_q8(c, q, lens, out)


@pytest.mark.parametrize("queries,heads,lens", [
    (1, 40, [3000] + [100] * 15), (20, 30, [5, 2900, 0, 1, 260, 3000] + [64] * 8), (130, 12, [70, 3000] + [200] * 14),
    (900, 5, [4000] + [130] * 11),
])
def test_q8_attention_rows_far_longer_than_the_others(queries, heads, lens):
    """More tiles than fit the GPU at a time: the long rows are cut up, the others run whole."""
    ops = _ops()
    c = _held_cache(len(lens), max(lens), heads, 12, spread=1.0)
    q = _randn(5, len(lens), queries, heads, 128).to(torch.bfloat16)
    d = _cuda(c)
    _check_q8(c, q, lens, ops.attn_kvcache_q8(q.to(DEV), d["k"], d["v"], d["k_exp"], d["v_exp"], lens))


def test_q8_attention_in_groups_of_heads():
    """Many queries over a cache too large to expand at once: 23 heads in groups of 12 and 11, one row nearly empty."""
    ops = _ops()
    S, H, n, lens = 50000, 23, 800, [50000, 3]
    g = torch.Generator(DEV).manual_seed(7)
    d = {x: torch.randint(0, 256, (2, S, H, 128), generator=g, dtype=torch.uint8, device=DEV) for x in ("k", "v")}
    d.update({x + "_exp": torch.randint(-8, -5, (2, S, H), generator=g, dtype=torch.int8, device=DEV) for x in ("k", "v")})
    q = torch.randn(2, n, H, 128, generator=g, device=DEV).to(torch.bfloat16)
    out = ops.attn_kvcache_q8(q, d["k"], d["v"], d["k_exp"], d["v_exp"], lens)
    some = [0, 11, 12, 22]
    for b, end in enumerate(lens):
        for h in some:                                     # the reference in 64 bits, a head at a time
            k, v = (ref.values(d[x][b:b + 1, :end, h:h + 1], d[x + "_exp"][b:b + 1, :end, h:h + 1]) for x in ("k", "v"))
            hi = torch.full((1, n), end)
            want, weight = ref.span_attention(q[b:b + 1, :, h:h + 1], k, v, torch.zeros_like(hi), hi, None)
            ref.check_attention(out[b:b + 1, :, h:h + 1], want, weight, end, [end])


@pytest.mark.parametrize("queries", [1, 200])
def test_q8_attention_exponents_far_apart(queries):
    """V scales that grow and shrink along the cache by 2^100 (the accumulator changes its unit), a V that is 0 for
    whole tiles, K vectors 2^40 smaller than their neighbours; NaN in one head only."""
    ops = _ops()
    S, H = 1500, 3
    c = _held_cache(1, S, H, 21)
    at = torch.arange(S)
    c["v_exp"][0, :, 0] = (c["v_exp"][0, :, 0] + (at // 128) * 8 - 50).to(torch.int8)      # grows tile by tile
    c["v_exp"][0, :, 1] = (c["v_exp"][0, :, 1] + 50 - (at // 128) * 8).to(torch.int8)      # shrinks
    c["v"][0, 128:512, 1], c["v_exp"][0, 128:512, 1] = 0, -126
    c["v"][0, 0:256, 0], c["v_exp"][0, 0:256, 0] = 0, -126
    c["k_exp"][0, ::3] -= 40
    c["v_exp"][0, 700, 2] = -128
    q = _randn(6, 1, queries, H, 128).to(torch.bfloat16)
    d = _cuda(c)
    out = ops.attn_kvcache_q8(q.to(DEV), d["k"], d["v"], d["k_exp"], d["v_exp"], [S])
    assert bool(torch.isnan(out[:, :, 2]).all())
    sub = {n: t[:, :, :2] for n, t in c.items()}
    _check_q8(sub, q[:, :, :2], [S], out[:, :, :2])


@pytest.mark.parametrize("queries", [3, 40])
def test_q8_attention_queries_far_apart_and_not_finite(queries):
    """A query row that is huge, lowest-valued or not finite changes no other row; V near bf16's largest value."""
    ops = _ops()
    S = 300
    c = _held_cache(1, S, 2, 77)
    c["v_exp"][:, :, 1] = 121
    q = _randn(6, 1, queries, 2, 128).to(torch.bfloat16)
    clean = q.clone()
    q[0, 0] = torch.finfo(torch.bfloat16).min
    q[0, 1, 0, 5], q[0, 1, 1, 7] = float("inf"), float("nan")
    d = _cuda(c)
    args = (d["k"], d["v"], d["k_exp"], d["v_exp"], [S])
    out, want = (ops.attn_kvcache_q8(t.to(DEV), *args) for t in (q, clean))
    assert torch.equal(out[:, 2:], want[:, 2:])
    assert bool(torch.isnan(out[:, 1]).any(-1).all()) and bool(torch.isfinite(want).all())
    k, v = (ref.values(c[n], c[n + "_exp"]) for n in ("k", "v"))
    end = torch.full((1, queries), S)
    exact, weight = ref.span_attention(clean.to(DEV), k.to(DEV), v.to(DEV), torch.zeros_like(end), end)
    ref.check_attention(want, exact, weight, S)


def test_q8_attention_strided_views_scale_and_growing_logits():
    ops = _ops()
    B, n, H, S = 2, 300, 2, 900
    c = _held_cache(B, S, H, 31)
    ramp = (torch.arange(S) // 300).to(torch.int8)          # K grows along the cache: the running maximum moves
    c["k_exp"] += ramp[None, :, None]
    big = {name: torch.zeros((B, S + 40, 3 * H) + t.shape[3:], dtype=t.dtype, device=DEV) for name, t in c.items()}
    view = {name: t[:, 20:S + 20, 1::3] for name, t in big.items()}
    for name in c:
        view[name].copy_(c[name])
    qkv = _randn(8, B, n, 3, H, 128).to(torch.bfloat16)
    buf = torch.zeros(B, n + 1, 2 * H, 128, dtype=torch.bfloat16, device=DEV)
    out = ops.attn_kvcache_q8(qkv.to(DEV)[:, :, 1], view["k"], view["v"], view["k_exp"], view["v_exp"], [S, S - 33],
                              out=buf[:, 1:, ::2], softmax_scale=0.05)
    _check_q8(c, qkv[:, :, 1], [S, S - 33], out, scale=0.05)
    assert not bool(buf[:, 0].any()) and not bool(buf[:, :, 1::2].any())


@pytest.mark.parametrize("queries", [1, 100, 900])
def test_q8_attention_cache_rows_broadcast_and_heads_outermost(queries):
    """The three ways the attention runs (few queries, expanded in the kernel, expanded first) over one cache row shared by
    all rows, and over caches whose heads lie outside the tokens."""
    ops = _ops()
    S, H = 333, 3
    c = _held_cache(1, S, H, 41, spread=1.0)
    q = _randn(9, 2, queries, H, 128).to(torch.bfloat16)
    lens = [333, 150]
    wide = {n: t.to(DEV).expand(2, *t.shape[1:]) for n, t in c.items()}
    out = ops.attn_kvcache_q8(q.to(DEV), wide["k"], wide["v"], wide["k_exp"], wide["v_exp"], lens)
    full = {n: t.expand(2, *t.shape[1:]) for n, t in c.items()}
    _check_q8(full, q, lens, out)
    outer = {n: t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for n, t in full.items()}
    out = ops.attn_kvcache_q8(q.to(DEV).transpose(1, 2).contiguous().transpose(1, 2), outer["k"], outer["v"], outer["k_exp"],
                              outer["v_exp"], lens)
    _check_q8(full, q, lens, out)


@pytest.mark.parametrize("queries", [2, 40, 800])
def test_8_bit_cache_with_offsets_past_32_bits(queries):
    """Tokens 5 MB apart: 1100 of them reach past 2^32 bytes.  Written, read back and attended there."""
    ops = _ops()
    S, H, n, step = 1100, 2, 6, 5 << 20
    big = torch.zeros(S * step, dtype=torch.uint8, device=DEV)
    view = lambda off: big[off:].as_strided((1, S, H, 128), (S * step, step, 128, 1))  # noqa: E731
    c = _held_cache(1, S, H, 51)
    d = {"k": view(0), "v": view(1 << 20)}
    for name in ("k", "v"):
        d[name].copy_(c[name])
        d[name + "_exp"] = big[(2 if name == "k" else 3) << 20:].view(torch.int8).as_strided((1, S, H), (S * step, step, 1))
        d[name + "_exp"].copy_(c[name + "_exp"])
    k, v = (_randn(s, 1, n, H, 128).to(torch.bfloat16) for s in (1, 2))
    want = _expected(c, k, v, (1, 2, 3), [5], [S - n])
    _append(d, k.to(DEV), k.to(DEV), v.to(DEV), (1, 2, 3), [5], [S - n])
    _same_cache(d, want)
    kr, _ = ops.kv_read_q8(d["k"], d["v"], d["k_exp"], d["v_exp"], [S - 2 * n], 2 * n)
    assert torch.equal(kr.double().cpu(), ref.values(want["k"][:, S - 2 * n:], want["k_exp"][:, S - 2 * n:]))
    q = _randn(3, 1, queries, H, 128).to(torch.bfloat16)
    _check_q8(want, q, [S], ops.attn_kvcache_q8(q.to(DEV), d["k"], d["v"], d["k_exp"], d["v_exp"], [S]))
    del big, d


# ------------------------------------------------------------------------------------------------ attention, spans
def _spans(kind, rows, n, S, seed=0):
    g = torch.Generator().manual_seed(seed)
    at = torch.arange(n)
    if kind == "all":
        return torch.zeros(rows, n, dtype=torch.int32), torch.full((rows, n), S, dtype=torch.int32)
    if kind == "lens":
        end = torch.randint(0, S + 1, (rows, 1), generator=g).expand(rows, n)
        return torch.zeros_like(end).int(), end.int()
    if kind == "causal":                                    # query i attends keys 0 .. i
        return torch.zeros(rows, n, dtype=torch.int32), (at + 1)[None].expand(rows, n).int()
    if kind == "blocks":                                    # blocks of 150 see themselves and what came before
        return torch.zeros(rows, n, dtype=torch.int32), ((at // 150 + 1) * 150).clamp_max(S)[None].expand(rows, n).int()
    if kind == "docs":                                      # clips of 70 packed into a row, every fifth one padding
        doc = at // 70
        begin, end = doc * 70, (doc * 70 + 70).clamp_max(S)
        end = torch.where(doc % 5 == 3, torch.zeros_like(end), end)
        return begin[None].expand(rows, n).int(), end[None].expand(rows, n).int()
    if kind == "window":
        return (at - 40)[None].expand(rows, n).int(), (at + 1)[None].expand(rows, n).int()
    a, b = (torch.randint(-5, S + 6, (rows, n), generator=g) for _ in range(2))   # free: clipped, some empty
    return torch.where(torch.rand(rows, n, generator=g) < 0.8, torch.minimum(a, b), a).int(), torch.maximum(a, b).int()


def _check_spans(q, k, v, begin, end, out, scale=None):
    want, weight = ref.span_attention(q.to(DEV), k.to(DEV), v.to(DEV), begin, end, scale)
    ref.check_attention(out, want, weight, k.shape[1])


@pytest.mark.parametrize("kind", ["all", "lens", "causal", "blocks", "docs", "window", "free"])
@pytest.mark.parametrize("rows,n,heads,S", [
    (1, 1, 1, 1), (1, 1, 2, 1000), (3, 5, 2, 129), (2, 128, 1, 128), (2, 300, 3, 300), (1, 1000, 2, 1000), (4, 600, 14, 200),
    (1, 2, 3, 20000),
])
def test_spans_attention(kind, rows, n, heads, S):
    ops = _ops()
    q, k, v = (_randn(s, rows, m, heads, 128).to(torch.bfloat16) for s, m in ((1, n), (2, S), (3, S)))
    begin, end = _spans(kind, rows, n, S, seed=n)
    out = ops.attn_spans(q.to(DEV), k.to(DEV), v.to(DEV), begin.to(DEV), end.to(DEV))
    _check_spans(q, k, v, begin, end, out)
    if kind in ("all", "lens", "causal"):                   # begin left out is 0
        assert torch.equal(out, ops.attn_spans(q.to(DEV), k.to(DEV), v.to(DEV), None, end.to(DEV)))
    ops.read_status(torch.device(DEV))


@pytest.mark.parametrize("kind", ["lens", "docs", "window"])
def test_spans_attention_with_anything_in_keys_that_nobody_attends(kind):
    """NaN, infinities and the type's lowest value in K and V of padding, between documents as well as behind the last."""
    ops = _ops()
    n = S = 777
    q, k, v = (_randn(s, 2, m, 2, 128).to(torch.bfloat16) for s, m in ((1, n), (2, S), (3, S)))
    begin, end = _spans(kind, 2, n, S, seed=5)
    if kind == "window":
        end[:, 200:330] = 0                                # nobody attends keys around 230 .. 289
    key = torch.arange(S)
    inside = ((key >= begin[..., None]) & (key < end[..., None])).any(1)
    assert bool((~inside).any())
    for t in (k, v):
        for b in range(2):
            t[b, ~inside[b], :, ::3] = float("nan")
            t[b, ~inside[b], :, 1::3] = float("inf")
            t[b, ~inside[b], :, 2::3] = torch.finfo(torch.bfloat16).min
    out = ops.attn_spans(q.to(DEV), k.to(DEV), v.to(DEV), begin.to(DEV), end.to(DEV))
    assert bool(torch.isfinite(out).all())
    _check_spans(q, k, v, begin, end, out)


def test_spans_attention_strides_broadcast_and_scale():
    ops = _ops()
    B, n, H, S = 3, 260, 2, 200
    q = _randn(1, B, n, 2 * H, 128).to(torch.bfloat16)[:, :, ::2]
    kv = _randn(2, 1, S, 2, H, 128).to(torch.bfloat16)
    k, v = (kv[:, :, i].expand(B, -1, -1, -1) for i in range(2))
    lens = torch.tensor([[200], [0], [77]], dtype=torch.int32)
    both = torch.zeros(B, n, 2, dtype=torch.int32)
    both[..., 0], both[..., 1] = 3, lens
    qd, kvd = q.to(DEV), kv.to(DEV)
    kd, vd = (kvd[:, :, i].expand(B, -1, -1, -1) for i in range(2))
    bd = both.to(DEV)
    out = ops.attn_spans(qd, kd, vd, bd[..., 0], bd[..., 1], softmax_scale=0.02)
    _check_spans(q, k, v, both[..., 0], both[..., 1], out, scale=0.02)
    wide = ops.attn_spans(qd, kd, vd, None, lens.to(DEV).expand(B, n))
    _check_spans(q, k, v, torch.zeros(B, n), lens.expand(B, n), wide)
    assert not bool(wide[1].any())


@pytest.mark.parametrize("n,S", [(200, 500), (300, 1700)])
def test_spans_attention_heads_outermost_and_offsets_past_32_bits(n, S):
    ops = _ops()
    H, step = 2, 2 << 20                                    # elements between tokens: 4 MB
    q, k, v = (_randn(s, 1, m, H, 128).to(torch.bfloat16) for s, m in ((1, n), (2, S), (3, S)))
    begin, end = _spans("free", 1, n, S, seed=3)
    outer = [t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) for t in (q, k, v)]
    _check_spans(q, k, v, begin, end, ops.attn_spans(*outer, begin.to(DEV), end.to(DEV)))
    big = torch.zeros(S * step, dtype=torch.bfloat16, device=DEV)
    kd, vd = (big[off:].as_strided((1, S, H, 128), (S * step, step, 128, 1)) for off in (0, 1 << 20))
    kd.copy_(k)
    vd.copy_(v)
    _check_spans(q, k, v, begin, end, ops.attn_spans(q.to(DEV), kd, vd, begin.to(DEV), end.to(DEV)))
    del big, kd, vd


@pytest.mark.parametrize("rows,n,heads,S", [(24, 2, 26, 994), (3, 300, 5, 900), (8, 130, 20, 1000), (2, 700, 5, 3000)])
def test_spans_attention_gives_the_same_bits_whatever_the_timing(rows, n, heads, S):
    """Fresh operands (nothing cached) and then the same again: tiles that a span covers next to tiles that it cuts, whose
    keys arrive late in the first call."""
    ops = _ops()
    g = torch.Generator(DEV).manual_seed(3)
    flush = torch.empty(1 << 26, device=DEV)
    for _ in range(40):
        q, k, v = (torch.randn(rows, m, heads, 128, generator=g, device=DEV).to(torch.bfloat16) for m in (n, S, S))
        a, b = (torch.randint(-5, S + 6, (rows, n), generator=g, device=DEV, dtype=torch.int32) for _ in range(2))
        a, b = torch.minimum(a, b), torch.maximum(a, b)
        flush.fill_(1.0)
        first, second, third = (ops.attn_spans(q, k, v, a, b) for _ in range(3))
        assert torch.equal(first, second) and torch.equal(second, third)


def test_span_attention_over_whole_rows_agrees_with_the_cache_kernel():
    ops = _ops()
    q, k, v = (_randn(s, 2, m, 3, 128).to(torch.bfloat16).to(DEV) for s, m in ((1, 500), (2, 900), (3, 900)))
    end = torch.tensor([[900], [517]], dtype=torch.int32, device=DEV).expand(2, 500)
    a, b = ops.attn_spans(q, k, v, None, end).float(), ops.attn_kvcache(q, k, v, [900, 517]).float()
    # the same arithmetic on the same tiles; parts may be cut differently
    assert (a - b).abs().max().item() <= 2.0 ** -7 * b.abs().max().item()


def test_empty_problems():
    ops = _ops()
    c = _cuda(_garbage_cache(2, 8, 2))
    z = torch.zeros(2, 0, 2, 128, dtype=torch.bfloat16, device=DEV)
    q = torch.ones(2, 3, 2, 128, dtype=torch.bfloat16, device=DEV)
    end = torch.full((2, 3), 5, dtype=torch.int32, device=DEV)
    assert ops.attn_kvcache_q8(z, c["k"], c["v"], c["k_exp"], c["v_exp"], [8, 8]).shape == z.shape
    assert not bool(ops.attn_spans(q, z, z, None, end).any())
    assert ops.attn_spans(z, q, q, None, end[:, :0]).shape == z.shape
    assert not bool(ops.attn_kvcache_q8(q, c["k"], c["v"], c["k_exp"], c["v_exp"], [0, 0]).any())
    assert ops.kv_read_q8(c["k"], c["v"], c["k_exp"], c["v_exp"], [0, 0], 0)[0].shape == z.shape


# ------------------------------------------------------------------------------------------------ together
def test_calls_on_two_streams_and_in_recorded_graphs_do_not_share_scratch():
    """Split launches (one query over a long cache) that may overlap: two streams, then two recorded graphs replayed on
    two streams with fresh inputs."""
    ops = _ops()
    S, H = 6000, 4
    sets = []
    for i in range(2):
        c = _held_cache(1, S, H, 40 + 10 * i)
        q = _randn(60 + i, 1, 1, H, 128).to(torch.bfloat16)
        k, v = (_randn(70 + i + j, 1, S, H, 128).to(torch.bfloat16) for j in (0, 5))
        sets.append((c, _cuda(c), q, q.to(DEV), k, v, k.to(DEV), v.to(DEV)))
    end = torch.full((1, 1), S, dtype=torch.int32, device=DEV)
    call = lambda s: (ops.attn_kvcache_q8(s[3], s[1]["k"], s[1]["v"], s[1]["k_exp"], s[1]["v_exp"], [S]),  # noqa: E731
                      ops.attn_spans(s[3], s[6], s[7], None, end))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sets:
        call(s)
    torch.cuda.synchronize()
    want = [call(s) for s in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(call(s))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    graphs, outs = [], []
    for st, s in zip(streams, sets):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call(s))
        graphs.append(g)
    sets[0][3].copy_(sets[1][2])                            # fresh inputs at the recorded addresses
    sets[1][3].copy_(sets[0][2])
    torch.cuda.synchronize()
    for _ in range(5):
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, other, o in zip(sets, sets[::-1], outs):
        _check_q8(s[0], other[2], [S], o[0])
        _check_spans(other[2], s[4], s[5], torch.zeros(1, 1), torch.full((1, 1), S), o[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_stream_of_steps_append_read_attend(dtype):
    """Several chunks into a wrapping 8-bit cache: bytes as the plain statement writes them, read back, attended."""
    ops = _ops()
    rows, heads, grid, cache = 2, 3, (1, 6, 11), 200
    n = 66
    plain = {n_: t for n_, t in _garbage_cache(rows, cache, heads).items()}
    plain["k_exp"].fill_(-128)
    plain["v_exp"].fill_(-128)
    dev = _cuda(plain)
    filled = 0
    for step in range(6):
        q, k, v = (_randn(100 + 3 * step + i, rows, n, heads, 128).to(dtype) for i in range(3))
        slot = (step % 3) * n
        filled = max(filled, slot + n)
        plain = _expected(plain, k, v, grid, [step, step + 7], [slot, slot])
        rq = _append(dev, q.to(DEV), k.to(DEV), v.to(DEV), grid, [step, step + 7], [slot, slot])
        _same_cache(dev, plain)
        kr, vr = ops.kv_read_q8(dev["k"], dev["v"], dev["k_exp"], dev["v_exp"], [slot, slot], n, dtype=dtype)
        assert torch.equal(vr.double().cpu(), ref.values(plain["v"], plain["v_exp"])[:, slot:slot + n])
        out = ops.attn_kvcache_q8(rq.to(torch.bfloat16), dev["k"], dev["v"], dev["k_exp"], dev["v_exp"], [filled, filled])
        _check_q8(plain, rq.to(torch.bfloat16).cpu(), [filled, filled], out)
    ops.read_status(torch.device(DEV))
