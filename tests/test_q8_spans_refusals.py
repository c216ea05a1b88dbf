"""What the 8-bit cache and key-span entry points refuse; all of it is decided on the host, before any CUDA call."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def native():
    from streamdiffusionv2_b200 import _native, build
    build.build()
    return _native


def _view(N, ptr=0x1000, row=128 * 64, tok=128, head=128):
    return ctypes.byref(N.View(ptr, row, tok, head))


def test_append_refusals(native):
    N = native
    lib = N.lib()

    def call(rows=1, n=4, heads=1, hd=128, cache=8, grid=(1, 2, 2), frames=(0,), slots=(0,), dtype=0, ke=True, table=0x4000,
             kc=None, step=None, ge=None, ge_val=None):
        views = [_view(N)] * 4 + [kc or _view(N), _view(N)] + [_view(N) if ke else None, _view(N)]
        return lib.sdv2_rope_kv_append_q8(*views, rows, n, heads, hd, cache, table, 1024, *grid,
                                          N.i64_array(frames) if frames is not None else None,
                                          N.i64_array(slots) if slots is not None else None, step, ge, ge, ge_val, ge_val,
                                          dtype, None, None)
    assert call(ke=False) == -1                              # no exponents
    assert call(hd=64) == -2 and call(hd=120) == -2          # head_dim
    assert call(rows=65, frames=[0] * 65, slots=[0] * 65) == -2
    assert call(slots=[5]) == -1 and call(slots=[-1]) == -1  # the slot leaves the cache
    assert call(frames=[1024]) == -1 and call(frames=[-1]) == -1
    assert call(grid=(1, 2, 3)) == -1 and call(n=0, grid=(0, 2, 2)) == -1
    assert call(dtype=2) == -1 and call(table=None) == -1
    assert call(kc=_view(N, ptr=0x1008)) == -3               # cache rows are written 8 bytes at a time, read 16
    assert call(kc=_view(N, tok=136)) == -3
    assert call(kc=_view(N, row=0)) == -1                    # rows of a cache that is written cannot be one row
    assert call(frames=None) == -1 and call(slots=None) == -1
    assert call(step=0x2004, frames=None, slots=None) == -3
    assert call(ge=0x3000) == -1                             # index tensors without their values


def test_read_refusals(native):
    N = native
    lib = N.lib()

    def call(rows=1, tokens=2, hd=128, cache=8, begin=(0,), dtype=0, out=None, heads=1):
        return lib.sdv2_kv_read_q8(*[_view(N)] * 4, out or _view(N), _view(N), rows, tokens, heads, hd, cache,
                                   N.i64_array(begin) if begin is not None else None, dtype, None)
    assert call(tokens=0) == -1 and call(rows=0) == -1 and call(begin=None) == -1
    assert call(begin=[7]) == -1 and call(begin=[-1]) == -1 and call(tokens=9) == -1
    assert call(hd=64) == -2 and call(rows=65, begin=[0] * 65) == -2 and call(heads=8192) == -2
    assert call(dtype=3) == -1 and call(out=_view(N, ptr=0x1002)) == -3 and call(out=_view(N, tok=129)) == -3


def test_attention_refusals(native):
    N = native
    lib = N.lib()

    def q8(rows=1, n=4, heads=1, hd=128, cache=8, lens=(8,), scale=0.1, q=None, k=None):
        return lib.sdv2_attn_kvcache_q8(q or _view(N), k or _view(N), _view(N), _view(N), _view(N), _view(N), rows, n, heads, hd,
                                        cache, N.i32_array(lens) if lens is not None else None, scale, None, 0, None, None)

    def spans(rows=1, n=4, heads=1, hd=128, keys=8, begin=None, end=0x5000, strides=(0, 0), scale=0.1, k=None):
        return lib.sdv2_attn_spans(_view(N), k or _view(N), _view(N), _view(N), rows, n, heads, hd, keys, begin, *strides, end,
                                   *strides, scale, None, 0, None, None)
    for call in (q8, spans):
        assert call(rows=0) == -1 and call(n=0) == -1 and call(heads=0) == -1
        assert call(hd=64) == -2
        assert call(heads=65536) == -2 and call(n=2 ** 31 - 1) == -2
        assert call(scale=0.0) == -1 and call(scale=float("nan")) == -1 and call(scale=float("inf")) == -1
        assert call(scale=3e38) == -1                        # infinite in log2 units
        assert call(k=_view(N, ptr=0x1008)) == -3
    assert q8(lens=None) == -1 and q8(lens=[9]) == -1 and q8(lens=[-1]) == -1 and q8(cache=0) == -1
    assert q8(rows=65, lens=[1] * 65) == -2 and q8(heads=8192) == -2 and q8(q=_view(N, row=0)) == -1
    assert spans(end=None) == -1 and spans(end=0x5002) == -1 and spans(begin=0x5001) == -1
    assert spans(strides=(-1, 0)) == -1 and spans(strides=(0, -1)) == -1 and spans(keys=0) == -1
    assert spans(k=_view(N, row=0)) == -1                    # K broadcast over rows but V not


def test_wrappers_refuse_wrong_tensors(native):
    """Shapes, types and devices are compared before anything is launched (host tensors do)."""
    from streamdiffusionv2_b200 import ops
    q = torch.zeros(2, 4, 3, 128, dtype=torch.bfloat16)
    c = ops.q8_cache(2, 10, 3, "cpu")
    assert c["k"].dtype == torch.uint8 and c["k_exp"].dtype == torch.int8 and c["v_exp"].shape == (2, 10, 3)
    cache = lambda **kw: [kw.get(n, c[n]) for n in ("k", "v", "k_exp", "v_exp")]  # noqa: E731
    table = torch.zeros(1024, 64, 2, dtype=torch.float64)
    bad = [dict(k=c["k"].to(torch.int8)), dict(k_exp=c["k_exp"].to(torch.uint8)), dict(v=c["v"][:, :9]), dict(v_exp=c["v_exp"][:1]),
           dict(k=c["k"][:, :, :2]), dict(v=c["v"].to("meta"))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.attn_kvcache_q8(q, *cache(**kw), [10, 10])
        with pytest.raises(ValueError):
            ops.rope_kv_append_q8(q, q, q, *cache(**kw), table, (1, 2, 2), [0, 0], [0, 0])
        if "k" not in kw:
            with pytest.raises(ValueError):
                ops.kv_read_q8(*cache(**kw), [0, 0], 2)
    with pytest.raises(ValueError):
        ops.attn_kvcache_q8(q.float(), *cache(), [10, 10])
    with pytest.raises(ValueError):
        ops.attn_kvcache_q8(q, *cache(), [10])
    with pytest.raises(ValueError):
        ops.rope_kv_append_q8(q, q.float(), q, *cache(), table, (1, 2, 2), [0, 0], [0, 0])
    with pytest.raises(ValueError):
        ops.rope_kv_append_q8(q, q, q, *cache(), table[:, :32], (1, 2, 2), [0, 0], [0, 0])
    with pytest.raises(ValueError):
        ops.kv_read_q8(*cache(), [0], 2)
    end = torch.zeros(2, 4, dtype=torch.int32)
    for args in ((q.float(), q, q, None, end), (q, q[:, :, :2], q, None, end), (q, q, q[:, :3], None, end), (q, q, q, None, end.long()),
                 (q, q, q, end[:, :3], end), (q, q, q, None, end[:1])):
        with pytest.raises(ValueError):
            ops.attn_spans(*args)


def test_an_8_bit_cache_refuses_fp32_models_before_it_is_written(native):
    from streamdiffusionv2_b200 import causal_attention as CA, ops
    cache = dict(ops.q8_cache(1, 8, 2, "cpu"), global_end_index=torch.zeros(1, dtype=torch.int64),
                 local_end_index=torch.zeros(1, dtype=torch.int64))
    q = torch.zeros(1, 4, 2, 128)
    with pytest.raises(ValueError, match="bf16"):
        CA.cached_attention(None, q, q, q, torch.tensor([[1, 2, 2]]), None, cache, 0)
