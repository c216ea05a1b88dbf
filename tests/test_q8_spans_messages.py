"""What the wrappers of the 8-bit cache and of key spans refuse by name, decided before anything is launched."""
import pytest
import torch

from streamdiffusionv2_b200 import build, ops


@pytest.fixture(scope="module", autouse=True)
def _built():
    build.build()


def test_spans_want_k_and_v_broadcast_over_rows_together():
    q = torch.zeros(2, 4, 3, 128, dtype=torch.bfloat16)
    end, one = torch.zeros(2, 4, dtype=torch.int32), q[:1].expand(2, -1, -1, -1)
    for k, v in ((one, q), (q, one)):
        with pytest.raises(ValueError, match="broadcast"):
            ops.attn_spans(q, k, v, None, end)


def test_no_gradient_is_dropped_silently():
    """None of these records a gradient: a tensor that wants one is refused while gradients are recorded, before a cache is
    written, and taken (here as far as: there is no CPU path) where they are not."""
    from streamdiffusionv2_b200 import causal_attention as ca
    q = torch.zeros(1, 4, 3, 128, dtype=torch.bfloat16)
    g = q.clone().requires_grad_()
    c = ops.q8_cache(1, 10, 3, "cpu")
    cache = [c[n] for n in ("k", "v", "k_exp", "v_exp")]
    table, end = torch.zeros(1024, 64, 2, dtype=torch.float64), torch.zeros(1, 4, dtype=torch.int32)
    kv = dict(c, global_end_index=torch.zeros(1, dtype=torch.int64), local_end_index=torch.zeros(1, dtype=torch.int64))
    weight = torch.ones(384, dtype=torch.bfloat16)
    calls = [lambda x, i=i: ops.rope_kv_append_q8(*[x if j == i else q for j in range(3)], *cache, table, (1, 2, 2), [0], [0]) for i in range(3)]
    calls += [lambda x: ops.rope_kv_append_q8(q, q, q, *cache, table, (1, 2, 2), [0], [0], q_out=x),
              lambda x: ops.attn_kvcache_q8(x, *cache, [4]), lambda x: ops.attn_kvcache_q8(q, *cache, [4], out=x)]
    calls += [lambda x, i=i: ops.attn_spans(*[x if j == i else q for j in range(3)], None, end) for i in range(3)]
    calls += [lambda x: ops.attn_spans(q, q, q, None, end, out=x), lambda x: ops.kv_read_q8(*cache, [0], 4, out=(q, x))]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError, match="gradient"):
            call(g)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            call(g)
    for i in range(3):
        qkv = [g if j == i else q for j in range(3)]
        with pytest.raises(RuntimeError, match="gradient"):
            ca.cached_attention(None, *qkv, torch.tensor([[1, 2, 2]]), None, kv, 0, norm=(weight, weight, 1e-6))
