"""Kernels that are set up while the one before them ends, launched back to back with nothing between them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)


def test_kernels_of_every_tensor_memory_size_follow_one_another():
    """Calls with 256 and 512 columns of tensor memory a block, with one and two blocks an SM, without any, and split into
    parts with a merge behind them, in changing orders without a pause: every one gives the bits that it gives alone."""
    from streamdiffusionv2_b200 import ops
    heads = 6
    c = ops.q8_cache(2, 2600, heads, DEV)
    for n in ("k", "v"):
        c[n].copy_(torch.randint(0, 256, c[n].shape, generator=torch.Generator().manual_seed(5), dtype=torch.uint8))
        c[n + "_exp"].copy_(torch.randint(-9, -5, c[n + "_exp"].shape, generator=torch.Generator().manual_seed(6)).to(torch.int8))
    cache = [c[n] for n in ("k", "v", "k_exp", "v_exp")]
    q = {n: _randn(n, 2, n, heads, 128) for n in (3, 200, 900)}
    k, v = _randn(1, 2, 2600, heads, 128), _randn(2, 2, 2600, heads, 128)
    end = {n: torch.full((2, 1), 2500, dtype=torch.int32, device=DEV).expand(2, n) for n in q}
    calls = [lambda: ops.attn_spans(q[900], k[:, :700], v[:, :700], None, end[900]),      # one query tile a block
             lambda: ops.attn_spans(q[900], k, v, None, end[900]),                        # two
             lambda: ops.attn_spans(q[200], k[:, :700], v[:, :700], None, end[200]),      # in parts
             lambda: ops.attn_spans(q[200], k, v, None, end[200]),
             lambda: ops.attn_kvcache_q8(q[3], *cache, [2600, 77]),
             lambda: ops.attn_kvcache_q8(q[200], *cache, [2600, 77]),
             lambda: ops.attn_kvcache_q8(q[900], *cache, [2600, 77]),                     # expanded first
             lambda: ops.kv_read_q8(*cache, [0, 5], 300)[1]]
    alone = []
    for f in calls:
        alone.append(f())
        torch.cuda.synchronize()
    order = torch.randint(0, len(calls), (400,), generator=torch.Generator().manual_seed(3)).tolist()
    got = [(i, calls[i]()) for i in order]
    for i, t in got:
        assert torch.equal(t, alone[i]), i
    ops.read_status(torch.device(DEV))
