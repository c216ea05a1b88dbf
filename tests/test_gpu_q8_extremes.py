"""Attention over the 8-bit cache at the ends of what its exponents can say."""
import pytest
import torch

import q8_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _randn(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("queries", [1, 8, 20, 32, 40, 900])
@pytest.mark.parametrize("low,high", [(100, 108), (105, 122), (121, 122)])
def test_keys_as_large_as_the_format_holds_against_queries_that_small(queries, low, high):
    """K exponents up to 121 (magnitudes of 2^127) in one head, with queries small enough that the scores are ordinary
    numbers; keys of another head are ordinary, and its queries too."""
    from streamdiffusionv2_b200 import ops
    S = 600
    k, v = _randn(1, 1, S, 2, 128), _randn(2, 1, S, 2, 128)
    q = _randn(3, 1, queries, 2, 128)
    k[:, :, 0] *= torch.exp2(torch.randint(low, high, (1, S, 1), generator=torch.Generator().manual_seed(4)).float() + 6 - 3)
    # largest K and q multiply to about 2^3 a product, signs at random: scores of a few units
    q[:, :, 0] *= 2.0 ** -(high - 1 + 6 - 3)
    q = q.to(torch.bfloat16)
    (kb, ke), (vb, ve) = ref.quantise(k.double()), ref.quantise(v.double())
    assert int(ke.max()) >= high - 3 and int(ke.max()) <= 121
    out = ops.attn_kvcache_q8(q.to(DEV), *(t.to(DEV) for t in (kb, vb, ke, ve)), [S])
    end = torch.full((1, queries), S)
    want, weight = ref.span_attention(q.to(DEV), ref.values(kb, ke).to(DEV), ref.values(vb, ve).to(DEV), torch.zeros_like(end), end)
    ref.check_attention(out, want, weight, S, (low, high))
    ops.read_status(torch.device(DEV))
