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
