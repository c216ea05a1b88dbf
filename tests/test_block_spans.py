"""Spans of clips in one pass against masks written out frame by frame."""
import pytest
import torch

from streamdiffusionv2_b200 import causal_attention as ca


def _attended(spans, tokens):
    """[rows, queries, keys] truth values of spans."""
    key = torch.arange(tokens)
    begin = torch.zeros_like(spans.end) if spans.begin is None else spans.begin
    return (key >= begin[..., None]) & (key < spans.end[..., None])


@pytest.mark.parametrize("frames,tokens,per,window", [
    (6, 1, 3, -1), (6, 4, 2, -1), (7, 3, 3, -1), (1, 5, 1, -1), (2, 5, 3, -1), (6, 4, 2, 2), (6, 4, 2, 3), (7, 3, 3, 3), (7, 3, 3, 4),
    (6, 1, 1, 1), (4, 2, 2, 100),
])
def test_spans_are_the_blocks_and_the_window(frames, tokens, per, window):
    """A token of frame f attends frames 0 .. e - 1 where e is its block's end (the clip's for a last block that is cut
    short), with a window only the last of these."""
    spans = ca.block_causal_spans(frames, tokens, per, "cpu", rows=2, window_frames=window)
    want = torch.zeros(frames * tokens, frames * tokens, dtype=torch.bool)
    for f in range(frames):
        end = min((f // per + 1) * per, frames)
        for g in range(frames):
            if g < end and (window < 0 or g >= end - window):
                want[f * tokens:(f + 1) * tokens, g * tokens:(g + 1) * tokens] = True
    assert spans.end.dtype == torch.int32 and spans.end.shape == (2, frames * tokens)
    assert torch.equal(_attended(spans, frames * tokens), want.expand(2, -1, -1))
    assert bool(want.diagonal().all())                     # a token attends itself


@pytest.mark.parametrize("per,window", [(3, 1), (3, 2), (2, 1), (0, -1), (-1, -1)])
def test_spans_refuse_windows_shorter_than_a_block_and_empty_blocks(per, window):
    """Early frames of a block would not attend themselves."""
    with pytest.raises(ValueError):
        ca.block_causal_spans(6, 2, per, "cpu", window_frames=window)
