"""CPU: what counts as an overlap of two matrices: the bytes they hold, not the span between their first and last.  (A call that passes these checks here ends at "expected a GPU".)"""
import pytest
import torch

from neuspeech1_amd import ops

F16 = torch.float16


def outs(rows):
    return dict(row_loss=torch.zeros(rows), loss=torch.zeros(1), nvalid=torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("first,second,match", [((0, 16), (16, 32), "expected a GPU"), ((16, 32), (0, 16), "expected a GPU"), ((0, 16), (24, 40), "expected a GPU"),
                                                ((0, 16), (8, 24), "overlaps"), ((24, 40), (16, 32), "overlaps"), ((0, 16), (0, 16), "overlaps")])
@pytest.mark.parametrize("shift", [0, 2])
def test_h_and_dh_in_one_buffer(first, second, match, shift):
    """columns of the same rows, or of rows further down, which the other matrix reaches as well"""
    buf = torch.zeros(8, 40, dtype=F16)
    h, dh = buf[:6, first[0]:first[1]], buf[shift:6 + shift, second[0]:second[1]]
    with pytest.raises(ValueError, match=match):
        ops.linear_cross_entropy(h, torch.zeros(50, 16, dtype=F16), torch.zeros(6, dtype=torch.int64), dh=dh, **outs(6))


def test_different_row_strides_are_told_apart_by_their_span_alone():
    buf = torch.zeros(400, dtype=F16)
    h, dh = buf[:240].view(6, 40)[:, :16], buf[160:].view(-1, 24)[:6, :16]
    with pytest.raises(ValueError, match="overlaps"):
        ops.linear_cross_entropy(h, torch.zeros(50, 16, dtype=F16), torch.zeros(6, dtype=torch.int64), dh=dh, **outs(6))


@pytest.mark.parametrize("cols,match", [((50, 100), "expected a GPU"), ((49, 99), "overlaps")])
def test_logits_and_their_gradient_side_by_side(cols, match):
    buf = torch.zeros(6, 120)
    with pytest.raises(ValueError, match=match):
        ops.distill_topk(buf[:, :50], torch.zeros(6, dtype=torch.int64), torch.zeros(6, 4), torch.zeros(6, 4, dtype=torch.int32), dlogits=buf[:, cols[0]:cols[1]], alpha=0.5, **outs(6))


def test_lists_beside_the_logits():
    buf = torch.zeros(6, 120)
    idx = torch.zeros(6, 120, dtype=torch.int32)
    for at, match in ((60, "expected a GPU"), (40, "overlaps")):
        with pytest.raises(ValueError, match=match):
            ops.topk_logits(buf[:, :50], 4, vals=buf[:, at:at + 4], idx=idx[:, :4])
