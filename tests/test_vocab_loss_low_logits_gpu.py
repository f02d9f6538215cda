"""GPU: linear_cross_entropy on rows whose logits all lie far below zero, in every form of the call."""
import pytest
import torch

from tests.test_vocab_loss_gpu import check_linear, make_linear, outputs

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from neuspeech1_amd import ops as o
    return o


FORMS = [("h", 0, 1.0, 0.0), ("hw", 0, 1.0, 0.0), ("h", 4, 1.0, 0.5), ("hw", 4, 1.0, 0.5), ("h", 4, 1.0, 1.0), ("h", 4, 2.0, 0.5), ("hw", 4, 1.5, 0.3), ("hw", 4, 4.0, 0.5), ("hw", 4, 3.0, 1.0)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,v", [(20, 300), (70, 257), (300, 600), (130, 2881)])
@pytest.mark.parametrize("grad,k,temp,alpha", FORMS)
@pytest.mark.parametrize("low", [-100.0, -600.0])
def test_rows_whose_logits_all_lie_low(ops, dev, dtype, rows, v, grad, k, temp, alpha, low):
    """a softmax does not change when a row's logits move together; the vocabulary ends inside the first 64, 128 or 192 columns of a 256-column tile, so that strips past it
    are formed and belong to no row"""
    h, w, labels, lists = make_linear(dev, rows, 64, v, dtype, seed=41, ignored=0.1, k=k)
    h[:, 0], w[:, 0] = 8.0, low / 8.0
    check_linear(ops, dev, h, w, labels, lists, temp, alpha, grad=grad, scale=8.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("grad,k", [("h", 0), ("hw", 0), ("h", 4)])
def test_low_rows_without_a_reference(ops, dev, dtype, grad, k):
    """products so large that the label's logit is no reference: what cancels leaves no digits to compare, but nothing may become infinite or NaN"""
    h, w, labels, lists = make_linear(dev, 300, 64, 300, dtype, seed=42, ignored=0.1, k=k)
    h[:, 0], w[:, 0] = 8.0, -40.0
    h[:, 1:3] = 2.0 ** 11
    w[:, 1], w[:, 2] = 2.0 ** 11, -2.0 ** 11
    o = outputs(dev, 300)
    got = {"dh": torch.full_like(h, 3.0), **({"dweight": torch.full_like(w, 3.0)} if "w" in grad else {})}
    kw = dict(top_vals=lists[0], top_idx=lists[1], temperature=1.0, alpha=0.5) if k else {}
    ops.linear_cross_entropy(h, w, labels, **o, **got, **kw)
    for x in (o["row_loss"], o["loss"], *got.values()):
        assert torch.isfinite(x).all()
