"""GPU: what a teacher's list may hold that no softmax can use."""
import pytest
import torch

from tests.test_vocab_loss_gpu import make_linear, outputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [9, 70])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temp,alpha", [(1.0, 0.5), (2.0, 0.5), (2.0, 1.0)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", ["one entry", "all entries"])
def test_a_teachers_overflow_shows_in_the_loss(dev, rows, dtype, temp, alpha, bad, which):
    """a NaN or +inf among the values of a row that counts makes that row's loss (and the mean) NaN, in both losses; the same behind a token that is no entry, or in an ignored row,
    does nothing, and no other row is touched"""
    from neuspeech1_amd import ops
    h, w, labels, _ = make_linear(dev, rows, 64, 300, dtype, seed=51, ignored=0.0)
    labels = labels.clamp(0, 299)
    labels[4] = -100
    tv = torch.randn(rows, 6, device=dev)
    ti = torch.randint(0, 300, (rows, 6), device=dev, dtype=torch.int32)
    ti[3, 2] = -1
    z = (h.float() @ w.float().t()).to(dtype)

    def both(tv):
        out = []
        for f, a, kw in ((ops.linear_cross_entropy, (h, w, labels), dict(top_vals=tv, top_idx=ti, dh=torch.empty_like(h))),
                         (ops.distill_topk, (z, labels, tv, ti), dict(dlogits=torch.empty_like(z)))):
            o = outputs(dev, rows)
            f(*a, temperature=temp, alpha=alpha, **o, **kw)
            out.append((o["row_loss"], o["loss"], kw.get("dh", kw.get("dlogits"))))
        return out
    good = both(tv)
    worse = tv.clone()
    worse[4] = bad                        # an ignored row
    worse[3, 2] = bad                     # no entry
    for a, b in zip(good, both(worse)):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    if which == "one entry":
        worse[7, 1] = bad
    else:
        worse[7] = bad
    rest = torch.arange(rows, device=dev) != 7
    for a, b in zip(good, both(worse)):
        assert torch.isnan(b[0][7]) and torch.isnan(b[1]).all() and not torch.isfinite(b[2][7]).all()
        assert torch.equal(a[0][rest], b[0][rest]) and torch.equal(a[2][rest], b[2][rest])
