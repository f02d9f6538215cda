"""CPU: what linear_cross_entropy, distill_topk and topk_logits refuse (before anything is launched), the workspace rule, and the
64-bit statement itself against autograd."""
import ctypes as C

import pytest
import torch

from neuspeech1_amd import lib, ops
from tests import vocab_loss_ref as R

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def outs(rows):
    return dict(row_loss=torch.zeros(rows), loss=torch.zeros(1), nvalid=torch.zeros(1, dtype=torch.int32))


def linear_args(rows=6, d=16, v=50, dtype=F16):
    return dict(h=torch.zeros(rows, d, dtype=dtype), weight=torch.zeros(v, d, dtype=dtype), labels=torch.zeros(rows, dtype=torch.int64), **outs(rows))


def lists(rows=6, k=4):
    return dict(top_vals=torch.zeros(rows, k), top_idx=torch.zeros(rows, k, dtype=torch.int32))


H = torch.zeros(6, 16, dtype=F16)
BAD_LINEAR = [
    (dict(h=torch.zeros(6, 16)), "dtype"),
    (dict(h=torch.zeros(6, 2, 8, dtype=F16)), "2-D"),
    (dict(h=torch.zeros(6, 12, dtype=F16), weight=torch.zeros(50, 12, dtype=F16)), "multiple of 8"),
    (dict(h=torch.zeros(6, 0, dtype=F16), weight=torch.zeros(50, 0, dtype=F16)), "multiple of 8"),
    (dict(h=torch.zeros(16, 6, dtype=F16).t()), "contiguous"),
    (dict(h=torch.zeros(6 * 20, dtype=F16)[:120].view(6, 20)[:, :16]), "16 bytes"),
    (dict(h=torch.zeros(6, 24, dtype=F16)[:, 4:20]), "16 bytes"),
    (dict(h=torch.zeros(1, 16, dtype=F16).expand(6, 16)), "overlap"),
    (dict(weight=torch.zeros(50, 24, dtype=F16)), "weight"),
    (dict(weight=torch.zeros(50, 16, dtype=BF16)), "weight"),
    (dict(weight=torch.zeros(0, 16, dtype=F16)), "no rows"),
    (dict(labels=None), "labels"),
    (dict(labels=torch.zeros(6, dtype=torch.int32)), "labels"),
    (dict(labels=torch.zeros(5, dtype=torch.int64)), "labels"),
    (dict(labels=torch.zeros(12, dtype=torch.int64)[::2]), "labels"),
    (dict(row_loss=torch.zeros(6, dtype=F16)), "row_loss"),
    (dict(loss=torch.zeros(2)), "loss"),
    (dict(nvalid=torch.zeros(1, dtype=torch.int64)), "nvalid"),
    (dict(loss_scale=torch.zeros(1, dtype=F16)), "loss_scale"),
    (dict(dh=torch.zeros(6, 16, dtype=BF16)), "dh"),
    (dict(dh=torch.zeros(5, 16, dtype=F16)), "dh"),
    (dict(h=H, dh=H), "overlaps"),
    (dict(dweight=torch.zeros(50, 16, dtype=BF16)), "dweight"),
    (dict(dweight=torch.zeros(49, 16, dtype=F16)), "dweight"),
    (dict(accumulate=True), "accumulate"),
    (dict(dweight=torch.zeros(50, 16, dtype=F16), accumulate=True), "accumulate"),
    (dict(alpha=0.5), "soft targets"),
    (dict(top_vals=torch.zeros(6, 4), alpha=0.5), "together"),
    (dict(**lists(k=257), alpha=0.5), "256"),
    (dict(**lists(k=0), alpha=0.5), "256"),
    (dict(**lists(rows=5), alpha=0.5), "top_vals"),
    (dict(top_vals=torch.zeros(6, 4), top_idx=torch.zeros(6, 4, dtype=torch.int64), alpha=0.5), "top_idx"),
    (dict(top_vals=torch.zeros(6, 8)[:, :4], top_idx=torch.zeros(6, 4, dtype=torch.int32), alpha=0.5), "row strides"),
    (dict(**lists(), alpha=1.5), "alpha"),
    (dict(**lists(), alpha=-0.1), "alpha"),
    (dict(**lists(), alpha=float("nan")), "alpha"),
    (dict(**lists(), alpha=0.5, temperature=0.04), "temperature"),
    (dict(**lists(), alpha=0.5, temperature=float("inf")), "temperature"),
    ({}, "expected a GPU"),
]


@pytest.mark.parametrize("change,match", BAD_LINEAR, ids=[m + str(i) for i, (_, m) in enumerate(BAD_LINEAR)])
def test_linear_cross_entropy_refuses(change, match):
    kw = dict(linear_args(), **change)
    with pytest.raises(ValueError, match=match):
        ops.linear_cross_entropy(kw.pop("h"), kw.pop("weight"), kw.pop("labels"), **kw)


BAD_DISTILL = [
    (dict(logits=torch.zeros(6, 50, dtype=torch.float64)), "dtype"),
    (dict(logits=torch.zeros(50, 6).t()), "contiguous"),
    (dict(labels=None, alpha=0.5), "labels"),
    (dict(alpha=0.0), "alpha"),
    (dict(alpha=2.0), "alpha"),
    (dict(temperature=-1.0), "temperature"),
    (dict(top_vals=torch.zeros(6, 300), top_idx=torch.zeros(6, 300, dtype=torch.int32)), "256"),
    (dict(dlogits=torch.zeros(6, 50, dtype=F16)), "dlogits"),
    (dict(dlogits=torch.zeros(6, 49)), "dlogits"),
    ({}, "expected a GPU"),
]


@pytest.mark.parametrize("change,match", BAD_DISTILL, ids=[m + str(i) for i, (_, m) in enumerate(BAD_DISTILL)])
def test_distill_topk_refuses(change, match):
    kw = dict(dict(logits=torch.zeros(6, 50), labels=torch.zeros(6, dtype=torch.int64), **lists(), **outs(6), alpha=0.5, temperature=2.0), **change)
    with pytest.raises(ValueError, match=match):
        ops.distill_topk(kw.pop("logits"), kw.pop("labels"), kw.pop("top_vals"), kw.pop("top_idx"), **kw)


def test_distill_topk_refuses_a_shifted_view_of_its_logits():
    buf = torch.zeros(6, 60)
    with pytest.raises(ValueError, match="overlaps"):
        ops.distill_topk(buf[:, :50], torch.zeros(6, dtype=torch.int64), *lists().values(), dlogits=buf[:, 4:54], alpha=0.5, **outs(6))


@pytest.mark.parametrize("change,match", [
    (dict(k=0), "k 0"), (dict(k=51), "k 51"), (dict(k=257), "k 257"), (dict(vals=torch.zeros(6, 5)), "vals"), (dict(idx=torch.zeros(6, 4, dtype=torch.int64)), "idx"),
    (dict(lse=torch.zeros(5)), "lse"), (dict(logits=torch.zeros(6, 50, dtype=torch.int32)), "dtype"), (dict(logits=torch.zeros(6, 0)), "k 4"), ({}, "expected a GPU")])
def test_topk_logits_refuses(change, match):
    kw = dict(dict(logits=torch.zeros(6, 50), k=4, vals=torch.zeros(6, 4), idx=torch.zeros(6, 4, dtype=torch.int32), lse=torch.zeros(6)), **change)
    with pytest.raises(ValueError, match=match):
        ops.topk_logits(kw.pop("logits"), kw.pop("k"), **kw)


def test_the_c_entry_points_refuse_too():
    so = lib.load()
    assert so.ns_linear_cross_entropy(None, None) == -1 and so.ns_distill_topk(None, None) == -1 and so.ns_topk_logits(None, None) == -1
    assert so.ns_linear_cross_entropy(C.byref(lib.LinearCeDesc()), None) == -1 and b"ns_linear_cross_entropy" in so.ns_last_error()
    assert so.ns_distill_topk(C.byref(lib.DistillDesc()), None) == -1 and b"ns_distill_topk" in so.ns_last_error()
    d = lib.TopkDesc()
    d.rows = 1
    assert so.ns_topk_logits(C.byref(d), None) == -1 and b"ns_topk_logits" in so.ns_last_error()


def test_workspace_rule():
    """one piece of dz stays within 256 MiB (all of it within 1 GiB where the head learns) however many rows and tokens there are, dh's partial sums within 128; the loss alone needs none of it; the list costs what it holds"""
    def need(rows, d, v, grad, k=0, head=False):
        a = linear_args(rows, d, v)
        if grad:
            a.update(dh=torch.empty_like(a["h"]))
        if head:
            a.update(dweight=torch.empty_like(a["weight"]))
        if k:
            a.update(lists(rows, k), alpha=0.5, temperature=2.0)
        return ops.linear_ce_workspace_bytes(a.pop("h"), a.pop("weight"), a.pop("labels"), **a)
    full = 2048 * 51968 * 2
    assert full < need(2048, 64, 51865, True) - need(2048, 64, 51865, False) <= full + 136 * (1 << 20)
    assert need(9000, 64, 51865, True) - need(9000, 64, 51865, False) <= 400 * (1 << 20) < 9000 * 51865 * 2
    assert 9000 * 51865 * 2 < need(9000, 64, 51865, True, head=True) < 9216 * 51968 * 2 + 256 * (1 << 20)
    assert need(11000, 64, 51865, True, head=True) < 400 * (1 << 20)
    assert need(100, 64, 1000, False, 64) > need(100, 64, 1000, False)
    assert need(1, 8, 1, True) > 0 and need(0, 8, 1, True) > 0
    assert lib.load().ns_linear_ce_workspace_bytes(C.byref(lib.LinearCeDesc())) == 0


def test_a_recorded_launch_list_needs_the_callers_workspace(monkeypatch):
    monkeypatch.setattr(ops, "_one_gpu", lambda *a: 0)
    a = linear_args()
    with ops.recording(ops.LaunchList()):
        with pytest.raises(ValueError, match="workspace"):
            ops.linear_cross_entropy(a.pop("h"), a.pop("weight"), a.pop("labels"), **a)


@pytest.mark.parametrize("temp,alpha", [(1.0, 0.0), (2.0, 0.5), (3.0, 1.0)])
def test_the_reference_gradient_is_autograds(temp, alpha):
    """the formula's gradient (what the GPU tests compare with) against autograd of the formula's loss and against differences, in 64 bits"""
    g = torch.Generator().manual_seed(3)
    rows, d, v, k = 12, 8, 30, 5
    h = torch.randn(rows, d, generator=g).half()
    w = torch.randn(v, d, generator=g).half()
    labels = torch.randint(0, v, (rows,), generator=g)
    labels[3] = -100
    tv = torch.randn(rows, k, generator=g)
    ti = torch.randint(-1, v + 1, (rows, k), generator=g, dtype=torch.int32)
    ti[5] = -1
    ti[6, 1] = ti[6, 0] = 7
    r = R.linear(h, w, labels, 1.0, None, temp, alpha, tv, ti)

    def loss(hd, wd):
        z = hd @ wd.t()
        ok = (labels >= 0) & (labels < v)
        total = 0.0
        for i in range(rows):
            if not ok[i]:
                continue
            total = total + (1 - alpha) * (torch.logsumexp(z[i], 0) - z[i, labels[i]])
            there = (ti[i] >= 0) & (ti[i] < v)
            if alpha and there.any():
                lp = torch.log_softmax(tv[i][there].double() / temp, 0)
                lq = torch.log_softmax(z[i] / temp, 0)[ti[i][there].long()]
                total = total + alpha * temp ** 2 * (lp.exp() * (lp - lq)).sum()
        return total / int(ok.sum())
    hd, wd = h.double().requires_grad_(), w.double().requires_grad_()
    value = loss(hd, wd)
    value.backward()
    torch.testing.assert_close(value.detach(), r["loss"], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(hd.grad, r["dh"], rtol=1e-10, atol=1e-12)
    torch.testing.assert_close(wd.grad, r["dw"], rtol=1e-10, atol=1e-12)
    u = torch.randn(rows, d, generator=g, dtype=torch.float64)
    with torch.no_grad():
        slope = (loss(hd + 1e-5 * u, wd) - loss(hd - 1e-5 * u, wd)) / 2e-5
    assert abs(float(slope) - float((r["dh"] * u).sum())) < 1e-8
