"""GPU: the vocabulary losses on rows that a trained model gives: almost certain of a token (vocab_loss_confident_ref derives the bounds)."""
import pytest
import torch

from tests import vocab_loss_confident_ref as C
from tests import vocab_loss_ref as R
from tests.test_vocab_loss_gpu import close, gen, outputs

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from neuspeech1_amd import ops as o
    return o


def make_confident(dev, rows, d, v, dtype, seed, common=0.3, low=0.0, rival=0.0):
    """hidden states along their label's row of the head, so that 1 - p runs from about a half down to 1e-7 over the rows; the head has a common component, so that the tail of
    a row's distribution does not average out.  rival: another token's row of the head joins in by this much, and 1 - p without it runs over that range"""
    g = gen(seed, dev)
    w = torch.randn(v, d, generator=g, device=dev) + common * torch.randn(1, d, generator=g, device=dev)
    w = (w * 2.0 * d ** -0.5).to(dtype)
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    h = torch.randn(rows, d, generator=g, device=dev) * 0.25
    if low:
        h[:, 0], w[:, 0] = 8.0, low / 8.0
    wd, hd = w.double(), h.double()
    along = wd[labels] + rival * wd[(labels + v // 2) % v]
    if low:
        along[:, 0] = 0.0
    want = torch.logspace(-0.3, -7.0, rows, dtype=torch.float64, device=dev)
    base, step = hd @ wd.t(), along @ wd.t()
    lo, hi = torch.zeros(rows, 1, dtype=torch.float64, device=dev), torch.full((rows, 1), 60.0, dtype=torch.float64, device=dev)
    for _ in range(40):
        mid = (lo + hi) / 2
        z = base + mid * step
        e = torch.exp(z - z.gather(1, labels.unsqueeze(1))).scatter(1, labels.unsqueeze(1), 0.0)
        if rival:
            e = e.scatter(1, ((labels + v // 2) % v).unsqueeze(1), 0.0)
        e = e.sum(1)
        more = (e / (1 + e) > want).unsqueeze(1)
        lo, hi = torch.where(more, mid, lo), torch.where(more, hi, mid)
    return (hd + hi * along).to(dtype), w, labels


def confident_lists(dev, rows, v, k, labels, seed, other):
    """a teacher that is as certain as the student: of the label, or (other) in every second row of another token"""
    g = gen(seed, dev)
    ti = (labels.unsqueeze(1) + 611 * torch.arange(k, device=dev)) % v
    tv = torch.cat([torch.linspace(2.0, 16.0, rows, device=dev).unsqueeze(1), torch.randn(rows, k - 1, generator=g, device=dev)], 1)
    if other:
        ti[::2, :2] = ti[::2, :2].flip(1)
    return tv.contiguous(), ti.int().contiguous()


def check_confident(ops, dev, h, w, labels, grad, lists=(None, None), temp=1.0, alpha=0.0, dw_dtype=None, scale=2.0 ** 19, parts=1, first=0, certain=True):
    rows = h.shape[0]
    o = outputs(dev, rows)
    got = {}
    if "h" in grad:
        got["dh"] = torch.full_like(h, 3.0)
    if "w" in grad:
        got["dweight"] = torch.full_like(w, 3.0, dtype=dw_dtype or w.dtype)
    kw = dict(top_vals=lists[0], top_idx=lists[1], temperature=temp, alpha=alpha) if lists[0] is not None else {}
    ops.linear_cross_entropy(h, w, labels, loss_scale=torch.tensor([scale], device=dev), **o, **got, **kw)
    dh, dh_tol, dw, dw_tol, left, floor = C.linear(h, w, labels, scale, temp, alpha, *lists, to_label=h.dtype == F16 and grad == "h" and lists[0] is None and rows > 64, dw_dtype=dw_dtype,
                                            parts=parts)
    if alpha == 0.0 and certain:
        assert float(left.min()) < 1e-6 and float(left.max()) > 0.05      # (the rows are what they are meant to be)
    if "h" in grad:
        close(got["dh"], dh, dh_tol, "dh")
        # as a whole: at most three roundings of a cell and one of the result (U each), and the logits: sqrt(d) u is what d roundings of random sign leave of a sum, twice over for two
        U = R.half_step(h.dtype)
        err = (got["dh"].double() - dh)[:, first:].norm(dim=1)
        sub = 2.0 ** -25 * h.shape[1] ** 0.5 if h.dtype == F16 else 0.0
        z_err = 2 * h.shape[1] ** 0.5 * R.U32 * (h.double().abs() @ w.double().abs().t()).amax(1)
        bad = ~(err <= (4 * U + z_err) * dh[:, first:].norm(dim=1) + sub + floor)
        assert not bad.any(), ("rows", bad.nonzero().flatten()[:8].tolist(), (err / dh.norm(dim=1))[bad][:8].tolist(), left[bad][:8].tolist())
    if "w" in grad:
        close(got["dweight"], dw, dw_tol, "dw")


@pytest.mark.parametrize("dtype,grad", [(F16, "h"), (F16, "hw"), (BF16, "h"), (BF16, "hw")])
@pytest.mark.parametrize("rows,d,v", [(64, 128, 5000), (40, 512, 5000), (200, 512, 5000), (96, 512, 51865), (300, 128, 1500)])
@pytest.mark.parametrize("low", [0.0, -100.0])
def test_confident_labels(ops, dev, dtype, rows, d, v, grad, low):
    """1 - p from a half to 1e-7: the gradient has its own digits, of the label's cell and of the tail, which adds up along the head's common component"""
    h, w, labels = make_confident(dev, rows, d, v, dtype, rows + d, low=low)
    check_confident(ops, dev, h, w, labels, grad, scale=2.0 ** 20, dw_dtype=F32 if grad == "hw" else None,
                    first=1 if low else 0)      # (column 0 of the head is one large number: what a row's cells add up to, which is nothing)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [8, 12, 30])
def test_few_confident_labels(ops, dev, dtype, rows):
    h, w, labels = make_confident(dev, rows, 256, 3000, dtype, rows)
    check_confident(ops, dev, h, w, labels, "hw", scale=2.0 ** 18, dw_dtype=F32, parts=2)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,d,v", [(200, 256, 3000), (64, 128, 3000), (90, 128, 51865)])
@pytest.mark.parametrize("temp,alpha", [(1.0, 0.5), (1.0, 1.0), (2.0, 0.5), (1.5, 0.3), (4.0, 0.5), (3.0, 1.0)])
@pytest.mark.parametrize("other", [False, True])
def test_confident_rows_with_a_confident_teacher(ops, dev, dtype, rows, d, v, temp, alpha, other):
    """soft targets that are as certain as the student: 1 - q against 1 - t, and p - 1 beside them"""
    h, w, labels = make_confident(dev, rows, d, v, dtype, rows + 1)
    lists = confident_lists(dev, rows, v, 5, labels, rows, other)
    for grad in ("h", "hw"):
        check_confident(ops, dev, h, w, labels, grad, lists, temp, alpha, dw_dtype=F32 if grad == "hw" else None)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_confident_beyond_all_rows_of_dz(ops, dev, dtype):
    """dz formed again, piece by piece: more than 1 GiB of it and the head learns"""
    h, w, labels = make_confident(dev, 300, 64, 9000, dtype, 5)
    rows = 2049
    h, labels = h.repeat(8, 1)[:rows].contiguous(), labels.repeat(8)[:rows].contiguous()
    pad = torch.zeros(262400 - 9000, 64, device=dev, dtype=dtype)
    pad[:, 0] = 1.0
    h[:, 0], w[:, 0] = 0.0, 0.0
    w = torch.cat([w, pad])
    h[:, 0] = -60.0                            # the other tokens lie 60 below zero: no part of any row
    o = outputs(dev, rows)
    dh, dw = torch.full_like(h, 3.0), torch.full((262400, 64), 3.0, device=dev)
    ops.linear_cross_entropy(h, w, labels, dh=dh, dweight=dw, loss_scale=torch.tensor([2.0 ** 20], device=dev), **o)
    want, tol, dwant, dtol, left, _ = C.linear(h, w[:9000].contiguous(), labels, 2.0 ** 20, dw_dtype=F32)
    assert float(left.min()) < 1e-6
    keep = slice(1, 64)                        # (column 0 is the pad's own)
    close(dh[:, keep], want[:, keep], tol[:, keep], "dh")
    close(dw[:9000, keep], dwant[:, keep], dtol[:, keep], "dw")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,d,v,rival", [(200, 256, 5000, 0.98), (96, 512, 51865, 0.9), (130, 512, 51865, 0.8), (40, 128, 3000, 0.95)])
def test_two_candidates_and_a_tail_far_below(ops, dev, dtype, rows, d, v, rival):
    """a rival that holds 2^-1 to 2^-20 of the label, all others far below both"""
    h, w, labels = make_confident(dev, rows, d, v, dtype, rows + d, rival=rival)
    check_confident(ops, dev, h, w, labels, "h", scale=2.0 ** 18, certain=False)


@pytest.mark.parametrize("rows,d,v,sharp", [(65, 136, 511, 1.0), (257, 264, 1001, 1.0), (300, 512, 2600, 2.0), (700, 776, 513, 0.0), (130, 64, 60001, 3.0), (2049, 64, 60001, 1.5)])
def test_fp16_cells_kept_relative_to_labels_of_every_kind(ops, dev, rows, d, v, sharp):
    """labels from the likeliest token to one among thousands, by the bounds that are relative to what a strip and a row hold"""
    g = gen(rows + v, dev)
    w = (torch.randn(v, d, generator=g, device=dev) * 2.0 * d ** -0.5).to(F16)
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    h = (torch.randn(rows, d, generator=g, device=dev) + sharp * torch.rand(rows, 1, generator=g, device=dev) * w[labels].float()).to(F16)
    check_confident(ops, dev, h, w, labels, "h", scale=2.0 ** 14, certain=False)


# ------------------------------------------------------------------------------------------------ over logits
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,v,first", [(40, 9, 0), (40, 1001, 3), (64, 5000, 0), (33, 51865, 1), (20, 70001, 0)])
@pytest.mark.parametrize("temp,alpha", [(1.0, 0.5), (2.0, 0.5), (4.0, 0.5), (1.5, 0.3), (2.0, 1.0)])
@pytest.mark.parametrize("who", ["label", "teacher"])
def test_distill_topk_on_almost_certain_rows(ops, dev, dtype, rows, v, first, temp, alpha, who):
    """student and teacher both certain of one token, the label or another: cells as exact as what the other tokens hold"""
    g = gen(rows + v, dev)
    buf = torch.randn(rows, v + first, generator=g, device=dev) * 2
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    labels[0], labels[1] = 0, v - 1
    sure = labels if who == "label" else (labels + v // 2) % v
    buf[:, first:].scatter_(1, sure.unsqueeze(1), torch.linspace(8.0, 26.0, rows, device=dev).unsqueeze(1) + (4.0 if v > 10000 else 0.0))
    buf = buf.to(dtype)
    z = buf[:, first:]
    ti = ((sure.unsqueeze(1) + torch.arange(4, device=dev)) % v).int().contiguous()
    tv = torch.cat([torch.linspace(20.0, 4.0, rows, device=dev).unsqueeze(1), torch.randn(rows, 3, generator=g, device=dev)], 1).contiguous()
    dz = torch.full_like(buf, 5.0)[:, first:]
    o = outputs(dev, rows)
    scale = 2.0 ** 14
    ops.distill_topk(z, labels, tv, ti, temperature=temp, alpha=alpha, dlogits=dz, loss_scale=torch.tensor([scale], device=dev), **o)
    cell, err, _, _ = C.cells(z.double(), torch.zeros(rows, dtype=torch.float64, device=dev), labels, temp, alpha, tv, ti)
    gs = scale / rows
    U = R.half_step(dtype)
    want = cell * gs
    small = {F16: 2.0 ** -25, BF16: 2.0 ** -126, F32: 2.0 ** -126}[dtype]
    close(dz, want, (err * gs + 4 * R.U32 * want.abs()) * (1 + U) + U * want.abs() + small, "dlogits")


# ------------------------------------------------------------------------------------------------ 33 to 64 labels
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,d,v", [(33, 256, 3000), (48, 512, 5001), (64, 264, 700), (50, 72, 51865)])
@pytest.mark.parametrize("grad,k,temp,alpha", [("hw", 0, 1.0, 0.0), ("h", 0, 1.0, 0.0), ("w", 0, 1.0, 0.0), ("hw", 5, 2.0, 0.3), ("h", 5, 1.0, 1.0), ("hw", 64, 1.0, 0.5)])
@pytest.mark.parametrize("shared", [False, True])
def test_33_to_64_labels_keep_their_digits(ops, dev, dtype, rows, d, v, grad, k, temp, alpha, shared):
    """dh and dW as a whole: no more than 1.15 times as far off as their own rounding.  Cells are 16-bit numbers, but a row's largest one in 256 tokens counts in fp32; what stays is
    the rounding of the others, whose squares add to less than a third of the result's own (1.15^2 - 1).  shared: several rows have the same label"""
    g = gen(rows + d, dev)
    w = (torch.randn(v, d, generator=g, device=dev) * 2.0 * d ** -0.5).to(dtype)
    labels = torch.randint(0, 3 if shared else v, (rows,), generator=g, device=dev) * (v // 3 if shared else 1)
    h = (torch.randn(rows, d, generator=g, device=dev) + w[labels].float()).to(dtype)
    lists = (None, None)
    if k:
        lists = ((6.0 - 2.5 * torch.log1p(torch.arange(k, device=dev).float()) + 0.3 * torch.randn(rows, k, generator=g, device=dev)).contiguous(),
                 ((labels.unsqueeze(1) + 611 * torch.arange(k, device=dev)) % v).int().contiguous())
    got = {n: torch.full_like(x, 3.0) for n, x in (("dh", h), ("dweight", w)) if n[1] in grad}
    more = dict(top_vals=lists[0], top_idx=lists[1], temperature=temp, alpha=alpha) if k else {}
    ops.linear_cross_entropy(h, w, labels, loss_scale=torch.tensor([2048.0], device=dev), **outputs(dev, rows), **got, **more)
    ref = R.linear(h, w, labels, 2048.0, None, temp, alpha, *lists)
    for n, x in got.items():
        want = ref["dh" if n == "dh" else "dw"]
        close(x, want, ref["dh_tol" if n == "dh" else "dw_tol"], n)
        own = (want.to(dtype).double() - want).norm()
        assert (x.double() - want).norm() <= 1.15 * own, (n, float((x.double() - want).norm() / own))
