"""GPU: linear_cross_entropy, distill_topk and topk_logits against their definitions in 64 bits (tests/vocab_loss_ref.py derives the tolerances)."""
import math

import pytest
import torch

from tests import vocab_loss_ref as R

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from neuspeech1_amd import ops as o
    return o


def gen(seed, dev):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def make_linear(dev, rows, d, v, dtype, seed=0, ignored=0.3, k=0, sharp=1.0):
    g = gen(seed + 1000 * rows + d, dev)
    w = (torch.randn(v, d, generator=g, device=dev) * 2.0 * d ** -0.5).to(dtype)
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    h = (torch.randn(rows, d, generator=g, device=dev) + sharp * w[labels].float()).to(dtype)
    off = torch.rand(rows, generator=g, device=dev) < ignored
    labels = torch.where(off, -100, labels)
    if rows > 4:
        labels[1], labels[2] = v, -1           # out of range: ignored as well
    return h, w, labels, (make_lists(dev, g, rows, v, k, labels) if k else (None, None))


def make_lists(dev, g, rows, v, k, labels):
    tv = torch.randn(rows, k, generator=g, device=dev) * 3
    ti = torch.randint(0, v, (rows, k), generator=g, device=dev, dtype=torch.int32)        # (repeats happen and add up)
    if k > 1:
        ti[:, 1] = torch.where((labels >= 0) & (labels < v), labels, 0).int()
        ti[::3, k - 1] = ti[::3, 0]            # the same token twice
        ti[::4, k // 2] = -1                   # an absent entry
    if rows > 6:
        ti[5] = -1                             # no list at all
        tv[6] = float("-inf")
        tv[3, 0] = float("-inf")
        ti[4, :] = v + 3                       # tokens outside the vocabulary
    return tv, ti


def outputs(dev, rows):
    return dict(row_loss=torch.full((rows,), 7.0, device=dev), loss=torch.full((1,), 7.0, device=dev), nvalid=torch.full((1,), 7, device=dev, dtype=torch.int32))


def close(got, want, tol, what):
    got = got.double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.numel(), float((got - want).abs()[bad].max()), float(tol[bad].min()), bad.nonzero()[:4].tolist())


def check_linear(ops, dev, h, w, labels, lists=(None, None), temp=1.0, alpha=0.0, scale=None, grad="hw", dw_dtype=None, parts=1, **kw):
    rows, d = h.shape
    o = outputs(dev, rows)
    dh = torch.full_like(h, 3.0) if "h" in grad else None
    dw = torch.full_like(w, 3.0, dtype=dw_dtype or w.dtype) if "w" in grad else None
    sc = None if scale is None else torch.tensor([scale], device=dev)
    more = dict(top_vals=lists[0], top_idx=lists[1], temperature=temp, alpha=alpha) if lists[0] is not None else {}
    ops.linear_cross_entropy(h, w, labels, dh=dh, dweight=dw, loss_scale=sc, **o, **more, **kw)
    torch.cuda.synchronize()
    ref = R.linear(h, w, labels, 1.0 if scale is None else scale, dw_dtype, temp, alpha, *lists, parts=parts, **(dict(floor=2.0 ** -29) if grad == "h" and lists[0] is None and rows > 64 else {}))
    assert int(o["nvalid"]) == ref["nvalid"]
    close(o["row_loss"], ref["row_loss"], ref["row_tol"], "row_loss")
    close(o["loss"], ref["loss"].reshape(1), ref["loss_tol"].reshape(1), "loss")
    if dh is not None:
        close(dh, ref["dh"], ref["dh_tol"], "dh")
    if dw is not None:
        close(dw, ref["dw"], ref["dw_tol"], "dw")
    return o, dh, dw


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,d,v", [(1, 8, 1), (1, 64, 300), (3, 72, 7), (5, 8, 257), (64, 64, 256), (16, 192, 300), (17, 136, 600), (32, 1288, 300),
                                      (33, 64, 5000), (64, 328, 2049), (65, 136, 511), (255, 256, 1000), (257, 264, 1001),
                                      (300, 512, 2600), (700, 776, 513)])
def test_linear_cross_entropy(ops, dev, dtype, rows, d, v):
    h, w, labels, _ = make_linear(dev, rows, d, v, dtype)
    check_linear(ops, dev, h, w, labels)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,d,v,k", [(1, 64, 300, 5), (9, 72, 50, 1), (30, 200, 900, 17), (130, 128, 1000, 64), (300, 256, 777, 256), (40, 64, 40, 40)])
@pytest.mark.parametrize("temp,alpha", [(1.0, 0.5), (2.0, 0.5), (3.5, 1.0), (1.0, 1.0), (0.5, 0.25), (2.0, 0.0)])
def test_linear_cross_entropy_with_a_teacher(ops, dev, dtype, rows, d, v, k, temp, alpha):
    h, w, labels, lists = make_linear(dev, rows, d, v, dtype, seed=1, k=k)
    check_linear(ops, dev, h, w, labels, lists, temp, alpha)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,live,d,v", [(1, 1, 64, 300), (2, 2, 512, 5000), (8, 8, 136, 257), (16, 5, 64, 1000), (32, 16, 72, 300), (64, 1, 64, 513), (64, 32, 200, 700)])
@pytest.mark.parametrize("k,temp,alpha", [(0, 1.0, 0.0), (7, 2.0, 0.5), (3, 1.0, 0.5)])
def test_few_labels_keep_their_digits(ops, dev, dtype, rows, live, d, v, k, temp, alpha):
    """the gradient of a few tokens is as exact as its own rounding: the one rounding of a label's cell would be a factor on all of it"""
    h, w, labels, lists = make_linear(dev, rows, d, v, dtype, seed=11, ignored=0.0, k=k)
    labels = torch.arange(rows, device=dev) * 7 % v
    h = (h.float() * 0.5 + w[labels].float()).to(dtype)
    labels[torch.randperm(rows, generator=gen(rows, dev), device=dev)[live:]] = -100
    check_linear(ops, dev, h, w, labels, lists, temp, alpha, parts=2, dw_dtype=F32 if rows == 16 else None)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("grad,dw_dtype", [("", None), ("h", None), ("w", None), ("w", F32), ("hw", F32)])
@pytest.mark.parametrize("rows", [12, 50, 90])
def test_linear_cross_entropy_gradients_on_request(ops, dev, dtype, grad, dw_dtype, rows):
    h, w, labels, _ = make_linear(dev, rows, 192, 700, dtype, seed=2)
    check_linear(ops, dev, h, w, labels, grad=grad, dw_dtype=dw_dtype, scale=32.0)


@pytest.mark.parametrize("rows", [20, 90])
def test_linear_cross_entropy_adds_to_a_float32_weight_gradient(ops, dev, rows):
    h, w, labels, _ = make_linear(dev, rows, 192, 700, BF16, seed=3)
    o = outputs(dev, rows)
    base = torch.randn(700, 192, device=dev)
    dw = base.clone()
    ops.linear_cross_entropy(h, w, labels, dweight=dw, accumulate=True, **o)
    ref = R.linear(h, w, labels, dw_dtype=F32)
    close(dw, ref["dw"] + base.double(), ref["dw_tol"] + 2 * R.U32 * (ref["dw"].abs() + base.double().abs()), "dw")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("grad,k,temp,alpha,ignored", [("hw", 3, 2.0, 0.5, 0.0), ("hw", 0, 1.0, 0.0, 0.1), ("hw", 3, 1.0, 0.5, 0.6), ("h", 0, 1.0, 0.0, 0.0), ("h", 3, 1.0, 0.5, 0.1),
                                                       ("h", 0, 1.0, 0.0, 0.5), ("h", 4, 3.0, 1.0, 0.0), ("", 0, 1.0, 0.0, 0.0),
                                                       ("hw", 3, 4.0, 0.5, 0.1), ("h", 3, 0.5, 0.5, 0.0)])
def test_linear_cross_entropy_beyond_one_workspace(ops, dev, dtype, grad, k, temp, alpha, ignored):
    """more rows x tokens than 256 MiB of dz: all of it where the head learns, pieces of the vocabulary where two softmaxes are mixed, chunks of rows (the last one full,
    partly filled or without a row) elsewhere"""
    h, w, labels, lists = make_linear(dev, 2049, 64, 60001, dtype, seed=4, ignored=ignored, k=k)
    check_linear(ops, dev, h, w, labels, lists, temp, alpha, grad=grad)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("k", [0, 3])
def test_linear_cross_entropy_beyond_all_rows_of_dz(ops, dev, dtype, k):
    """more than 1 GiB of dz and the head learns: pieces of the vocabulary"""
    h, w, labels, lists = make_linear(dev, 2049, 64, 240001, dtype, seed=12, ignored=0.1, k=k)
    check_linear(ops, dev, h, w, labels, lists, 1.0, 0.5 if k else 0.0)


@pytest.mark.parametrize("rows", [14, 60, 300])
def test_rows_without_a_label_are_not_read(ops, dev, rows):
    """infinities and NaN in masked rows reach neither loss nor gradients; their gradient is zero"""
    h, w, labels, lists = make_linear(dev, rows, 128, 600, BF16, seed=5, k=9)
    off = ~((labels >= 0) & (labels < 600))
    h[off] = float("nan")
    h[off.nonzero()[::2, 0]] = float("inf")
    lists[0][off] = float("nan")
    o, dh, dw = check_linear(ops, dev, h, w, labels, lists, 2.0, 0.5)
    assert (dh[off] == 0).all() and (o["row_loss"][off] == 0).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("rows", [9, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("k,alpha,temp", [(0, 0.0, 1.0), (4, 0.5, 1.0), (4, 0.5, 2.0), (4, 0.5, 4.0)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_an_overflow_in_a_labelled_row_shows(ops, dev, rows, dtype, k, alpha, temp, bad):
    """a NaN or infinity in a row that counts: loss, its row of dh and dW are not finite (what a loss scaler looks for), the other rows' dh keep their values"""
    h, w, labels, lists = make_linear(dev, rows, 72, 700, dtype, seed=19, ignored=0.0, k=k)
    kw = dict(top_vals=lists[0], top_idx=lists[1], temperature=temp, alpha=alpha) if k else {}
    good = dict(outputs(dev, rows), dh=torch.empty_like(h), dweight=torch.empty_like(w))
    ops.linear_cross_entropy(h, w, labels, **good, **kw)
    h[7, 5] = bad
    for grad in (("dh",), ("dh", "dweight")):
        got = dict(outputs(dev, rows), **{n: torch.empty_like(good[n]) for n in grad})
        ops.linear_cross_entropy(h, w, labels, **got, **kw)
        assert not torch.isfinite(got["loss"]).any() and not torch.isfinite(got["row_loss"][7]) and not torch.isfinite(got["dh"][7]).all()
        if "dweight" in grad:
            assert not torch.isfinite(got["dweight"]).all()
        rest = torch.arange(rows, device=dev) != 7
        near = (got["dh"][rest].double() - good["dh"][rest].double()).abs() <= 8 * R.half_step(dtype) * good["dh"][rest].double().abs().amax(1, keepdim=True)
        assert near.all()


@pytest.mark.parametrize("rows", [0, 1, 70])
def test_no_row_has_a_label(ops, dev, rows):
    h = torch.full((rows, 64), float("nan"), device=dev, dtype=F16)
    w = torch.randn(300, 64, device=dev).half()
    labels = torch.full((rows,), -100, device=dev, dtype=torch.int64)
    o = outputs(dev, rows)
    dh, dw = torch.full_like(h, 3.0), torch.full_like(w, 3.0)
    ops.linear_cross_entropy(h, w, labels, dh=dh, dweight=dw, **o)
    assert int(o["nvalid"]) == 0 and float(o["loss"]) == 0 and (o["row_loss"] == 0).all() and (dh == 0).all() and (dw == 0).all()


@pytest.mark.parametrize("rows", [13, 130])
def test_strided_operands_and_what_lies_beside_them(ops, dev, rows):
    g = gen(6, dev)
    d, v = 72, 301
    hb = torch.full((rows, 136), float("nan"), device=dev, dtype=F16)
    wb = torch.full((v + 3, 200), float("inf"), device=dev, dtype=F16)
    h, w = hb[:, 64:136], wb[2:v + 2, 8:80]
    h.copy_(torch.randn(rows, d, generator=g, device=dev))
    w.copy_(torch.randn(v, d, generator=g, device=dev) * 0.2)
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    o = outputs(dev, rows)
    dhb = torch.full((rows + 2, 96), 5.0, device=dev, dtype=F16)
    dwb = torch.full((v + 2, 80), 5.0, device=dev, dtype=F32)
    dh, dw = dhb[1:rows + 1, 16:88], dwb[1:v + 1, 8:80]
    ops.linear_cross_entropy(h, w, labels, dh=dh, dweight=dw, **o)
    ref = R.linear(h, w, labels, dw_dtype=F32)
    close(dh, ref["dh"], ref["dh_tol"], "dh")
    close(dw, ref["dw"], ref["dw_tol"], "dw")
    close(o["row_loss"], ref["row_loss"], ref["row_tol"], "row_loss")
    for buf, view in ((dhb, dh), (dwb, dw)):
        view.fill_(5.0)
        assert (buf == 5.0).all()


def test_large_logits(ops, dev):
    """logits of hundreds: the softmax is one-hot, every exponential stays finite"""
    h, w, labels, _ = make_linear(dev, 70, 64, 500, BF16, seed=7, sharp=0.0)
    check_linear(ops, dev, h * 64, w * 4, labels)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("dw_dtype", [None, F32])
@pytest.mark.parametrize("rows,d,v,tokens", [(9000, 72, 300, 1), (4100, 264, 700, 3), (700, 200, 513, 2)])
def test_many_rows_share_a_label(ops, dev, dtype, dw_dtype, rows, d, v, tokens):
    h, w, labels, _ = make_linear(dev, rows, d, v, dtype, seed=16, ignored=0.05)
    labels = torch.where((labels >= 0) & (labels < v), labels % tokens * (v // tokens) + v // tokens - 1, labels)
    check_linear(ops, dev, h, w, labels, scale=16.0, dw_dtype=dw_dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", [24, 93, 600])
@pytest.mark.parametrize("grad,k,temp,alpha", [("hw", 0, 1.0, 0.0), ("h", 0, 1.0, 0.0), ("hw", 5, 2.0, 0.3), ("h", 5, 1.0, 1.0), ("hw", 7, 1.0, 0.5), ("hw", 3, 4.0, 0.5)])
def test_the_largest_cells_keep_their_digits(ops, dev, dtype, rows, grad, k, temp, alpha):
    """a row's gradient, and a token's row of dW, is mostly one or two cells times a vector: as a whole no more than 1.3 times as far off as its own rounding (one
    rounding of every cell by itself would make that the square root of 2, and more where few rows average it out)"""
    h, w, labels, _ = make_linear(dev, rows, 256, 3000, dtype, seed=17, ignored=0.0)
    labels %= 3000
    lists = (None, None)
    if k:
        g = gen(rows, dev)
        lists = (6.0 - 2.5 * torch.log1p(torch.arange(k, device=dev).float()) + 0.3 * torch.randn(rows, k, generator=g, device=dev),
                 ((labels.unsqueeze(1) + 611 * torch.arange(k, device=dev)) % 3000).int())
    o = outputs(dev, rows)
    got = dict(dh=torch.empty_like(h), **({"dweight": torch.empty_like(w)} if "w" in grad else {}))
    more = dict(top_vals=lists[0], top_idx=lists[1], temperature=temp, alpha=alpha) if k else {}
    sc = torch.tensor([2048.0], device=dev)
    ops.linear_cross_entropy(h, w, labels, loss_scale=sc, **o, **got, **more)
    ref = R.linear(h, w, labels, 2048.0, None, temp, alpha, *lists)
    for n, x in got.items():
        want = ref["dh" if n == "dh" else "dw"]
        own = (want.to(dtype).double() - want).norm()             # what the result's own rounding costs
        assert (x.double() - want).norm() <= 1.3 * own, n


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sharp", [4.0, 12.0])
def test_labels_that_are_almost_certain(ops, dev, dtype, sharp):
    """1 - p from 0.5 down to nothing: the gradient keeps its own digits, none is lost to p's"""
    h, w, labels, _ = make_linear(dev, 200, 128, 1500, dtype, seed=15, ignored=0.1, sharp=0.0)
    h = (h.float() * 0.3 + sharp * w[labels.clamp(0, 1499)].float() * torch.linspace(0.5, 1.0, 200, device=dev).unsqueeze(1)).to(dtype)
    for grad in ("h", "hw"):
        check_linear(ops, dev, h, w, labels, grad=grad, scale=64.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,v,grad,k,alpha,temp", [(300, 2600, "hw", 0, 0.0, 1.0), (300, 2600, "hw", 5, 0.5, 1.0), (130, 900, "h", 3, 1.0, 2.0), (300, 2600, "h", 0, 0.0, 1.0), (100, 70, "w", 0, 0.0, 1.0), (2049, 60001, "h", 0, 0.0, 1.0)])
def test_labels_far_below_the_largest_logit(ops, dev, dtype, rows, v, grad, k, alpha, temp):
    """rows from nearly flat to logits of hundreds, the label anywhere among them: a reference taken from the label's logit holds for some rows, by a little
    for others and not for the rest; one row of a tile, all of them or none; label and maximum in one strip and far apart"""
    h, w, labels, lists = make_linear(dev, rows, 64, v, dtype, seed=13, ignored=0.1, k=k, sharp=0.0)
    grow = torch.linspace(0.05, 12.0, rows, device=dev).unsqueeze(1)
    for i, part in enumerate((grow, torch.where(torch.arange(rows, device=dev).unsqueeze(1) % 97 == 0, 12.0, 0.3), torch.full_like(grow, 6.0))):
        check_linear(ops, dev, (h * part).to(dtype), w, labels, lists, temp, alpha, grad=grad, scale=8.0)
        if rows > 2000:
            break


def test_labels_whose_logit_is_a_small_difference_of_large_products(ops, dev):
    """the gathered logit and the tile's may then differ by more than a reference allows for; rows that lose all digits are held to no value, the others to theirs"""
    h, w, labels, _ = make_linear(dev, 300, 64, 700, BF16, seed=14, ignored=0.0)
    w[:, 32:] = -w[:, :32]
    big = torch.arange(300, device=dev) % 3 == 0
    h[:, 32:] = torch.where(big.unsqueeze(1), h[:, :32], h[:, 32:])
    h[big] *= 2.0 ** 40                        # products of 2^40 that cancel in pairs: logits of zero but for what the order of the sum leaves
    o = outputs(dev, 300)
    dh = torch.full_like(h, 3.0)
    ops.linear_cross_entropy(h, w, labels, dh=dh, **o)
    ref = R.linear(h, w, labels)
    small = (labels >= 0) & (labels < 700) & ~big
    close(o["row_loss"][small], ref["row_loss"][small], ref["row_tol"][small], "row_loss")
    assert torch.isfinite(o["row_loss"]).all() and torch.isfinite(dh).all()
    close(dh[small], ref["dh"][small], ref["dh_tol"][small], "dh")


@pytest.mark.parametrize("rows", [40, 600])
def test_same_inputs_give_the_same_bits_and_workspaces_are_not_shared(ops, dev, rows):
    """repeated, interleaved with another call, on another stream and with a caller's workspace: equal bits; nothing past the workspace is written"""
    h, w, labels, lists = make_linear(dev, rows, 256, 3001, F16, seed=8, k=20)
    h2, w2, labels2, _ = make_linear(dev, 500, 128, 900, F16, seed=9)
    kw = dict(top_vals=lists[0], top_idx=lists[1], temperature=2.0, alpha=0.5)

    def once(**more):
        o = outputs(dev, rows)
        dh, dw = torch.empty_like(h), torch.empty_like(w)
        ops.linear_cross_entropy(h, w, labels, dh=dh, dweight=dw, **o, **kw, **more)
        return [o["row_loss"], o["loss"], dh, dw]
    a = once()
    o2 = outputs(dev, 500)
    ops.linear_cross_entropy(h2, w2, labels2, dh=torch.empty_like(h2), **o2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = once()
    c = once()
    need = ops.linear_ce_workspace_bytes(h, w, labels, dh=torch.empty_like(h), dweight=torch.empty_like(w), **outputs(dev, rows), **kw)
    ws = torch.full((need + 4096,), 0xA5, device=dev, dtype=torch.uint8)
    e = once(workspace=ws[:need])
    torch.cuda.synchronize()
    assert (ws[need:] == 0xA5).all()
    for other in (b, c, e):
        for x, y in zip(a, other):
            assert torch.equal(x, y)
    with pytest.raises(ValueError, match="workspace"):
        once(workspace=ws[:need - 256])


@pytest.mark.parametrize("rows", [9, 70, 600])
@pytest.mark.parametrize("dtype,grad,k,alpha,temp", [(F16, "h", 0, 0.0, 1.0), (BF16, "h", 0, 0.0, 1.0), (BF16, "hw", 0, 0.0, 1.0), (BF16, "w", 0, 0.0, 1.0), (BF16, "h", 5, 0.5, 1.0),
                                                     (BF16, "hw", 5, 0.5, 1.0), (F16, "hw", 0, 0.0, 1.0), (F16, "h", 5, 1.0, 2.0), (F16, "hw", 5, 0.5, 2.0), (BF16, "hw", 5, 0.5, 4.0)])
def test_what_a_workspace_holds_does_not_matter(ops, dev, rows, dtype, grad, k, alpha, temp):
    """every form of the call over workspaces full of NaN, of other numbers and of the call before, with NaN in the masked rows: the same bits, on another stream too, twice over at a time"""
    h, w, labels, lists = make_linear(dev, rows, 136, 1300, dtype, seed=18, ignored=0.4, k=k)
    off = ~((labels >= 0) & (labels < 1300))
    h[off] = float("nan")
    kw = dict(top_vals=lists[0], top_idx=lists[1], temperature=temp, alpha=alpha) if k else {}

    def bufs():
        b = outputs(dev, rows)
        if "h" in grad:
            b["dh"] = torch.full_like(h, 3.0)
        if "w" in grad:
            b["dweight"] = torch.full_like(w, 3.0)
        return b
    first = bufs()
    ops.linear_cross_entropy(h, w, labels, **first, **kw)
    need = ops.linear_ce_workspace_bytes(h, w, labels, **first, **kw)
    side = torch.cuda.Stream()
    got = []
    for fill in (0xFF, 0x3C, 0x00):
        ws = torch.full((2, (need + 255) // 256 * 256), fill, device=dev, dtype=torch.uint8)
        side.wait_stream(torch.cuda.current_stream())
        for i in range(2):
            b = bufs()
            ops.linear_cross_entropy(h, w, labels, workspace=ws[0], **b, **kw)
            got.append(b)
        with torch.cuda.stream(side):
            b = bufs()
            ops.linear_cross_entropy(h, w, labels, workspace=ws[1], **b, **kw)
            got.append(b)
        torch.cuda.synchronize()
    for b in got:
        for n in first:
            assert torch.equal(b[n], first[n]), n
    if "h" in grad:
        assert (first["dh"][off] == 0).all() and torch.isfinite(first["dh"]).all()
    if "w" in grad:
        assert torch.isfinite(first["dweight"]).all()


@pytest.mark.parametrize("rows", [50, 260])
def test_captured_graphs_replay_with_new_data(ops, dev, rows):
    """two graphs, replayed several times between eager calls, against eager results"""
    sets = [make_linear(dev, rows, 128, 1200, BF16, seed=s, k=6) for s in (10, 11, 12)]
    h, w, labels = (t.clone() for t in sets[0][:3])
    tv, ti = (t.clone() for t in sets[0][3])

    def bufs():
        return dict(outputs(dev, rows), dh=torch.empty_like(h), dweight=torch.empty_like(w))

    def call(b):
        ops.linear_cross_entropy(h, w, labels, top_vals=tv, top_idx=ti, temperature=2.0, alpha=0.5, **b)

    def call_hard(b):
        ops.linear_cross_entropy(h, w, labels, **b)
    eager, ga, gb = bufs(), bufs(), bufs()
    call(eager)
    torch.cuda.synchronize()
    from neuspeech1_amd.lib import capture_section
    graphs = []
    for fn, b in ((call, ga), (call_hard, gb)):
        g = torch.cuda.CUDAGraph()
        with capture_section(), torch.cuda.graph(g, capture_error_mode="thread_local"):
            fn(b)
        graphs.append(g)
    for hh, ww, ll, (a, i) in sets + sets[:1]:
        h.copy_(hh), w.copy_(ww), labels.copy_(ll), tv.copy_(a), ti.copy_(i)
        for fn, g, b in ((call, graphs[0], ga), (call_hard, graphs[1], gb)):
            fn(eager)
            want = {n: t.clone() for n, t in eager.items()}
            g.replay()
            torch.cuda.synchronize()
            for n in want:
                assert torch.equal(b[n], want[n]), n


def test_gradients_against_differences_of_the_loss(ops, dev):
    """central differences of the kernel's own loss along random directions.  h is a multiple of 2^-5 and the step 2^-4 times directions of -1, 0, 1:
    the moved h is exact.  The loss along a line has a third derivative below 2 r^3 a row, r = the range of the logits' change per step."""
    g = gen(13, dev)
    rows, d, v, eps = 40, 64, 200, 2.0 ** -4
    w = (torch.randn(v, d, generator=g, device=dev) * 0.25).half()
    h = (torch.randn(rows, d, generator=g, device=dev) * 32).round().div(32).half()
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    tv, ti = make_lists(dev, g, rows, v, 7, labels)
    kw = dict(top_vals=tv, top_idx=ti, temperature=2.0, alpha=0.5)
    dh = torch.empty_like(h)
    ops.linear_cross_entropy(h, w, labels, dh=dh, loss_scale=torch.tensor([256.0], device=dev), **outputs(dev, rows), **kw)
    ref = R.linear(h, w, labels, 256.0, None, 2.0, 0.5, tv, ti)
    for _ in range(4):
        u = torch.randint(-1, 2, (rows, d), generator=g, device=dev).half()
        f = []
        for s in (1, -1):
            o = outputs(dev, rows)
            ops.linear_cross_entropy(h + s * eps * u, w, labels, **o, **kw)
            f.append(o["row_loss"].double())
        slope = (f[0] - f[1]) / (2 * eps)
        line = u.double() @ w.double().t()
        r = line.amax(1) - line.amin(1)
        got = (dh.double() / 256.0 * rows * u.double()).sum(1)
        tol = eps ** 2 / 6 * 2 * r ** 3 + ref["row_tol"] * 1.5 / eps + (ref["dh_tol"] / 256.0 * rows).sum(1)
        assert ((slope - got).abs() <= tol).all()
        assert float((slope - got).abs().mean()) < 0.05 * float(got.abs().mean())


# ------------------------------------------------------------------------------------------------ distillation over logits
def make_logits(dev, rows, v, dtype, seed, pad=0, first=0, ignored=0.3, k=5):
    g = gen(seed, dev)
    buf = (torch.randn(rows, v + pad + first, generator=g, device=dev) * 3).to(dtype)
    z = buf[:, first:first + v]
    labels = torch.randint(0, v, (rows,), generator=g, device=dev)
    labels = torch.where(torch.rand(rows, generator=g, device=dev) < ignored, -100, labels)
    return buf, z, labels, make_lists(dev, g, rows, v, k, labels)


def check_distill(ops, dev, z, labels, lists, temp, alpha, dz=None, scale=None):
    rows, v = z.shape
    zd = z.double()
    o = outputs(dev, rows)
    sc = None if scale is None else torch.tensor([scale], device=dev)
    ops.distill_topk(z, labels, *lists, temperature=temp, alpha=alpha, dlogits=dz, loss_scale=sc, **o)
    torch.cuda.synchronize()
    valid = torch.ones(rows, dtype=torch.bool, device=dev) if labels is None else (labels >= 0) & (labels < v)
    ref = R.losses(torch.where(valid.unsqueeze(1), zd, torch.zeros_like(zd)), torch.zeros((), dtype=torch.float64, device=dev), labels, temp, alpha, *lists)
    assert int(o["nvalid"]) == ref["nvalid"]
    close(o["row_loss"], ref["row_loss"], ref["row_tol"], "row_loss")
    close(o["loss"], ref["loss"].reshape(1), ref["loss_tol"].reshape(1), "loss")
    if dz is not None:
        gs = (scale or 1.0) / ref["n"]
        U = R.half_step(z.dtype)
        want = ref["cell"] * gs
        small = {F16: 2.0 ** -25, BF16: 2.0 ** -126, F32: 2.0 ** -126}[z.dtype]
        close(dz, want, (ref["cell_err"] * gs + 4 * R.U32 * want.abs()) * (1 + U) + U * want.abs() + small, "dlogits")
    return o


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,v,pad,first,k", [(1, 1, 0, 0, 1), (7, 9, 0, 0, 3), (9, 1000, 24, 0, 8), (8, 1001, 2, 3, 33), (3, 2050, 1, 1, 256), (5, 9001, 0, 0, 64),
                                                (2, 33003, 5, 2, 12), (3, 51865, 103, 0, 64), (2, 70001, 0, 0, 20)])
@pytest.mark.parametrize("temp,alpha", [(2.0, 0.5), (1.0, 0.5), (4.0, 1.0), (4.0, 0.5), (1.5, 0.3)])
def test_distill_topk(ops, dev, dtype, rows, v, pad, first, k, temp, alpha):
    buf, z, labels, lists = make_logits(dev, rows, v, dtype, rows + v, pad, first, k=k)
    ob = torch.full_like(buf, 5.0)
    dz = ob[:, first:first + v]
    check_distill(ops, dev, z, labels, lists, temp, alpha, dz, scale=64.0)
    dz.fill_(5.0)
    assert (ob == 5.0).all()                                   # columns beside the view are left as they were
    other = torch.full((rows, v + 9), 5.0, device=dev, dtype=dtype)[:, 3:v + 3]      # another alignment than the logits'
    check_distill(ops, dev, z, labels, lists, temp, alpha, other)
    check_distill(ops, dev, z, labels, lists, temp, alpha)     # the loss alone


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("v", [300, 5000, 66000])
def test_distill_topk_in_place(ops, dev, dtype, v):
    buf, z, labels, lists = make_logits(dev, 9, v, dtype, 21, 1, 0, k=9)
    out = torch.empty_like(z)
    ops.distill_topk(z, labels, *lists, temperature=2.0, alpha=0.5, dlogits=out, **outputs(dev, 9))
    keep = buf[:, v:].clone()
    ops.distill_topk(z, labels, *lists, temperature=2.0, alpha=0.5, dlogits=z, **outputs(dev, 9))
    assert torch.equal(z, out) and torch.equal(buf[:, v:], keep)


def test_distill_topk_without_labels_and_with_masked_rows(ops, dev):
    buf, z, labels, lists = make_logits(dev, 20, 700, F32, 22, k=4)
    check_distill(ops, dev, z, None, lists, 2.0, 1.0, torch.empty_like(z))
    off = labels < 0
    z[off] = float("nan")
    lists[0][off] = float("nan")
    dz = torch.empty_like(z)
    o = check_distill(ops, dev, z, labels, lists, 2.0, 0.5, dz)
    assert (dz[off] == 0).all() and (o["row_loss"][off] == 0).all()
    labels.fill_(-100)
    o = check_distill(ops, dev, z, labels, lists, 2.0, 0.5, dz)
    assert (dz == 0).all() and float(o["loss"]) == 0
    o = outputs(dev, 0)
    ops.distill_topk(z[:0], labels[:0], lists[0][:0], lists[1][:0], alpha=0.5, dlogits=dz[:0], **o)
    assert float(o["loss"]) == 0 and int(o["nvalid"]) == 0


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_distill_topk_with_masked_logits(ops, dev, dtype):
    """student logits of -inf and of the type's lowest value: finite losses where the targets do not name them, zero probability there; a row of the lowest
    value alone is a uniform distribution"""
    buf, z, labels, lists = make_logits(dev, 6, 900, dtype, 23, ignored=0.0, k=5)
    named = torch.zeros(6, 900, dtype=torch.bool, device=dev)
    named.scatter_(1, lists[1].clamp(0, 899).long(), True)
    named.scatter_(1, labels.clamp(0, 899).unsqueeze(1), True)
    z[:, ::3] = torch.where(named[:, ::3], z[:, ::3], float("-inf"))
    z[:, 1::3] = torch.where(named[:, 1::3], z[:, 1::3], torch.finfo(dtype).min)
    z[2] = torch.finfo(dtype).min
    dz = torch.empty_like(z)
    o = outputs(dev, 6)
    ops.distill_topk(z, labels, *lists, temperature=2.0, alpha=0.5, dlogits=dz, **o)
    ref = R.losses(z.double(), torch.zeros((), dtype=torch.float64, device=dev), labels, 2.0, 0.5, *lists)
    fin = torch.isfinite(ref["row_loss"])
    assert torch.isfinite(o["row_loss"][fin]).all() and fin.any() and torch.isfinite(dz[fin]).all()
    assert ((o["row_loss"].double() - ref["row_loss"]).abs()[fin] <= 1e-4).all()      # (z of -65504 in the tolerance's |z| would say nothing)
    rest = [0, 1, 3, 4, 5]
    assert (dz[rest, ::3][~named[rest, ::3]] == 0).all() and (dz[rest, 1::3][~named[rest, 1::3]] == 0).all()
    flat = dz[2][~named[2]].double() * 6
    assert ((flat - 1.5 / 900).abs() <= (2 * R.half_step(dtype) + 200 * R.U32) * 1.5 / 900).all()       # w1 + w2 = 0.5 + 0.5 * 2 over 900 tokens


# ------------------------------------------------------------------------------------------------ the teacher's lists
def ref_topk(z, k):
    z = z.double()
    key = torch.where(torch.isnan(z), torch.full_like(z, float("inf")), z)
    nan = torch.isnan(z)
    vals, idx = [], []
    for r in range(z.shape[0]):
        order = sorted(range(z.shape[1]), key=lambda c: (not bool(nan[r, c]), -float(key[r, c]), c)) if z.shape[1] <= 600 else None
        if order is None:
            order = torch.sort(z[r] + 0.0, descending=True, stable=True).indices[:k].tolist()
        idx.append(order[:k])
        vals.append([float(z[r, c]) for c in order[:k]])
    return torch.tensor(vals, dtype=torch.float64), torch.tensor(idx)


def check_topk(ops, dev, z, k):
    rows, v = z.shape
    vals = torch.empty(rows, k, device=dev)
    idx = torch.empty(rows, k, device=dev, dtype=torch.int32)
    lse = torch.empty(rows, device=dev)
    ops.topk_logits(z, k, vals=vals, idx=idx, lse=lse)
    rv, ri = ref_topk(z.cpu(), k)
    assert torch.equal(idx.cpu().long(), ri)
    assert torch.equal(torch.nan_to_num(vals.cpu().double(), nan=1e30), torch.nan_to_num(rv, nan=1e30))
    want = torch.logsumexp(z.double(), 1)
    fin = torch.isfinite(want)
    close(lse[fin], want[fin], (160 + 8 * z.double().abs().amax(1)[fin].clamp(min=1)) * R.U32, "lse")
    return vals, idx, lse


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,v,pad,first,k", [(1, 1, 0, 0, 1), (4, 9, 0, 0, 9), (5, 257, 3, 1, 256), (3, 1000, 0, 0, 128), (3, 2050, 1, 2, 7), (2, 9001, 0, 0, 256),
                                                (2, 33003, 5, 3, 100), (3, 51865, 103, 0, 64), (2, 70001, 1, 0, 33)])
def test_topk_logits(ops, dev, dtype, rows, v, pad, first, k):
    g = gen(v + k, dev)
    z = (torch.randn(rows, v + pad + first, generator=g, device=dev) * 3).to(dtype)[:, first:first + v]
    check_topk(ops, dev, z, k)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("v", [500, 9001, 51865])
def test_topk_logits_of_equal_values(ops, dev, dtype, v):
    """rows of one value, of two values, of the lowest value and -inf, of zeros of both signs: lowest tokens first, and the long way round the buffer"""
    z = torch.zeros(6, v, device=dev, dtype=dtype)
    z[0] = 1.5
    z[1] = 1.0
    z[1, 5::7] = 2.0
    z[2] = float("-inf")
    z[2, 3] = torch.finfo(dtype).min
    z[3, ::2] = -0.0
    z[4] = torch.arange(v, device=dev).remainder(5).to(dtype)
    z[5] = 3.0
    z[5, v - 20:] = 4.0
    check_topk(ops, dev, z, 64)


def test_topk_logits_with_infinities_and_nan(ops, dev):
    z = torch.randn(3, 400, device=dev)
    z[0, 100], z[0, 50] = float("inf"), float("inf")
    z[1, 7], z[1, 300], z[1, 2] = float("nan"), -float("nan"), float("inf")
    z[2] = float("-inf")
    vals, idx, lse = check_topk(ops, dev, z, 5)
    assert idx[1, :3].tolist() == [7, 300, 2] and lse[0] == float("inf") and torch.isnan(lse[1]) and lse[2] == float("-inf")


# ------------------------------------------------------------------------------------------------ together
def test_teacher_lists_distil_a_student_head(ops, dev):
    """a teacher's logits -> its lists -> the student's head without logits, and over logits: the same loss and, through the head, the same gradient;
    a captured step learns: replays equal eager calls"""
    g = gen(31, dev)
    rows, d, v, k = 200, 128, 1500, 32
    teacher = (torch.randn(rows, v + 20, generator=g, device=dev) * 3).half()[:, :v]
    h, w, labels, _ = make_linear(dev, rows, d, v, F16, seed=32)
    tv, ti = torch.empty(rows, k, device=dev), torch.empty(rows, k, device=dev, dtype=torch.int32)
    lse = torch.empty(rows, device=dev)
    ops.topk_logits(teacher, k, vals=tv, idx=ti, lse=lse)
    scale = torch.tensor([256.0], device=dev)
    a, b = outputs(dev, rows), outputs(dev, rows)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ops.linear_cross_entropy(h, w, labels, top_vals=tv, top_idx=ti, temperature=2.0, alpha=0.5, dh=dh, dweight=dw, loss_scale=scale, **a)
    z = h.float() @ w.float().t()
    dz = torch.empty_like(z)
    ops.distill_topk(z, labels, tv, ti, temperature=2.0, alpha=0.5, dlogits=dz, loss_scale=scale, **b)
    ref = R.linear(h, w, labels, 256.0, None, 2.0, 0.5, tv, ti)
    close(a["row_loss"], ref["row_loss"], ref["row_tol"], "row_loss, linear")
    close(b["row_loss"], ref["row_loss"], ref["row_tol"], "row_loss, logits")
    close(dh, ref["dh"], ref["dh_tol"], "dh")
    close(dw, ref["dw"], ref["dw_tol"], "dw")
    close(dz.double() @ w.double(), ref["dh"], ref["dh_tol"], "dz W")
    # hard labels alone: ops.cross_entropy over fp16 logits is the same loss up to the logits' rounding (2^-11 of |z| <= 32)
    hard = outputs(dev, rows)
    ops.linear_cross_entropy(h, w, labels, **hard)
    z16 = torch.zeros(rows, (v + 7) // 8 * 8, device=dev, dtype=F16)
    z16[:, :v] = z
    old = outputs(dev, rows)
    ops.cross_entropy(z16, labels, rows, v, z16.shape[1], old["row_loss"], None, old["nvalid"], None, old["loss"])
    assert int(old["nvalid"]) == int(hard["nvalid"])
    assert float((old["row_loss"] - hard["row_loss"]).abs().max()) <= 2 * 2.0 ** -11 * float(z.abs().max()) + 1e-4
    from neuspeech1_amd.lib import capture_section
    graph = torch.cuda.CUDAGraph()
    got = [torch.empty_like(t) for t in (dh, dw, dz)]
    c, e = outputs(dev, rows), outputs(dev, rows)
    torch.cuda.synchronize()
    with capture_section(), torch.cuda.graph(graph, capture_error_mode="thread_local"):
        ops.topk_logits(teacher, k, vals=tv, idx=ti, lse=lse)
        ops.linear_cross_entropy(h, w, labels, top_vals=tv, top_idx=ti, temperature=2.0, alpha=0.5, dh=got[0], dweight=got[1], loss_scale=scale, **c)
        ops.distill_topk(z, labels, tv, ti, temperature=2.0, alpha=0.5, dlogits=got[2], loss_scale=scale, **e)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got + [c["row_loss"], e["row_loss"]], (dh, dw, dz, a["row_loss"], b["row_loss"])):
            assert torch.equal(x, y)
        w.sub_((dw.float() / 256).half())                       # the student learns; the graph reads the new weight
        z.copy_(h.float() @ w.float().t())
        ops.linear_cross_entropy(h, w, labels, top_vals=tv, top_idx=ti, temperature=2.0, alpha=0.5, dh=dh, dweight=dw, loss_scale=scale, **a)
        ops.distill_topk(z, labels, tv, ti, temperature=2.0, alpha=0.5, dlogits=dz, loss_scale=scale, **b)
        torch.cuda.synchronize()
    assert math.isfinite(float(a["loss"]))
