"""CPU: sizes that one launch cannot hold are refused before anything is launched (no address given here is ever read)."""
import ctypes as C

import pytest

from neuspeech1_amd import lib

AT = 1 << 20          # stands for a device address: aligned, never followed


def distill(rows, vocab, dtype):
    d = lib.DistillDesc()
    for n in ("logits", "labels", "top_vals", "top_idx", "row_loss", "loss_dev", "nvalid_dev", "dlogits"):
        setattr(d, n, AT)
    d.ldz = d.lddz = vocab
    d.rows, d.vocab, d.k, d.ld_top, d.dtype, d.temperature, d.alpha = rows, vocab, 4, 4, dtype, 1.0, 1.0
    return d


@pytest.mark.parametrize("rows,vocab,dtype", [(1 << 24, 100, lib.NS_F16), (1 << 24, 4103, lib.NS_BF16), (1 << 22, 51865, lib.NS_F16), (1 << 22, 2100, lib.NS_F32), (2 ** 31 - 1, 1, lib.NS_F32)])
def test_rows_that_one_launch_cannot_hold(rows, vocab, dtype):
    so = lib.load()
    assert so.ns_distill_topk(C.byref(distill(rows, vocab, dtype)), None) == -1 and b"too many" in so.ns_last_error()
    d = lib.TopkDesc()
    d.logits, d.vals, d.idx, d.ldz, d.ldo = AT, AT, AT, vocab, 1
    d.rows, d.vocab, d.k, d.dtype = rows, vocab, 1, dtype
    assert so.ns_topk_logits(C.byref(d), None) == -1 and b"too many" in so.ns_last_error()


@pytest.mark.parametrize("rows,d,vocab", [(1 << 21, 65536, 300), (1 << 21, 1280, 300000), (600000, 2048, 262144)])
def test_a_dh_that_one_launch_cannot_hold(rows, d, vocab):
    so = lib.load()
    a = lib.LinearCeDesc()
    for n in ("h", "w", "labels", "row_loss", "loss_dev", "nvalid_dev", "dh", "workspace"):
        setattr(a, n, AT)
    a.ldh = a.ldw = a.lddh = d
    a.rows, a.vocab, a.d, a.dtype, a.temperature = rows, vocab, d, lib.NS_BF16, 1.0
    a.workspace_bytes = so.ns_linear_ce_workspace_bytes(C.byref(a))
    assert so.ns_linear_cross_entropy(C.byref(a), None) == -1 and b"too many" in so.ns_last_error()
