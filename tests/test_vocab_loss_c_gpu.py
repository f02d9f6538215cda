"""GPU: the C entry points of the vocabulary losses where the Python calls never lead."""
import ctypes as C

import pytest
import torch

from neuspeech1_amd import lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,code", [(torch.float16, lib.NS_F16), (torch.bfloat16, lib.NS_BF16)])
@pytest.mark.parametrize("with_dw", [False, True])
def test_no_rows_with_gradients_asked_for(dev, dtype, code, with_dw):
    """rows = 0 with dh set: a loss of zero over no rows, dW zero, nothing else written"""
    so = lib.load()
    w = torch.randn(300, 64, device=dev).to(dtype)
    dh, dw = torch.full((4, 64), 3.0, device=dev, dtype=dtype), torch.full_like(w, 3.0)
    loss, nvalid = torch.full((1,), 7.0, device=dev), torch.full((1,), 7, device=dev, dtype=torch.int32)
    d = lib.LinearCeDesc()
    d.w, d.ldw, d.ldh, d.dh, d.lddh = w.data_ptr(), 64, 64, dh.data_ptr(), 64
    if with_dw:
        d.dw, d.lddw = dw.data_ptr(), 64
    d.loss_dev, d.nvalid_dev = loss.data_ptr(), nvalid.data_ptr()
    d.rows, d.vocab, d.d, d.dtype, d.temperature = 0, 300, 64, code, 1.0
    need = so.ns_linear_ce_workspace_bytes(C.byref(d))
    ws = torch.empty(need, device=dev, dtype=torch.uint8)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    assert so.ns_linear_cross_entropy(C.byref(d), torch.cuda.current_stream().cuda_stream) == 0, so.ns_last_error()
    torch.cuda.synchronize()
    assert float(loss) == 0 and int(nvalid) == 0 and (dh == 3.0).all() and (dw == (0.0 if with_dw else 3.0)).all()


def test_gradients_beside_their_operands_in_one_buffer(dev):
    """h | dh and logits | dlogits as columns of one buffer: the values they have apart, and nothing else of the buffer is written.  (A row of logits that starts elsewhere within 16 bytes is
    added up in another order: dlogits by its bound against 64 bits.)"""
    from neuspeech1_amd import ops
    from tests import vocab_loss_ref as R
    from tests.test_vocab_loss_gpu import close, make_linear, make_logits, outputs
    for rows in (30, 200):
        h, w, labels, _ = make_linear(dev, rows, 64, 300, torch.float16, seed=61)
        buf = torch.full((rows, 160), 5.0, device=dev, dtype=torch.float16)
        buf[:, :64] = h
        want = torch.empty_like(h)
        ops.linear_cross_entropy(h, w, labels, dh=want, **outputs(dev, rows))
        ops.linear_cross_entropy(buf[:, :64], w, labels, dh=buf[:, 80:144], **outputs(dev, rows))
        assert torch.equal(buf[:, 80:144], want) and torch.equal(buf[:, :64], h) and (buf[:, 64:80] == 5.0).all() and (buf[:, 144:] == 5.0).all()
        _, z, labels, (tv, ti) = make_logits(dev, rows, 301, torch.float32, 62)
        buf = torch.full((rows, 700), 5.0, device=dev)
        buf[:, :301] = z
        ops.distill_topk(buf[:, :301], labels, tv, ti, alpha=0.5, dlogits=buf[:, 303:604], **outputs(dev, rows))
        ref = R.losses(z.double(), torch.zeros((), dtype=torch.float64, device=dev), labels, 1.0, 0.5, tv, ti)
        want = ref["cell"] / ref["n"]
        close(buf[:, 303:604], want, ref["cell_err"] / ref["n"] + 6 * R.U32 * want.abs() + 2.0 ** -126, "dlogits")
        assert torch.equal(buf[:, :301], z) and (buf[:, 301:303] == 5.0).all() and (buf[:, 604:] == 5.0).all()
