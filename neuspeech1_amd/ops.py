"""Thin torch-tensor front end over the C ABI (ctypes).  PyTorch supplies device
memory and streams only; every FLOP happens in libneuspeech_hip.so."""
from __future__ import annotations

import ctypes as C

import torch

from . import lib as L
from .lib import (AdamWCfg, AttnDesc, CastJob, GemmDesc, RowMap, NS_GEMM_ATOMIC32, NS_GEMM_COLSUM_A, NS_GEMM_DGELU, NS_GEMM_DROP_A,
                  NS_GEMM_GELU, NS_GEMM_GELU_SAVE_GRAD, NS_GEMM_MUL_P16, NS_GEMM_TN)

__all__ = ["gemm", "rowmap", "ptr", "layernorm_fwd", "layernorm_bwd", "signal_pack", "feed_pack", "embed_pos", "attn_fwd",
           "attn_bwd", "cross_entropy", "linear_cross_entropy", "linear_ce_workspace_bytes", "distill_topk", "topk_logits", "dgelu_mul", "colsum", "argmax_rows", "grad_norm", "adamw_step", "cast_jobs", "make_cast_jobs",
           "NS_GEMM_GELU", "NS_GEMM_DGELU", "NS_GEMM_TN", "NS_GEMM_ATOMIC32", "NS_GEMM_DROP_A", "NS_GEMM_GELU_SAVE_GRAD",
           "NS_GEMM_MUL_P16", "NS_GEMM_COLSUM_A"]


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    """hipStream_t of torch's CURRENT stream on the current device (graph capture and the DP side stream switch it).
    The raw accessor is ~20x cheaper than torch.cuda.current_stream(): 374 launches per training step call this."""
    if _raw_stream is not None:
        return _raw_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


# ---- launch lists: a host-side stand-in for a hipGraph where capturing one does not pay (generate.py: short generations).
# While a list is being RECORDED on this thread, entry points are not launched but appended -- function, marshalled arguments -- exactly
# as a stream capture records instead of executing; replay() then issues them on the current stream at ~1 us of host time per launch,
# where building a descriptor through ctypes costs ~10 us (40 field stores, a dozen data_ptr() calls): a decode step of ~80 launches is
# 0.8-1.0 ms of host work built afresh against 0.84 ms of GPU time, i.e. host-bound on a slow host, and 0.1 ms replayed.
import threading as _threading

_tls = _threading.local()


class LaunchList:
    """Entries hold RAW device addresses (the marshalled ctypes arguments), exactly as a captured hipGraph does: `keep` is where the
    recorder parks whatever owns that memory (generate.py: the decode session whose tensors the launches point into), so a list can
    never outlive its buffers.  Only entry points that go through _call() are recorded: a torch op issued inside a recorded region runs
    once, at record time, and is absent from every replay -- NS_LISTS_VERIFY=1 makes generate() check a freshly recorded list against
    eager launches (tests/test_generate_gpu.py)."""
    __slots__ = ("calls", "keep")

    def __init__(self):
        self.calls = []
        self.keep = None

    def replay(self):
        st = _stream()
        for fn, name, args in self.calls:
            rc = fn(*args, st)
            if rc:
                L.check(rc, name)


class recording:
    """with ops.recording(launch_list): ... -- this thread's entry-point calls are recorded into the list, not launched"""

    def __init__(self, lst: LaunchList):
        self.lst = lst

    def __enter__(self):
        assert getattr(_tls, "rec", None) is None, "nested ops.recording"
        _tls.rec = self.lst
        return self.lst

    def __exit__(self, *exc):
        _tls.rec = None
        return False


STEP_PROFILE = None   # set to a list by bench.py: every entry-point launch is then bracketed by HIP events on the launch stream and recorded as
#                       (class, flop, algorithmic bytes, e0, e1); the class / work come from the wrapper (_work) or default to the entry point's name


def _work(cls: str, flop: float = 0.0, nbytes: float = 0.0):
    """wrapper -> _call: the class and the ALGORITHMIC work (FLOP, HBM bytes: every operand once) of the launch that follows"""
    if STEP_PROFILE is not None:
        _tls.work = (cls, float(flop), float(nbytes))


def _call(name: str, *args):
    fn = getattr(L.load(), name)
    rec = getattr(_tls, "rec", None)
    if rec is not None:
        rec.calls.append((fn, name, args))
        return
    if STEP_PROFILE is None:
        L.check(fn(*args, _stream()), name)
        return
    work = getattr(_tls, "work", None) or (name[3:] if name.startswith("ns_") else name, 0.0, 0.0)
    _tls.work = None
    st = torch.cuda.current_stream()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record(st)
    L.check(fn(*args, _stream()), name)
    e1.record(st)
    STEP_PROFILE.append((*work, e0, e1))


def ptr(t, off: int = 0) -> int:
    """Device address of tensor element `off` (0 for None)."""
    if t is None:
        return 0
    if isinstance(t, int):
        return t
    if isinstance(t, tuple):
        t, off = t
    return t.data_ptr() + off * t.element_size()


def rowmap(ld: int, seg_rows: int = 0, seg_stride: int = 0) -> RowMap:
    return RowMap(int(seg_stride), int(seg_rows), int(ld))


_ZERO_MAP = RowMap(0, 0, 0)
GEMM_PROFILE = None   # set to a list by bench.py to time every GEMM launch with HIP events


def _fill_gemm_desc(d, *, A, am, K, B, ldb=None, bm=None, M, N, A2=None, am2=None, K2=0, B2=None, ldb2=0, a2_ngroup=0,
                    bias=None, C16=None, c16m=None, G16=None, g16m=None, P16=None, p16m=None, R32=None, H32=None, h32m=None,
                    pos=None, pos_rows=0, C32=None, ldc32=0, flags=0, splits=1, drop_p=0.0, drop_seed=0, alpha=0.0,
                    side_B=None, side_ldb=0, side_n=0, side_out=None, side_drop_p=0.0, side_drop_seed=0, k_alg=None, seed_dev=None):
    d.side_B, d.side_ldb, d.side_n, d.side_out = ptr(side_B), side_ldb, side_n, ptr(side_out)
    d.side_drop_p, d.side_drop_seed = side_drop_p, side_drop_seed
    d.seed_dev = ptr(seed_dev)
    d.A, d.am, d.K = ptr(A), am, K
    d.B = ptr(B)
    d.bm = bm if bm is not None else rowmap(ldb)
    d.A2, d.am2, d.K2 = ptr(A2), (am2 if am2 is not None else _ZERO_MAP), K2
    d.B2, d.ldb2, d.a2_ngroup = ptr(B2), ldb2, a2_ngroup
    d.M, d.N = M, N
    d.bias = ptr(bias)
    d.C16, d.c16m = ptr(C16), (c16m if c16m is not None else _ZERO_MAP)
    d.G16, d.g16m = ptr(G16), (g16m if g16m is not None else _ZERO_MAP)
    d.P16, d.p16m = ptr(P16), (p16m if p16m is not None else _ZERO_MAP)
    d.R32, d.H32, d.h32m = ptr(R32), ptr(H32), (h32m if h32m is not None else _ZERO_MAP)
    d.pos, d.pos_rows = ptr(pos), pos_rows
    d.C32, d.ldc32 = ptr(C32), ldc32
    d.flags, d.splits = flags, splits
    d.drop_p, d.drop_seed, d.alpha = drop_p, drop_seed, alpha
    return d


def _gemm_kind(kw) -> str:
    """which kernel family ns_gemm dispatches this launch to (mirrors csrc/ns_gemm.hip)"""
    M, N, flags = kw["M"], kw["N"], kw.get("flags", 0)
    if flags & NS_GEMM_TN:
        return "tn"
    if N <= 96 or (M <= 1024 and N <= 4096):
        return "nt32"
    return "nt256" if (N >= 256 and (M >= 2048 or (M >= 128 and N >= 8192)) and ((M + 255) // 256) * ((N + 255) // 256) >= 192) else "nt128"


def _gemm_work(kw):
    """(FLOP, algorithmic HBM bytes) of one ns_gemm launch: every operand and every output once.  A row-mapped A (the conv stem's overlapping
    k = 3 windows over a halo image) counts the image once, not its three views."""
    M, N, K, K2, flags = kw["M"], kw["N"], kw["K"], kw.get("K2", 0), kw.get("flags", 0)
    side = kw.get("side_n", 0) if kw.get("side_B") is not None else 0      # side product: 2 M N side_n more
    flop = 2.0 * M * N * ((kw.get("k_alg") or K) + K2 + side)
    am = kw.get("am")
    if flags & NS_GEMM_TN:      # C32 (M x N) += A^T B over K reduction rows: A is (K, M), B is (K, N)
        by = 2.0 * K * (M + N) + 4.0 * M * N
        return flop, by
    if am is not None and am.seg_rows > 0 and am.ld < K:      # overlapping rows: the (segments x seg_stride) image once
        a_bytes = 2.0 * (M / am.seg_rows) * am.seg_stride
    else:
        a_bytes = 2.0 * M * K
    by = a_bytes + 2.0 * N * K + 2.0 * (M + N) * K2
    for name, w in (("C16", 2), ("G16", 2), ("P16", 2), ("R32", 4), ("H32", 4), ("C32", 4)):
        if kw.get(name) is not None:
            by += float(w) * M * N
    if kw.get("bias") is not None:
        by += 4.0 * N
    if side:
        by += 2.0 * side * N + 4.0 * ((N + 255) // 256) * M * side
    return flop, by


def _gemm_epi(kw) -> str:
    flags = kw.get("flags", 0)
    e = "res" if kw.get("H32") is not None else ("dgelu" if flags & (NS_GEMM_DGELU | NS_GEMM_MUL_P16) else ("gelu" if flags & NS_GEMM_GELU else "plain"))
    if kw.get("side_B") is not None:
        e += "+side"
    if kw.get("K2", 0):
        e += "+k2"
    if kw.get("drop_p", 0.0) > 0.0:
        e += "+drop"
    return e


def gemm(**kw):
    """ns_gemm (keyword arguments = the descriptor's fields, see _fill_gemm_desc).  k_alg: the ALGORITHMIC reduction length where K
    carries padding (the first conv: 3 x ch against 3 x ch_pad); only the bench's FLOP count reads it"""
    d = _fill_gemm_desc(GemmDesc(), **kw)
    if STEP_PROFILE is not None:
        kind = _gemm_kind(kw)
        _work(f"gemm {kind} {_gemm_epi(kw)} K={kw['K']} N={kw['N']}" if kind == "nt256" else f"gemm {kind}", *_gemm_work(kw))
    if GEMM_PROFILE is None:
        _call("ns_gemm", C.byref(d))
        return
    # bench.py roofline leg: HIP events on the launch stream around every GEMM launch
    kind = _gemm_kind(kw)
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record(torch.cuda.current_stream())
    _call("ns_gemm", C.byref(d))
    e1.record(torch.cuda.current_stream())
    fl, by = _gemm_work(kw)
    GEMM_PROFILE.append((kind, fl, e0, e1, by))


def gemm_ln_supported(M: int, N: int, K: int, K2: int = 0, lda: int | None = None) -> bool:
    """the shape test of the library AND ns_gemm_ln's operand-extent test (32-bit buffer offsets: the last row of A, row stride lda, must
    end below 2 GiB -- e.g. fc2 of a very large batch), so that a caller falls back to ns_gemm + ns_layernorm_fwd instead of raising"""
    lda = K if lda is None else lda
    return bool(L.load().ns_gemm_ln_supported(M, N, K, K2)) and 2 * ((M - 1) * lda + K + 64) < 0x7FFF0000


def gemm_ln(*, gamma, beta, x16, ldx, mean=None, rstd=None, eps=1e-5, **kw):
    """ns_gemm_ln: the residual Linear described by **kw (as for gemm: N = 512, R32, H32) + the LayerNorm that reads H32"""
    q = L.GemmLnDesc()
    _fill_gemm_desc(q.g, **kw)
    q.gamma, q.beta, q.eps, q.ldx = ptr(gamma), ptr(beta), eps, ldx
    q.x16, q.mean, q.rstd = ptr(x16), ptr(mean), ptr(rstd)
    fl, by = _gemm_work(kw)
    by += kw["M"] * (2.0 * kw["N"] + 8.0)      # + the LayerNorm's x16 row and its statistics
    _work("gemm rowln (+LayerNorm)", fl, by)
    if GEMM_PROFILE is None:
        _call("ns_gemm_ln", C.byref(q))
        return
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record(torch.cuda.current_stream())
    _call("ns_gemm_ln", C.byref(q))
    e1.record(torch.cuda.current_stream())
    GEMM_PROFILE.append(("rowln", fl, e0, e1, by))


def gemm_side_supported(M: int, N: int, K: int) -> bool:
    return bool(L.load().ns_gemm_side_supported(M, N, K))


def gemm_side_reduce(slabs, tiles, M, alpha, u16, ldu):
    _work("side_reduce", 0.0, M * 32 * (4.0 * tiles + 2.0))
    _call("ns_gemm_side_reduce", ptr(slabs), tiles, M, alpha, ptr(u16), ldu)


def layernorm_fwd(x32, gamma, beta, y16, mean, rstd, rows, d, y32=None, eps=1e-5):
    _work("layernorm_fwd", 0.0, rows * (d * (6.0 + (4.0 if y32 is not None else 0.0)) + 8.0))
    _call("ns_layernorm_fwd", ptr(x32), ptr(gamma), ptr(beta), ptr(y16), ptr(y32), ptr(mean), ptr(rstd),
                                      rows, d, eps)


def layernorm_bwd(dy, dy_is_f32, x32, mean, rstd, gamma, dres, dx32, dx16, rows, d):
    _work("layernorm_bwd", 0.0, rows * (d * ((4.0 if dy_is_f32 else 2.0) + 4.0 + (4.0 if dres is not None else 0.0)
                                              + (4.0 if dx32 is not None else 0.0) + (2.0 if dx16 is not None else 0.0)) + 8.0))
    _call("ns_layernorm_bwd", ptr(dy), int(dy_is_f32), ptr(x32), ptr(mean), ptr(rstd), ptr(gamma), ptr(dres),
                                      ptr(dx32), ptr(dx16), rows, d)


def signal_pack(x32, out16, B, ch, T, Cp):
    _work("signal_pack", 0.0, B * (4.0 * ch * T + 2.0 * (T + 2) * Cp))
    _call("ns_signal_pack", ptr(x32), ptr(out16), B, ch, T, Cp)


def feed_pack(items_dev, B, ch, T, Cp, out16, x32=None):
    """items_dev: device uint8/int64 tensor holding B ns_feed_item records (32 bytes each)"""
    _call("ns_feed_pack", ptr(items_dev), B, ch, T, Cp, ptr(out16), ptr(x32))


def embed_pos(ids, E32, P32, h32, rows, Lseq, d, pos0=0, pos0_dev=None):
    _call("ns_embed_pos", ptr(ids), ptr(E32), ptr(P32), ptr(h32), rows, Lseq, d, pos0, ptr(pos0_dev))


def dgelu_mul(a16, pre16, out16, out_map, rows, cols, pre_is_grad=False):
    _call("ns_dgelu_mul", ptr(a16), ptr(pre16), ptr(out16), C.byref(out_map), rows, cols, int(pre_is_grad))


def colsum(a16, out32, rows, cols, ld, alpha=1.0):
    _call("ns_colsum", ptr(a16), ptr(out32), rows, cols, ld, alpha)


def _attn_desc(Q, K, V, O, B, H, Lq, Lk, ldq, ldk, ldv, ldo, causal, LSE=None, dO=None, dQ=None, dK=None, dV=None,
               Delta=None, lddo=0, lddq=0, lddk=0, lddv=0, workspace=None):
    d = AttnDesc()
    if workspace is not None:       # one-pass backward (ns_attn_bwd_workspace_bytes > 0 for this shape)
        d.workspace, d.workspace_bytes = ptr(workspace), workspace.numel() * workspace.element_size()
    d.Q, d.K, d.V, d.O = ptr(Q), ptr(K), ptr(V), ptr(O)
    d.dO, d.dQ, d.dK, d.dV = ptr(dO), ptr(dQ), ptr(dK), ptr(dV)
    d.LSE, d.Delta = ptr(LSE), ptr(Delta)
    d.B, d.H, d.Lq, d.Lk, d.head_dim = B, H, Lq, Lk, 64
    d.ldq, d.ldk, d.ldv, d.ldo = ldq, ldk, ldv, ldo
    d.lddo, d.lddq, d.lddk, d.lddv = lddo, lddq, lddk, lddv
    d.causal = int(causal)
    return d


def _attn_work(kw, bwd: bool):
    B, H, Lq, Lk = kw["B"], kw["H"], kw["Lq"], kw["Lk"]
    causal = bool(kw.get("causal"))
    fl = 4.0 * B * H * Lq * Lk * 64 * (0.5 if causal else 1.0)
    by = 2.0 * B * H * 64 * (2 * Lq + 2 * Lk) + 4.0 * B * H * Lq         # Q, O, K, V + LSE
    if bwd:
        return 2.5 * fl, 2.0 * by + 4.0 * B * H * Lq                       # + dO, dQ, dK, dV, delta (five products against two)
    return fl, by


def attn_fwd(**kw):
    d = _attn_desc(**kw)
    _work("attn_fwd" + (" causal" if kw.get("causal") else "") + (" (few queries)" if kw["Lq"] <= 64 else ""), *_attn_work(kw, False))
    _call("ns_attn_fwd", C.byref(d))


def attn_bwd_workspace_bytes(B, H, Lq, Lk, causal=False) -> int:
    return int(L.load().ns_attn_bwd_workspace_bytes(B, H, Lq, Lk, int(causal)))


def attn_bwd(**kw):
    d = _attn_desc(**kw)
    _work("attn_bwd" + (" one pass" if kw.get("workspace") is not None and kw["Lq"] > 64 else "") + (" causal" if kw.get("causal") else "")
          + (" (few queries)" if kw["Lq"] <= 64 else ""), *_attn_work(kw, True))
    _call("ns_attn_bwd", C.byref(d))


def cross_entropy(logits16, labels, rows, V, ldv, row_loss, dlogits16, nvalid_dev, loss_scale_dev, loss_dev):
    _work("cross_entropy", 0.0, rows * V * (2.0 + (2.0 if dlogits16 is not None else 0.0)))
    _call("ns_cross_entropy", ptr(logits16), ptr(labels), rows, V, ldv, ptr(row_loss), ptr(dlogits16),
                                      ptr(nvalid_dev), ptr(loss_scale_dev), ptr(loss_dev))


# ---- losses over the vocabulary.  Shapes and types come from the tensors; what the kernels cannot take is refused here with a ValueError.
# (These calls take ~10 us of GPU time at the small end: messages are only formatted when something is refused, attributes read once.)
_DTYPES = {torch.float16: L.NS_F16, torch.bfloat16: L.NS_BF16, torch.float32: L.NS_F32}
_HALF_TYPES = (torch.float16, torch.bfloat16)
_F32_ONLY, _I32_ONLY = (torch.float32,), (torch.int32,)


def _matrix(name, t, rows, cols, dtypes):
    """(rows, columns, row stride in elements) of a 2-D tensor with unit column stride; rows / cols: what they have to be (None: any)"""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError(f"{name}: a 2-D tensor")
    n, m = t.shape
    if (rows is not None and n != rows) or (cols is not None and m != cols):
        raise ValueError(f"{name}: shape {(n, m)}, expected ({'any' if rows is None else rows}, {'any' if cols is None else cols})")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype}, expected one of {tuple(dtypes)}")
    ld, one = t.stride()
    if m > 1 and one != 1:
        raise ValueError(f"{name}: columns must be contiguous (strides {t.stride()})")
    if n <= 1:
        return n, m, m
    if ld < m:
        raise ValueError(f"{name}: rows overlap (strides {t.stride()})")
    return n, m, ld


def _vector(name, t, n, dtype):
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.numel() == n and t.is_contiguous()):
        raise ValueError(f"{name}: a contiguous tensor of {n} {dtype}")
    return t.data_ptr()


def _area(at, rows, cols, ld, size):
    """(first byte, bytes of a row, bytes from row to row, bytes from the first to the last) of a matrix"""
    return at, cols * size, ld * size, ((rows - 1) * ld + cols) * size if rows > 0 and cols > 0 else 0


def _apart(name, area, *others):
    """the matrix `area` shares no byte with the others, given as (what, area).  Columns beside each other in one buffer are apart."""
    a, wa, la, na = area
    for what, (b, wb, lb, nb) in others:
        if na > 0 and nb > 0 and a < b + nb and b < a + na:
            if la == lb and wa + wb <= la and wa <= (b - a) % la <= la - wb:
                continue
            raise ValueError(f"{name} overlaps {what}")


def _one_gpu(*tensors) -> int:
    """ordinal of the GPU that all of them are on; None entries are skipped"""
    dev = None
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d != dev:
                if d < 0:
                    raise ValueError(f"a tensor is on {t.device}, expected a GPU")
                if dev is not None:
                    raise ValueError(f"a tensor is on {t.device}, the others are on cuda:{dev}")
                dev = d
    return dev


def _call_on(dev: int, name, d):
    """launch on the current stream of GPU `dev`, whatever device is current"""
    if dev == torch.cuda.current_device():
        _call(name, C.byref(d))
    else:
        with torch.cuda.device(dev):
            _call(name, C.byref(d))


def _targets(d, rows, labels, row_loss, loss, nvalid, loss_scale, top_vals, top_idx, temperature, alpha):
    """the arguments that both losses share, checked and written into the descriptor"""
    if labels is not None:
        d.labels = _vector("labels", labels, rows, torch.int64)
    d.row_loss = _vector("row_loss", row_loss, rows, torch.float32)
    d.loss_dev = _vector("loss", loss, 1, torch.float32)
    d.nvalid_dev = _vector("nvalid", nvalid, 1, torch.int32)
    if loss_scale is not None:
        d.loss_scale_dev = _vector("loss_scale", loss_scale, 1, torch.float32)
    d.rows, d.temperature, d.alpha = rows, temperature, alpha
    if top_vals is None and top_idx is None:
        if alpha != 0.0:
            raise ValueError(f"alpha {alpha}: soft targets need top_vals and top_idx")
        return
    if top_vals is None or top_idx is None:
        raise ValueError("top_vals and top_idx come together")
    _, k, ld = _matrix("top_vals", top_vals, rows, None, _F32_ONLY)
    _, _, li = _matrix("top_idx", top_idx, rows, k, _I32_ONLY)
    if ld != li:
        raise ValueError(f"top_vals and top_idx: different row strides ({ld}, {li})")
    if not 1 <= k <= 256:
        raise ValueError(f"top_vals: {k} entries a row, 1 to 256 are supported")
    if not 0.05 <= temperature <= 100.0:
        raise ValueError(f"temperature {temperature}: expected 0.05 to 100")
    if not 0.0 <= alpha <= 1.0:
        raise ValueError(f"alpha {alpha}: expected 0 to 1")
    d.k, d.ld_top, d.top_vals, d.top_idx = k, ld, top_vals.data_ptr(), top_idx.data_ptr()


def _head_operand(name, t, rows, cols, dtypes):
    n, m, ld = _matrix(name, t, rows, cols, dtypes)
    if m % 8 or not 8 <= m <= 1 << 16:
        raise ValueError(f"{name}: {m} columns, a multiple of 8 up to 65536 is supported")
    at = t.data_ptr()
    if ld % 8 or ld >= 1 << 21 or at % 16:
        raise ValueError(f"{name}: rows must start on 16 bytes (row stride {ld} elements, below {1 << 21})")
    return n, m, ld, at


def _linear_ce_desc(h, weight, labels, row_loss, loss, nvalid, dh, dweight, loss_scale, top_vals, top_idx, temperature, alpha, accumulate):
    d = L.LinearCeDesc()
    rows, width, d.ldh, d.h = _head_operand("h", h, None, None, _HALF_TYPES)
    dtype = h.dtype
    vocab, _, d.ldw, d.w = _head_operand("weight", weight, None, width, (dtype,))
    if vocab < 1:
        raise ValueError("weight: no rows")
    if rows > 1 << 21:
        raise ValueError(f"h: {rows} rows, up to {1 << 21} are supported")
    if labels is None:
        raise ValueError("labels: a tensor, -100 for a row that does not count")
    d.vocab, d.d, d.dtype = vocab, width, _DTYPES[dtype]
    _targets(d, rows, labels, row_loss, loss, nvalid, loss_scale, top_vals, top_idx, temperature, alpha)
    if dh is not None or dweight is not None:
        taken = (("h", _area(d.h or 0, rows, width, d.ldh, 2)), ("weight", _area(d.w, vocab, width, d.ldw, 2)))
        if dh is not None:
            _, _, d.lddh, at = _head_operand("dh", dh, rows, width, (dtype,))
            area = _area(at, rows, width, d.lddh, 2)
            _apart("dh", area, *taken)
            taken += (("dh", area),)
            d.dh = at if rows else 0              # (no rows: nothing to write)
        if dweight is not None:
            _, _, d.lddw, d.dw = _head_operand("dweight", dweight, vocab, width, (dtype, torch.float32))
            d.dw_f32 = int(dweight.dtype == torch.float32)
            _apart("dweight", _area(d.dw, vocab, width, d.lddw, 4 if d.dw_f32 else 2), *taken)
    if accumulate:
        if dweight is None or not d.dw_f32:
            raise ValueError("accumulate: adds to a float32 dweight only")
        d.dw_add = 1
    return d


def linear_ce_workspace_bytes(h, weight, labels, *, row_loss, loss, nvalid, dh=None, dweight=None, loss_scale=None, top_vals=None, top_idx=None,
                              temperature=1.0, alpha=0.0, accumulate=False) -> int:
    """workspace of linear_cross_entropy for these arguments"""
    return int(L.load().ns_linear_ce_workspace_bytes(C.byref(_linear_ce_desc(h, weight, labels, row_loss, loss, nvalid, dh, dweight, loss_scale, top_vals,
                                                                             top_idx, float(temperature), float(alpha), accumulate))))


def linear_cross_entropy(h, weight, labels, *, row_loss, loss, nvalid, dh=None, dweight=None, loss_scale=None, top_vals=None, top_idx=None,
                         temperature=1.0, alpha=0.0, accumulate=False, workspace=None):
    """The LM head and its loss without the logits (ns_linear_cross_entropy): z = h weight^T only ever exists as tiles.

    h (rows, d), weight (vocab, d): float16 or bfloat16; labels (rows) int64, outside [0, vocab) = the row is ignored.  Written: row_loss (rows) and
    loss (1) float32, nvalid (1) int32, dh like h, dweight like weight or float32 (`accumulate`: added to a float32 one): gradients of
    loss_scale x loss.  top_vals / top_idx (rows, k): a teacher's top logits and tokens (topk_logits), mixed in by `alpha` at `temperature`:
    loss = mean of (1 - alpha) CE + alpha T^2 KL.
    workspace: a uint8 tensor of linear_ce_workspace_bytes(...) (default: allocated for the call, on the current stream).  A captured graph keeps
    the default's memory in its own pool; two graphs that may run at the same time must not share an explicit one."""
    d = _linear_ce_desc(h, weight, labels, row_loss, loss, nvalid, dh, dweight, loss_scale, top_vals, top_idx, float(temperature), float(alpha), accumulate)
    dev = _one_gpu(h, weight, labels, row_loss, loss, nvalid, dh, dweight, loss_scale, top_vals, top_idx, workspace)
    need = L.load().ns_linear_ce_workspace_bytes(C.byref(d))
    if workspace is None:
        if getattr(_tls, "rec", None) is not None:
            raise ValueError("a recorded launch list replays raw addresses: pass a workspace that outlives it")
        workspace = torch.empty(need, device=h.device, dtype=torch.uint8)
    elif not (workspace.dtype == torch.uint8 and workspace.is_contiguous() and workspace.numel() >= need and workspace.data_ptr() % 16 == 0):
        raise ValueError(f"workspace: {need} contiguous bytes of uint8 that start on 16 bytes")
    d.workspace, d.workspace_bytes = workspace.data_ptr(), workspace.numel()
    if STEP_PROFILE is not None:
        n, v, w = d.rows, d.vocab, d.d
        _work("linear_cross_entropy", 2.0 * n * v * w * (1 + (dh is not None) + (dweight is not None)),
              2.0 * (n * w + v * w) + (2.0 * n * w if dh is not None else 0.0) + ((4.0 if d.dw_f32 else 2.0) * v * w if dweight is not None else 0.0))
    _call_on(dev, "ns_linear_cross_entropy", d)


def distill_topk(logits, labels, top_vals, top_idx, *, row_loss, loss, nvalid, temperature=1.0, alpha=1.0, dlogits=None, loss_scale=None):
    """Distillation from a teacher's top logits over logits that exist (ns_distill_topk): loss = mean of (1 - alpha) CE + alpha T^2 KL and, with
    dlogits, the gradient of loss_scale x loss with respect to the logits (like logits; may be the logits themselves).

    logits (rows, vocab) float16, bfloat16 or float32, rows at any stride (a [:, :vocab] view of a padded buffer: the padding is not
    touched); labels as in linear_cross_entropy, or None with alpha = 1: every row counts; top_vals / top_idx (rows, k) float32 / int32, k <= 256."""
    d = L.DistillDesc()
    rows, vocab, d.ldz = _matrix("logits", logits, None, None, _DTYPES)
    if vocab < 1:
        raise ValueError("logits: no columns")
    if labels is None and alpha != 1.0:
        raise ValueError(f"alpha {alpha}: the hard term needs labels")
    if top_vals is None or not alpha > 0.0:
        raise ValueError("top_vals, top_idx and alpha > 0: without them this is cross_entropy")
    _targets(d, rows, labels, row_loss, loss, nvalid, loss_scale, top_vals, top_idx, float(temperature), float(alpha))
    d.logits, d.vocab, d.dtype = logits.data_ptr(), vocab, _DTYPES[logits.dtype]
    if dlogits is not None:
        _, _, d.lddz = _matrix("dlogits", dlogits, rows, vocab, (logits.dtype,))
        d.dlogits = dlogits.data_ptr()
        if d.dlogits != d.logits or d.lddz != d.ldz:
            size = logits.element_size()
            _apart("dlogits", _area(d.dlogits or 0, rows, vocab, d.lddz, size), ("logits", _area(d.logits or 0, rows, vocab, d.ldz, size)))
    dev = _one_gpu(logits, labels, top_vals, top_idx, row_loss, loss, nvalid, dlogits, loss_scale)
    if STEP_PROFILE is not None:
        _work("distill_topk", 0.0, logits.element_size() * rows * vocab * (2.0 if dlogits is not None else 1.0) + 8.0 * rows * d.k)
    _call_on(dev, "ns_distill_topk", d)


def topk_logits(logits, k, *, vals, idx, lse=None):
    """A teacher's lists (ns_topk_logits): the k (<= 256) largest logits of each row, largest first, equal ones by the lowest token.

    logits (rows, vocab) float16, bfloat16 or float32, rows at any stride; vals (rows, k) float32, idx (rows, k) int32, lse (rows) float32: the
    row's log-sum-exp."""
    d = L.TopkDesc()
    rows, vocab, d.ldz = _matrix("logits", logits, None, None, _DTYPES)
    if not (isinstance(k, int) and 1 <= k <= 256 and k <= vocab):
        raise ValueError(f"k {k}: expected 1 to {min(256, vocab)}")
    _, _, d.ldo = _matrix("vals", vals, rows, k, _F32_ONLY)
    _, _, ldi = _matrix("idx", idx, rows, k, _I32_ONLY)
    if ldi != d.ldo:
        raise ValueError(f"vals and idx: different row strides ({d.ldo}, {ldi})")
    if lse is not None:
        d.lse = _vector("lse", lse, rows, torch.float32)
    d.logits, d.vals, d.idx = logits.data_ptr(), vals.data_ptr(), idx.data_ptr()
    z = ("logits", _area(d.logits or 0, rows, vocab, d.ldz, logits.element_size()))
    _apart("vals", _area(d.vals or 0, rows, k, d.ldo, 4), z)
    _apart("idx", _area(d.idx or 0, rows, k, d.ldo, 4), z)
    dev = _one_gpu(logits, vals, idx, lse)
    d.rows, d.vocab, d.k, d.dtype = rows, vocab, k, _DTYPES[logits.dtype]
    if STEP_PROFILE is not None:
        _work("topk_logits", 0.0, logits.element_size() * rows * vocab + 8.0 * rows * k)
    _call_on(dev, "ns_topk_logits", d)


def argmax_rows(logits16, rows, V, ldv, out):
    _call("ns_argmax_rows", ptr(logits16), rows, V, ldv, ptr(out))


def grad_norm(g32, n, workspace, norm2_dev, found_inf_dev):
    _work("grad_norm", 0.0, 4.0 * n)
    _call("ns_grad_norm", ptr(g32), n, ptr(workspace), ptr(norm2_dev), ptr(found_inf_dev))


def adamw_step(p, g, m, v, n, cfg: AdamWCfg, step_dev, norm2_dev, found_inf_dev, loss_scale_dev, growth_tracker_dev):
    _work("adamw_step", 0.0, 28.0 * n)
    _call("ns_adamw_step", ptr(p), ptr(g), ptr(m), ptr(v), n, C.byref(cfg), ptr(step_dev), ptr(norm2_dev),
                                   ptr(found_inf_dev), ptr(loss_scale_dev), ptr(growth_tracker_dev))


def zero_(*tensors):
    """clear up to 8 tensors per launch with ns_zero_spans (a kernel, never a memset node: see the header)"""
    ts = [t for t in tensors if t is not None and t.numel() > 0]
    for i in range(0, len(ts), 8):
        chunk = ts[i:i + 8]
        arr = (L.Span * len(chunk))()
        for j, t in enumerate(chunk):
            assert t.is_contiguous()
            arr[j] = L.Span(t.data_ptr(), t.numel() * t.element_size())
        _work("zero_spans", 0.0, float(sum(t.numel() * t.element_size() for t in chunk)))
        _call("ns_zero_spans", arr, len(chunk))


def zeros(*shape, device, dtype):
    """torch.zeros without torch's fill kernel"""
    t = torch.empty(*shape, device=device, dtype=dtype)
    zero_(t)
    return t


def add_i32(counter_dev, v=1, n=1):
    """v added to n consecutive int32 device counters in one launch"""
    _call("ns_add_i32", ptr(counter_dev), int(n), int(v))


def make_cast_jobs(jobs, device) -> tuple[torch.Tensor, int]:
    """jobs: list of (src_ptr, dst_ptr, rows, cols, ld_src, ld_dst, scale, transpose) -> device table."""
    arr = (CastJob * len(jobs))()
    for i, job in enumerate(jobs):
        s, dptr, r, c, lds, ldd, sc, tr = job[:8]
        arr[i] = CastJob(s, dptr, r, c, lds, ldd, sc, int(tr), job[8] if len(job) > 8 else 0)
    raw = bytes(arr)
    t = torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(device)
    return t, len(jobs)


def cast_jobs(table: torch.Tensor, njobs: int):
    _call("ns_cast_jobs", ptr(table), njobs)


# ----------------------------------------------------------------------------- decode loop
def attn_decode(*, Q, K, V, O, groups, nq, H, Lk, Lk_max, ldq, ldk, ldv, ldo, anc=None, anc_ld=0, kv_group_stride=0,
                kv_pos_stride=0, kv_len_dev=None, Knew=None, Vnew=None, ldnew=0, slot0=0):
    d = L.AttnDecodeDesc()
    d.Q, d.K, d.V, d.O = ptr(Q), ptr(K), ptr(V), ptr(O)
    d.anc, d.kv_len_dev = ptr(anc), ptr(kv_len_dev)
    d.groups, d.nq, d.H, d.Lk, d.Lk_max, d.head_dim = groups, nq, H, Lk, Lk_max, 64
    d.ldq, d.ldk, d.ldv, d.ldo, d.anc_ld = ldq, ldk, ldv, ldo, anc_ld
    d.kv_group_stride, d.kv_pos_stride = kv_group_stride, kv_pos_stride
    d.Knew, d.Vnew, d.ldnew, d.slot0 = ptr(Knew), ptr(Vnew), ldnew, slot0
    _call("ns_attn_decode", C.byref(d))


def attn_fewq(*, Q, K, Vt, O, groups, nq, H, Lk, ldq, ldk, ldvt, ldo):
    d = L.AttnFewqDesc()
    d.Q, d.K, d.Vt, d.O = ptr(Q), ptr(K), ptr(Vt), ptr(O)
    d.groups, d.nq, d.H, d.Lk, d.ldq, d.ldk, d.ldvt, d.ldo = groups, nq, H, Lk, ldq, ldk, ldvt, ldo
    _call("ns_attn_fewq", C.byref(d))


def vt_pack(v16, ldv, vt16, groups, H, Lk, ldvt):
    _call("ns_vt_pack", ptr(v16), ldv, ptr(vt16), groups, H, Lk, ldvt)


def logits_process(*, logits16, scores32, ids, rows, V, ldv, ids_ld, cur_len, begin_index, log_softmax, beam_scores=None,
                   repetition_penalty=1.0, no_repeat_ngram=0, suppress=None, n_suppress=0, begin_suppress=None,
                   n_begin_suppress=0, cur_len_dev=None, bias1=None, seq_tok=None, seq_off=None, seq_bias=None, n_seq=0,
                   forced=None, n_forced=0):
    d = L.LogitsProcDesc()
    d.forced, d.n_forced = ptr(forced), n_forced
    d.logits16, d.scores32, d.ids, d.beam_scores = ptr(logits16), ptr(scores32), ptr(ids), ptr(beam_scores)
    d.suppress, d.begin_suppress, d.cur_len_dev = ptr(suppress), ptr(begin_suppress), ptr(cur_len_dev)
    d.rows, d.V, d.ldv, d.ids_ld, d.cur_len, d.begin_index = rows, V, ldv, ids_ld, cur_len, begin_index
    d.n_suppress, d.n_begin_suppress, d.no_repeat_ngram, d.log_softmax = n_suppress, n_begin_suppress, no_repeat_ngram, int(log_softmax)
    d.repetition_penalty = repetition_penalty
    d.bias1, d.seq_tok, d.seq_off, d.seq_bias, d.n_seq = ptr(bias1), ptr(seq_tok), ptr(seq_off), ptr(seq_bias), n_seq
    _call("ns_logits_process", C.byref(d))


SELECT_MAX_LDV = 26 * 256 * 8


def logits_select(*, logits16, ids, rows, V, ldv, ids_ld, cur_len, begin_index, log_softmax, k, group_rows, cand_vals,
                  cand_idx, beam_scores=None, repetition_penalty=1.0, no_repeat_ngram=0, suppress=None, n_suppress=0,
                  begin_suppress=None, n_begin_suppress=0, cur_len_dev=None, scores32=None, forced=None, n_forced=0,
                  bias1=None, seq_tok=None, seq_off=None, seq_bias=None, n_seq=0):
    d = L.LogitsProcDesc()
    d.forced, d.n_forced = ptr(forced), n_forced
    d.bias1, d.seq_tok, d.seq_off, d.seq_bias, d.n_seq = ptr(bias1), ptr(seq_tok), ptr(seq_off), ptr(seq_bias), n_seq
    d.logits16, d.scores32, d.ids, d.beam_scores = ptr(logits16), None, ptr(ids), ptr(beam_scores)
    d.suppress, d.begin_suppress, d.cur_len_dev = ptr(suppress), ptr(begin_suppress), ptr(cur_len_dev)
    d.rows, d.V, d.ldv, d.ids_ld, d.cur_len, d.begin_index = rows, V, ldv, ids_ld, cur_len, begin_index
    d.n_suppress, d.n_begin_suppress, d.no_repeat_ngram, d.log_softmax = n_suppress, n_begin_suppress, no_repeat_ngram, int(log_softmax)
    d.repetition_penalty = repetition_penalty
    _call("ns_logits_select", C.byref(d), k, group_rows, ptr(cand_vals), ptr(cand_idx))


def topk_merge(cand_vals, cand_idx, groups, ncand, k, vals, idx):
    _call("ns_topk_merge", ptr(cand_vals), ptr(cand_idx), groups, ncand, k, ptr(vals), ptr(idx))


_topk_ws = {}


def topk_groups(x32, groups, n, k, vals, idx):
    key = (x32.device, groups, n, k)
    ws = _topk_ws.get(key)
    if ws is None:
        ws = torch.empty(L.load().ns_topk_workspace_bytes(groups, n, k), device=x32.device, dtype=torch.uint8)
        _topk_ws[key] = ws
    _call("ns_topk_groups", ptr(x32), groups, n, k, ptr(vals), ptr(idx), ptr(ws))


def beam_update(**kw):
    d = L.BeamDesc()
    for k, v in kw.items():
        setattr(d, k, ptr(v) if isinstance(v, (torch.Tensor, tuple)) or v is None else v)
    _call("ns_beam_update", C.byref(d))


def anc_update(anc_in, anc_out, parent, rows, ld, cur, cur_dev=None):
    _call("ns_anc_update", ptr(anc_in), ptr(anc_out), ptr(parent), rows, ld, cur, ptr(cur_dev))


def greedy_update(scores, rows, V, seqs, ld, cur, eos, pad, done, any_open, next_tok, cur_dev=None, best_idx=None):
    _call("ns_greedy_update", ptr(scores), rows, V, ptr(seqs), ld, cur, ptr(cur_dev), eos, pad, ptr(done), ptr(any_open),
                                      ptr(next_tok), ptr(best_idx))


# ----------------------------------------------------------------------------- AdaLoRA
def adalora_fold_grads(dBf, B, E, dB, dE, N, r, s):
    _call("ns_adalora_fold_grads", ptr(dBf), ptr(B), ptr(E), ptr(dB), ptr(dE), N, r, s)


def make_fold_jobs(jobs, device):
    """jobs: list of (dBf_ptr, B_ptr, E_ptr, dB_ptr, dE_ptr, N, r, s)"""
    arr = (L.AdaloraFoldJob * len(jobs))()
    for i, j in enumerate(jobs):
        arr[i] = L.AdaloraFoldJob(*j)
    return torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).to(device), len(jobs)


def adalora_fold_jobs(table, njobs):
    _call("ns_adalora_fold_jobs", ptr(table), njobs)


def make_orth_jobs(jobs, device):
    """jobs: list of (P_ptr, G_ptr, r, len, ld, is_b)"""
    arr = (L.OrthJob * len(jobs))()
    for i, j in enumerate(jobs):
        arr[i] = L.OrthJob(*j)
    return torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8).to(device), len(jobs)


_orth_ws = {}
_retired_ws = []   # outgrown workspaces stay allocated: graphs captured while they were current replay with their address


def orth_reg(table, njobs, weight_over_num, loss_scale_dev, reg_out_dev):
    need = L.load().ns_orth_reg_workspace_bytes(njobs)
    ws = _orth_ws.get(reg_out_dev.device)
    if ws is None or ws.numel() < need:
        if ws is not None:
            _retired_ws.append(ws)      # a captured training step (hipGraph) may still hold its address
        ws = torch.empty(need, device=reg_out_dev.device, dtype=torch.uint8)
        _orth_ws[reg_out_dev.device] = ws
    _call("ns_orth_reg", ptr(table), njobs, weight_over_num, ptr(loss_scale_dev), ptr(reg_out_dev), ptr(ws), ws.numel())


# ----------------------------------------------------------------------------- LoRA backward (du + dB in one pass over dy)
def lora_bwd_supported(N: int, r: int, G: int) -> bool:
    return bool(L.load().ns_lora_bwd_supported(N, r, G))


_lora_ws = {}


def lora_bwd_dudb(*, dy, ldy, u, ldu, du, lddu, sBT, dB, lddb, M, N, r, alpha_du, alpha_db, splits=0, slabs=True):
    """sBT / dB / alpha_db: one entry per column group of dy (q | k | v: three, else one).  slabs: dB partials through a
    workspace + reduce launch (one cached workspace per device, sized for the largest request) instead of fp32 atomics"""
    d = L.LoraBwdDesc()
    dev = (du[0] if isinstance(du, tuple) else du).device      # (tensor, element offset) pairs address a column group of a stacked buffer
    if slabs:
        need = L.load().ns_lora_bwd_workspace_bytes(M, N, len(sBT), splits)
        ws = _lora_ws.get(dev)
        if ws is None or ws.numel() < need:
            if ws is not None:
                _retired_ws.append(ws)
            ws = torch.empty(need, device=dev, dtype=torch.uint8)
            _lora_ws[dev] = ws
        d.workspace, d.workspace_bytes = ptr(ws), ws.numel()
    d.dy, d.u, d.du = ptr(dy), ptr(u), ptr(du)
    G = len(sBT)
    for g in range(G):
        d.sBT[g], d.dB[g], d.alpha_db[g] = ptr(sBT[g]), ptr(dB[g]), alpha_db[g]
    d.M, d.N, d.r, d.G = M, N, r, G
    d.ldy, d.ldu, d.lddu, d.lddb = ldy, ldu, lddu, lddb
    d.alpha_du, d.splits = alpha_du, splits
    _work("lora_bwd_dudb (+reduce)", 2.0 * M * G * N * r * 2, 2.0 * M * G * N + 2.0 * M * G * r * 2 + 2.0 * G * N * r + 4.0 * G * N * r)
    _call("ns_lora_bwd_dudb", C.byref(d))
