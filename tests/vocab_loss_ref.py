"""64-bit statement of the vocabulary losses and of how far the kernels may be from it, for the tests of linear_cross_entropy / distill_topk.

Tolerances are bounds, term by term, on what the kernels round (u = 2^-24 for fp32, U = half a step of the 16-bit type):
  logits      a dot product of d products in fp32, any order: |dz| <= (d + 4) u (|h| |W|^T)
  exp         argument a = (z - max) c: rounded twice (2 u |a|), the instruction itself within 1 ulp (2 u); a term e^a with |a| large counts
              little (|a| e^a <= 0.37), so a sum of such terms and each p = e^a / sum is within 8 u of that rounding where p matters; n terms in
              16-term runs, lane and tile trees and <= 32 merges: <= 64 u more.  Together: E = 2 max|dz| c + (96 + 2 |a|) u
  a cell      dz_ij = w1 p + w2 q - w1 [j = label] - w2 sum t: E on the p and q terms, (k + 12) u on t, and two roundings to the cell's type (the
              exponential relative to its strip, then dz; of two softmaxes the first one's exponential may be the T-th power of a rounded one, T <= 2: three)
  a product   of n cells: the cells' errors times |operand|, n u of the sum of absolute values, one rounding at the end"""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def targets(vocab, top_vals, top_idx, temp):
    """dense (rows, vocab) soft targets, which rows have any, and the lists' probabilities"""
    there = (top_idx >= 0) & (top_idx < vocab)
    t = torch.where(there, top_vals.double() / temp, float("-inf"))
    m = t.amax(1, keepdim=True)
    some = torch.isfinite(m).squeeze(1)
    e = torch.exp(torch.where(some.unsqueeze(1), t - m, torch.full_like(t, float("-inf"))))
    p = torch.where(some.unsqueeze(1), e / e.sum(1, keepdim=True).clamp(min=1e-300), torch.zeros_like(e))
    dense = torch.zeros(top_vals.shape[0], vocab, dtype=torch.float64, device=top_vals.device)
    dense.scatter_add_(1, torch.where(there, top_idx, 0).long(), torch.where(there, p, torch.zeros_like(p)))
    logp = torch.where(p > 0, torch.log(p.clamp(min=1e-300)), torch.zeros_like(p))
    return dense, some, p, logp, there


def losses(z, dz_err, labels, temp=1.0, alpha=0.0, top_vals=None, top_idx=None):
    """z (rows, vocab) float64 and a bound on each row's logit error -> dict of row_loss, loss, cell (d sum(row_loss) / dz) and their tolerances"""
    rows, v = z.shape
    k = 0 if top_vals is None else top_vals.shape[1]
    valid = torch.ones(rows, dtype=torch.bool, device=z.device) if labels is None else (labels >= 0) & (labels < v)
    lab = torch.zeros(rows, dtype=torch.int64, device=z.device) if labels is None else torch.where(valid, labels, 0)
    row = torch.zeros(rows, dtype=torch.float64, device=z.device)
    tol = torch.zeros_like(row)
    cell = torch.zeros_like(z)
    cell_err = torch.zeros_like(z)
    prob = torch.zeros_like(z)                  # the dense part of a cell: what is rounded before a label's or a list's part comes off
    mag = z.abs().amax(1).clamp(min=1.0)
    # (every term is unchanged when a row's logits move together: with the maximum taken out, lse - z keeps its digits also where |z| is 1e38)
    top = z.amax(1, keepdim=True)
    z = z - torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    dz_err = dz_err.expand(rows) if dz_err.dim() == 0 else dz_err
    if alpha < 1.0:
        w1 = 1.0 - alpha
        lse = torch.logsumexp(z, 1)
        p = torch.exp(z - lse.unsqueeze(1))
        row += w1 * (lse - z.gather(1, lab.unsqueeze(1)).squeeze(1))
        tol += w1 * (2 * dz_err + (160 + 8 * mag) * U32)
        one = torch.nn.functional.one_hot(lab, v).double()
        cell += w1 * (p - one)
        prob += w1 * p
        a = (z - z.amax(1, keepdim=True)).abs()
        cell_err += w1 * (p * (2 * dz_err.unsqueeze(1) + (96 + 4 * a + 4 * mag.unsqueeze(1)) * U32) + 4 * U32 * one)
    if k and alpha > 0.0:
        dense, some, tp, logp, there = targets(v, top_vals, top_idx, temp)
        zt = z / temp
        lse = torch.logsumexp(zt, 1)
        q = torch.exp(zt - lse.unsqueeze(1))
        logq = zt.gather(1, torch.where(there, top_idx, 0).long()) - lse.unsqueeze(1)
        kl = torch.where(tp > 0, tp * (logp - logq), torch.zeros_like(tp)).sum(1)
        row += torch.where(some, alpha * temp * temp * kl, torch.zeros_like(kl))
        big = torch.where(tp > 0, (logp.abs() + logq.abs()) * tp, torch.zeros_like(tp)).sum(1)
        tmag = torch.where(there & torch.isfinite(top_vals), top_vals.double().abs() / temp, torch.zeros_like(tp)).amax(1).clamp(min=1.0)
        rel = (k + 24 + 6 * tmag) * U32
        tol += alpha * temp * temp * (2 * dz_err / temp + (160 + 8 * mag / temp) * U32 + rel * (1 + big))
        w2 = alpha * temp
        a = (zt - zt.amax(1, keepdim=True)).abs()
        on = some.double().unsqueeze(1)
        cell += w2 * on * (q - dense)
        prob += w2 * on * q
        cell_err += w2 * on * (q * (2 * dz_err.unsqueeze(1) / temp + (96 + 4 * a + 4 * mag.unsqueeze(1)) * U32) + dense * rel.unsqueeze(1))
    off = ~valid
    row[off] = 0
    tol[off] = 0
    cell[off] = 0
    cell_err[off] = 0
    prob[off] = 0
    n = max(int(valid.sum()), 1)
    return dict(row_loss=row, row_tol=tol + 4 * U32 * row.abs(), loss=row.sum() / n, loss_tol=(tol.sum() + (rows + 4) * U32 * row.abs().sum()) / n, cell=cell,
                cell_err=cell_err, prob=prob, n=n, nvalid=int(valid.sum()))


def linear(h, w, labels, scale=1.0, dw_dtype=None, temp=1.0, alpha=0.0, top_vals=None, top_idx=None, parts=1, floor=3 * 2.0 ** -40):
    """linear_cross_entropy in 64 bits: losses' dict + dh, dw and their tolerances.  Rows without a label are taken out first.  parts = 2: the cells are
    sums of two numbers of their type (the first off by U of the cell, the second by U of that; formed from fp32, so 2 u of the terms as well).  floor: what fp16's
    smallest step leaves of a cell: half of it, twice, at a factor of at least 2^15 / 2^(w1 + w2).  2^-29 where exponentials are kept relative to the label's: half a
    step (2^-25) times the row's factor, at most p 2 / 2^6, and 2^-39 of a second rounding in a row whose reference changes."""
    rows, d = h.shape
    v = w.shape[0]
    U = half_step(h.dtype)
    valid = (labels >= 0) & (labels < v)
    hd = torch.where(valid.unsqueeze(1), h, torch.zeros_like(h)).double()
    wd = w.double()
    z = hd @ wd.t()
    dz_err = ((d + 4) * U32 * (hd.abs() @ wd.abs().t())).amax(1) if rows else torch.zeros(0, dtype=torch.float64, device=h.device)
    r = losses(z, dz_err, labels, temp, alpha, top_vals, top_idx)
    g = scale / r["n"]
    # (the cells of labels and lists are formed in fp32 from their own logits: their dense part is not rounded by itself)
    prob = r["prob"].clone()
    prob.scatter_(1, torch.where(valid, labels, 0).unsqueeze(1), 0.0)
    if top_idx is not None:
        prob.scatter_(1, torch.where((top_idx >= 0) & (top_idx < v), top_idx, 0).long(), 0.0)
        prob[:, 0] = r["prob"][:, 0]
    tiny = floor if h.dtype == torch.float16 else 0.0
    tiny *= max(1.0, 2.0 * ((1 - alpha) + alpha * temp))
    each = U * (3 + 3 * U) if parts == 1 else U * U + 2 * U32
    cell_tol = r["cell_err"] + each * (r["cell"].abs() + prob + r["cell_err"]) + tiny * valid.double().unsqueeze(1)
    for name, out, err, mass, n, dt in (("dh", r["cell"] @ wd, cell_tol @ wd.abs(), r["cell"].abs() @ wd.abs(), v, h.dtype),
                                        ("dw", r["cell"].t() @ hd, cell_tol.t() @ hd.abs(), r["cell"].abs().t() @ hd.abs(), rows, dw_dtype or w.dtype)):
        out, err = out * g, (err + (n + 8) * U32 * mass) * g
        small = 2.0 ** -25 if dt == torch.float16 else 2.0 ** -126
        r[name] = out
        r[name + "_tol"] = err + (half_step(dt) if dt != torch.float32 else U32) * (out.abs() + err) + 4 * U32 * out.abs() + small
    return r
