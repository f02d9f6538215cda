"""64-bit statement of the vocabulary losses' gradients for rows that are almost certain, and bounds on it that are relative to what such a row has left.

With p_j = softmax(z)_j, q_j = softmax(z / T)_j and t_j the teacher's probabilities, a cell of dz is  w1 (p_j - [j = label]) + w2 (q_j - t_j).  At one token of the row
p, q and t may all be close to 1; there 1 - p, 1 - q and 1 - t are sums over the other tokens (here and in the kernels), so that their bounds are relative to themselves:
  1 - p        every term within E = 2 max|dz| c + (96 + 4 |a| + 4 |z|) u  (see vocab_loss_ref), so is their sum;  1 - t within (k + 24 + 6 |t logits|) u
  a 16-bit cell  two roundings (three for two softmaxes): U (3 + 3 U) of it; the row's largest ones once, in fp32
  fp16         half of its smallest step, 2^-25, times the factor of the row.  Cells kept relative to the label's (labels alone, dh alone): a strip of 64 tokens is kept so
               only if its largest value is at least 2^-8, so the step is at most 2^-17 of the strip's largest cell; what is brought to the row's reference later loses
               2^-25 of it, where the row's other tokens hold V 2^-14 at least: 2^-11 (1 - p) / V a cell, or 2^-39 of the row's largest.  Elsewhere cells carry a
               factor of at least 2^15 / 2^(w1 + w2), and are rounded twice: 3 2^-40 max(1, 2 (w1 + w2))."""
import torch

from tests.vocab_loss_ref import U32, half_step


def softmax_and_rest(z):
    """softmax of each row and 1 - softmax, both with their own digits"""
    e = torch.exp(z - z.amax(1, keepdim=True))
    total = e.sum(1, keepdim=True)
    p = e / total
    top = z.argmax(1, keepdim=True)
    rest = 1.0 - p
    others = e.scatter(1, top, 0.0).sum(1, keepdim=True) / total
    return p, rest.scatter(1, top, others)


def teacher(v, tv, ti, temp):
    """(t, 1 - t) as dense rows, each with its own digits, and which rows have a list"""
    there = (ti >= 0) & (ti < v)
    x = torch.where(there, tv.double() / temp, float("-inf"))
    some = torch.isfinite(x.amax(1))
    e = torch.where(there, torch.exp(x - torch.where(some, x.amax(1), torch.zeros_like(x[:, 0])).unsqueeze(1)), torch.zeros_like(x))
    e = torch.where(some.unsqueeze(1), e, torch.zeros_like(e))
    total = e.sum(1, keepdim=True).clamp(min=1e-300)
    t = torch.zeros(tv.shape[0], v, dtype=torch.float64, device=tv.device)
    t.scatter_add_(1, torch.where(there, ti, 0).long(), e)
    top = t.argmax(1, keepdim=True)
    others = t.scatter(1, top, 0.0).sum(1, keepdim=True) / total
    t = t / total
    rest = (1.0 - t).scatter(1, top, others)
    return t, rest, some


def cells(z, dz_err, labels, temp=1.0, alpha=0.0, tv=None, ti=None):
    """cells of dz (d sum(row_loss) / dz), bounds on what fp32 loses of them, the sizes that 16-bit roundings go by, and 1 - p; every row has a label"""
    n, v = z.shape
    lab = torch.nn.functional.one_hot(labels, v).bool()
    mag = z.abs().amax(1, keepdim=True).clamp(min=1.0)
    cell, err, size = torch.zeros_like(z), torch.zeros_like(z), torch.zeros_like(z)
    left = None
    if alpha < 1.0:
        p, rest = softmax_and_rest(z)
        left = rest.gather(1, labels.unsqueeze(1)).squeeze(1)
        E = 2 * dz_err.unsqueeze(1) + (96 + 4 * (z - z.amax(1, keepdim=True)).abs() + 4 * mag) * U32
        part = torch.where(lab, -rest, p)
        cell += (1 - alpha) * part
        err += (1 - alpha) * part.abs() * (E + 8 * U32)
        size += (1 - alpha) * part.abs()
    if tv is not None and alpha > 0.0:
        k = tv.shape[1]
        w2 = alpha * temp
        q, qrest = softmax_and_rest(z / temp)
        t, trest, some = teacher(v, tv, ti, temp)
        on = some.double().unsqueeze(1)
        E = 2 * dz_err.unsqueeze(1) / temp + (96 + 4 * ((z - z.amax(1, keepdim=True)) / temp).abs() + 4 * mag / temp) * U32
        rel = (k + 24 + 6 * (torch.where((ti >= 0) & (ti < v) & torch.isfinite(tv), tv.double().abs(), torch.zeros_like(tv.double())).amax(1, keepdim=True) / temp).clamp(min=1.0)) * U32
        near = q > 0.5                          # one token of a row at most: its difference is taken between what the others hold
        cell += on * w2 * torch.where(near, trest - qrest, q - t)
        err += on * w2 * (torch.where(near, qrest, q) * (E + 8 * U32) + torch.where(near, trest, t) * rel)
        size += on * w2 * torch.where(near, qrest, q)
        if left is None:
            left = torch.where(some, qrest.amin(1), torch.zeros_like(qrest[:, 0]))
    return cell, err, size, left


def linear(h, w, labels, scale=1.0, temp=1.0, alpha=0.0, tv=None, ti=None, to_label=False, dw_dtype=None, parts=1):
    """(dh, its bound, dw, its bound, 1 - p, a row's part of dh's bound that fp16's smallest step makes) of linear_cross_entropy.  to_label: fp16 cells are kept relative to the
    label's"""
    n, d = h.shape
    v = w.shape[0]
    U = half_step(h.dtype)
    hd, wd = h.double(), w.double()
    z = hd @ wd.t()
    dz_err = ((d + 4) * U32 * (hd.abs() @ wd.abs().t())).amax(1)
    cell, err, size, left = cells(z, dz_err, labels, temp, alpha, tv, ti)
    g = scale / n
    tol = err + (U * (3 + 3 * U) if parts == 1 else U * U + 2 * U32) * (cell.abs() + size + err)
    floor = torch.zeros_like(cell)
    if h.dtype == torch.float16:
        if to_label:
            p = torch.softmax(z, 1).scatter(1, labels.unsqueeze(1), 0.0)
            strips = torch.nn.functional.pad(p, (0, -v % 64)).view(n, -1, 64).amax(2)
            floor = 2.0 ** -17 * strips.repeat_interleave(64, 1)[:, :v] + 2.0 ** -11 * left.unsqueeze(1) / v + 2.0 ** -38 * p.amax(1, keepdim=True)
        else:
            floor = floor + 3 * 2.0 ** -40 * max(1.0, 2.0 * ((1 - alpha) + alpha * temp))
    tol = tol + floor
    out = []
    for x, e, mass, m, dt in ((cell @ wd, tol @ wd.abs(), cell.abs() @ wd.abs(), v, h.dtype), (cell.t() @ hd, tol.t() @ hd.abs(), cell.abs().t() @ hd.abs(), n, dw_dtype or w.dtype)):
        x, e = x * g, (e + (m + 8) * U32 * mass) * g
        out += [x, e + (half_step(dt) if dt != torch.float32 else U32) * (x.abs() + e) + 4 * U32 * x.abs() + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)]
    return (*out, left, (floor @ wd.abs()).norm(dim=1) * g)
