"""Cases of the training losses over a large vocabulary: what is timed and what the outputs have to be.

Three operators that a training step of this framework ends with:

  linear    `ops.linear_cross_entropy`: the LM head and the softmax cross entropy in one call that never holds the (rows, vocabulary) logits,
            with the gradients of the hidden states and of the head; with a teacher's top logits it is the distillation loss of the same head
  distill   `ops.distill_topk`: distillation from a teacher's top logits (+ the hard-label cross entropy) over logits that exist, with their gradient
  topk      `ops.topk_logits`: the teacher's side: the k largest logits of each row, in order, and the row's log-sum-exp

`own` chooses between the framework's kernels and plain torch in 32 bits."""
import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
WHISPER_VOCAB = 51865


def listed():
    return [
        # one target token alone: a latency probe of the whole loss + gradient path
        dict(name="head one token", op="linear", rows=1, d=512, vocab=WHISPER_VOCAB, dtype="f16", ignored=0.0, grad="h", k=0, temp=1.0, alpha=0.0),
        # whisper-base, batch 64, labels padded to 32 tokens, adapters only (the head is frozen): loss + gradient of the decoder's output
        dict(name="head base adapters", op="linear", rows=2048, d=512, vocab=WHISPER_VOCAB, dtype="f16", ignored=0.4, grad="h", k=0, temp=1.0, alpha=0.0),
        # the same model fully fine-tuned: the head's weight learns too
        dict(name="head base full", op="linear", rows=2048, d=512, vocab=WHISPER_VOCAB, dtype="bf16", ignored=0.1, grad="hw", k=0, temp=1.0, alpha=0.0),
        # whisper-large-v2's width, long transcripts: the largest training case
        dict(name="head large full", op="linear", rows=8192, d=1280, vocab=WHISPER_VOCAB, dtype="bf16", ignored=0.0, grad="hw", k=0, temp=1.0, alpha=0.0),
        # a validation pass: the loss alone, a ragged number of rows
        dict(name="head large loss only", op="linear", rows=5633, d=1280, vocab=WHISPER_VOCAB, dtype="f16", ignored=0.25, grad="none", k=0, temp=1.0, alpha=0.0),
        # distilling into whisper-base: soft and hard targets at temperature 2, everything learns
        dict(name="head distill base", op="linear", rows=2048, d=512, vocab=WHISPER_VOCAB, dtype="f16", ignored=0.3, grad="hw", k=64, temp=2.0, alpha=0.5),
        # soft targets alone, few rows, a short list
        dict(name="head distill ragged", op="linear", rows=777, d=768, vocab=WHISPER_VOCAB, dtype="bf16", ignored=0.2, grad="h", k=20, temp=1.0, alpha=1.0),
        # the toy configuration that the tests train: launches and latency
        dict(name="distill toy", op="distill", rows=37, vocab=1000, pad=24, dtype="f32", ignored=0.2, grad="z", k=8, temp=2.0, alpha=0.5),
        # whisper's padded vocabulary, batch 64: soft and hard targets over logits that the step holds anyway
        dict(name="distill base", op="distill", rows=2048, vocab=WHISPER_VOCAB, pad=103, dtype="f16", ignored=0.3, grad="z", k=64, temp=2.0, alpha=0.5),
        # soft targets alone, a long list, bfloat16 logits
        dict(name="distill long list", op="distill", rows=4096, vocab=WHISPER_VOCAB, pad=103, dtype="bf16", ignored=0.0, grad="z", k=128, temp=1.0, alpha=1.0),
        # a teacher that answers five beams
        dict(name="teacher five rows", op="topk", rows=5, vocab=WHISPER_VOCAB, pad=103, dtype="f16", k=16),
        # a teacher's pass over a training batch
        dict(name="teacher batch", op="topk", rows=4096, vocab=WHISPER_VOCAB, pad=103, dtype="f16", k=64),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "distill", "distill", "topk"])
    vocab = rng.choice([WHISPER_VOCAB, WHISPER_VOCAB, _log(rng, 1000, 60000)])
    if op == "linear":
        d = 8 * rng.randint(8, 160)
        k = rng.choice([0, 0, rng.randint(1, 128)])
        rows = _log(rng, 1, 6000 if k else 8192)
        return dict(op=op, rows=rows, d=d, vocab=vocab, dtype=rng.choice(["f16", "bf16"]), ignored=rng.choice([0.0, 0.25, 0.5]),
                    grad=rng.choice(["none", "h", "hw"]), k=k, temp=rng.choice([1.0, 1.5, 2.0, 4.0]) if k else 1.0,
                    alpha=rng.choice([0.3, 0.5, 0.9, 1.0]) if k else 0.0)
    pad = rng.choice([0, 1, 103, -vocab % 8])
    rows = _log(rng, 1, 4096)
    if op == "distill":
        return dict(op=op, rows=rows, vocab=vocab, pad=pad, dtype=rng.choice(["f16", "bf16", "f32"]), ignored=rng.choice([0.0, 0.25, 0.5]),
                    grad=rng.choice(["none", "z", "z"]), k=rng.randint(1, 128), temp=rng.choice([1.0, 1.5, 2.0, 4.0]), alpha=rng.choice([0.3, 0.5, 0.9, 1.0]))
    return dict(op=op, rows=rows, vocab=vocab, pad=pad, dtype=rng.choice(["f16", "bf16", "f32"]), k=rng.randint(1, 128))


def _ignored(case):
    return int(case["rows"] * case["ignored"])


def _teacher(case, labels, g, dev):
    """a teacher's list per row: distinct tokens, falling logits; half of the lists begin with the label; some rows have a shorter list or none"""
    n, v, k = case["rows"], case["vocab"], case["k"]
    start = torch.randint(0, v, (n, 1), generator=g, device=dev)
    idx = (start + 7919 * torch.arange(k, device=dev)) % v
    first = torch.rand(n, generator=g, device=dev) < 0.5
    idx[:, 0] = torch.where(first & (labels >= 0), labels, idx[:, 0])
    vals = 12.0 - 3.0 * torch.log1p(torch.arange(k, device=dev, dtype=torch.float32)) + 0.3 * torch.randn(n, k, generator=g, device=dev)
    vals = vals.sort(dim=1, descending=True).values
    keep = torch.where(torch.rand(n, 1, generator=g, device=dev) < 0.1, torch.randint(0, k + 1, (n, 1), generator=g, device=dev), k)
    idx = torch.where(torch.arange(k, device=dev) < keep, idx, -1)
    return vals.contiguous(), idx.to(torch.int32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    n, v, dt = case["rows"], case["vocab"], DT[case["dtype"]]
    s = {"case": case}
    if case["op"] == "topk":
        z = torch.randn(n, v + case["pad"], generator=g, device=dev) * 3.0
        s["logits"] = z.to(dt)[:, :v]
        s["vals"] = torch.empty(n, case["k"], device=dev)
        s["idx"] = torch.empty(n, case["k"], device=dev, dtype=torch.int32)
        s["lse"] = torch.empty(n, device=dev)
        return s
    labels = torch.randint(0, v, (n,), generator=g, device=dev)
    if case["op"] == "linear":
        d = case["d"]
        w = torch.randn(v, d, generator=g, device=dev) * (2.0 * d ** -0.5)
        h = torch.randn(n, d, generator=g, device=dev)
        h = h + w[labels] * (1.0 + torch.rand(n, 1, generator=g, device=dev))      # a model that has learnt something: the label's logit stands out
        s["h"], s["w"] = h.to(dt), w.to(dt)
        if case["grad"] != "none":
            s["dh"] = torch.empty_like(s["h"])
        if case["grad"] == "hw":
            s["dw"] = torch.empty_like(s["w"])
    else:
        z = torch.randn(n, v + case["pad"], generator=g, device=dev) * 2.0
        z.scatter_add_(1, labels.unsqueeze(1), 8.0 * torch.rand(n, 1, generator=g, device=dev))
        s["logits"] = z.to(dt)[:, :v]
        if case["grad"] == "z":
            s["dz"] = torch.empty(n, v + case["pad"], device=dev, dtype=dt)[:, :v]
    off = torch.randperm(n, generator=g, device=dev)[:_ignored(case)]
    labels[off] = -100
    s["labels"] = labels
    if case["k"]:
        s["top_vals"], s["top_idx"] = _teacher(case, labels, g, dev)
    s["scale"] = torch.tensor([1.0 if case["dtype"] != "f16" else 2048.0], device=dev)      # fp16 gradients travel with a loss scale
    s["row_loss"] = torch.empty(n, device=dev)
    s["loss"] = torch.empty(1, device=dev)
    s["nvalid"] = torch.empty(1, device=dev, dtype=torch.int32)
    return s


# ---------------------------------------------------------------- the framework's operators
def _run_own(s):
    from neuspeech1_amd import ops
    case = s["case"]
    if case["op"] == "topk":
        ops.topk_logits(s["logits"], case["k"], vals=s["vals"], idx=s["idx"], lse=s["lse"])
        return [s["vals"], s["idx"], s["lse"]]
    kw = dict(row_loss=s["row_loss"], loss=s["loss"], nvalid=s["nvalid"], loss_scale=s["scale"])
    if case["k"]:
        kw.update(top_vals=s["top_vals"], top_idx=s["top_idx"], temperature=case["temp"], alpha=case["alpha"])
    if case["op"] == "linear":
        ops.linear_cross_entropy(s["h"], s["w"], s["labels"], dh=s.get("dh"), dweight=s.get("dw"), **kw)
        return [s["loss"], s["row_loss"]] + [s[x] for x in ("dh", "dw") if x in s]
    ops.distill_topk(s["logits"], s["labels"], dlogits=s.get("dz"), **kw)
    return [s["loss"], s["row_loss"]] + ([s["dz"]] if "dz" in s else [])


# ---------------------------------------------------------------- plain torch, 32 bits
def _plain_losses(z, s, want_grad):
    """row losses over float32 logits z, their mean, and (want_grad) the gradient of scale x mean with respect to z"""
    case, labels = s["case"], s["labels"]
    n, v = z.shape
    valid = (labels >= 0) & (labels < v)
    nv = valid.sum().clamp(min=1)
    safe = torch.where(valid, labels, 0)
    temp, alpha = case["temp"], case["alpha"]
    rows = torch.zeros(n, device=z.device)
    grad = torch.zeros_like(z) if want_grad else None
    if alpha < 1.0:
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        rows = rows + (1.0 - alpha) * ((top + torch.log(total)).squeeze(1) - z.gather(1, safe.unsqueeze(1)).squeeze(1))
        if want_grad:
            p = e / total
            p.scatter_add_(1, safe.unsqueeze(1), torch.full((n, 1), -1.0, device=z.device))
            grad += (1.0 - alpha) * p
    if case["k"]:
        idx = s["top_idx"].long()
        there = (idx >= 0) & (idx < v)
        some = there.any(1, keepdim=True)
        col = torch.where(there, idx, 0)
        t = torch.where(there, s["top_vals"] / temp, torch.full_like(s["top_vals"], -3.0e38))
        t = t - t.amax(1, keepdim=True)
        et = torch.where(there, torch.exp(t), torch.zeros_like(t))
        st = et.sum(1, keepdim=True)
        prob = torch.where(some, et / st.clamp(min=1e-30), torch.zeros_like(et))
        logp = t - torch.log(st.clamp(min=1e-30))
        zt = z / temp
        top = zt.amax(1, keepdim=True)
        e = torch.exp(zt - top)
        total = e.sum(1, keepdim=True)
        logq = zt.gather(1, col) - (top + torch.log(total))
        kl = torch.where(prob > 0, prob * (logp - logq), torch.zeros_like(prob)).sum(1)
        rows = rows + alpha * temp * temp * kl
        if want_grad:
            q = torch.where(some, e / total, torch.zeros_like(e))
            q.scatter_add_(1, col, -prob)
            grad += alpha * temp * q
    rows = torch.where(valid, rows, torch.zeros_like(rows))
    if want_grad:
        grad = torch.where(valid.unsqueeze(1), grad * (s["scale"] / nv), torch.zeros_like(grad))
    return rows.sum().reshape(1) / nv, rows, grad


def _run_plain(s):
    case = s["case"]
    if case["op"] == "topk":
        z = s["logits"].float()
        top = z.amax(1, keepdim=True)
        lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True))).squeeze(1)
        vals, idx = torch.sort(z, dim=1, descending=True, stable=True)
        k = case["k"]
        return [vals[:, :k].contiguous(), idx[:, :k].to(torch.int32), lse]
    if case["op"] == "distill":
        loss, rows, dz = _plain_losses(s["logits"].float(), s, case["grad"] == "z")
        return [loss, rows] + ([dz.to(s["logits"].dtype)] if dz is not None else [])
    h, w = s["h"].float(), s["w"].float()
    loss, rows, dz = _plain_losses(h @ w.t(), s, case["grad"] != "none")
    out = [loss, rows]
    if case["grad"] != "none":
        out.append((dz @ w).to(s["h"].dtype))
    if case["grad"] == "hw":
        out.append((dz.t() @ h).to(s["w"].dtype))
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    n, v, k = case["rows"], case["vocab"], case["k"]
    size = {"f16": 2, "bf16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "topk":
        return {"bytes": float(n * (v * size + 8 * k + 4)), "flops": 2.0 * n * v}
    on = n - _ignored(case)
    side = 16.0 * n + 8.0 * on * k
    if case["op"] == "distill":
        softmaxes = (1 if case["alpha"] < 1.0 and case["temp"] != 1.0 else 0) + 1
        return {"bytes": side + float(size) * on * v + (float(size) * n * v if case["grad"] == "z" else 0.0), "flops": 3.0 * softmaxes * on * v}
    d = case["d"]
    products = {"none": 1, "h": 2, "hw": 3}[case["grad"]]
    out = {"none": 0, "h": n * d, "hw": n * d + v * d}[case["grad"]]
    return {"bytes": side + 2.0 * (on * d + v * d + out), "flops": 2.0 * products * on * v * d}


# ---------------------------------------------------------------- 64 bits, from the definitions
def _exact_rows(z, labels, vals, idx, temp, alpha, grad):
    """z: float64 logits of some rows.  Each row's target distributions are written out and the loss is their divergence from the softmax:
    (1 - alpha) * -log softmax(z)[label] + alpha * temp^2 * KL(softmax(vals / temp) || softmax(z / temp)); ignored rows: zero."""
    n, v = z.shape
    loss = torch.zeros(n, dtype=torch.float64, device=z.device)
    dz = torch.zeros_like(z) if grad else None
    ok = (labels >= 0) & (labels < v)
    r = torch.nonzero(ok).flatten()
    if len(r) == 0:
        return loss, dz
    zr = z[r]
    here = torch.arange(len(r), device=z.device)
    if alpha < 1.0:
        lp = zr - torch.logsumexp(zr, 1, keepdim=True)
        loss[r] += -(1.0 - alpha) * lp[here, labels[r]]
        if grad:
            gz = lp.exp_()
            gz[here, labels[r]] -= 1.0
            dz[r] += (1.0 - alpha) * gz
    if idx is not None:
        ids = idx[r].long()
        there = (ids >= 0) & (ids < v)
        t = torch.where(there, vals[r].double() / temp, torch.tensor(float("-inf"), dtype=torch.float64, device=z.device))
        has = there.any(1)
        t = torch.where(has.unsqueeze(1), t, torch.zeros_like(t))
        logp = t - torch.logsumexp(t, 1, keepdim=True)
        p = torch.where(there & has.unsqueeze(1), logp.exp(), torch.zeros_like(logp))
        lq = zr / temp
        lq = lq - torch.logsumexp(lq, 1, keepdim=True)
        cols = ids.clamp(min=0, max=v - 1)
        terms = p * (torch.where(p > 0, logp, torch.zeros_like(logp)) - lq.gather(1, cols))
        loss[r] += alpha * temp * temp * terms.sum(1)
        if grad:
            gz = lq.exp_()
            gz = gz.scatter_add(1, cols, -p) * has.unsqueeze(1)
            dz[r] += alpha * temp * gz
    return loss, dz


def exact(case, seed):
    if case["rows"] * case["vocab"] * case.get("d", 64) > 1e12:
        return None
    s = prepare(case, seed)
    n, v = case["rows"], case["vocab"]
    step = max(1, min(n, int(1.2e8) // v))
    if case["op"] == "topk":
        vals, idx, lse = [], [], []
        for a in range(0, n, step):
            z = s["logits"][a:a + step].double()
            lse.append(torch.logsumexp(z, 1))
            order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :case["k"]]
            idx.append(order)
            vals.append(z.gather(1, order))
        return [torch.cat(vals), torch.cat(idx), torch.cat(lse)]
    linear = case["op"] == "linear"
    labels, vals, idx = s["labels"], s.get("top_vals"), s.get("top_idx")
    grad = case["grad"] != "none"
    factor = float(s["scale"]) / max(int(((labels >= 0) & (labels < v)).sum()), 1)
    rows, dh, dzs = [], [], []
    w = s["w"].double() if linear else None
    dw = torch.zeros_like(w) if case["grad"] == "hw" else None
    for a in range(0, n, step):
        b = min(n, a + step)
        z = s["h"][a:b].double() @ w.t() if linear else s["logits"][a:b].double()
        row, dz = _exact_rows(z, labels[a:b], None if vals is None else vals[a:b], None if idx is None else idx[a:b], case["temp"], case["alpha"], grad)
        rows.append(row)
        if grad:
            dz *= factor
            if linear:
                dh.append(dz @ w)
                if dw is not None:
                    dw += dz.t() @ s["h"][a:b].double()
            else:
                dzs.append(dz)
    rows = torch.cat(rows)
    out = [rows.sum().reshape(1) / max(int(((labels >= 0) & (labels < v)).sum()), 1), rows]
    if linear and grad:
        out.append(torch.cat(dh))
        if dw is not None:
            out.append(dw)
    elif grad:
        out.append(torch.cat(dzs))
    return out
