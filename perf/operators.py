"""The loss heads of fea_amd.functional as measured work: linear_cross_entropy (a projection and a softmax cross entropy over
its outputs) and linear_distillation (the same projection against a teacher's top logits), forward alone and with the gradients.

`own = True` runs the framework's kernels, `own = False` the same mathematics in elementary torch operations in 32 bits."""
import torch

own = False


# ---- the cases ----------------------------------------------------------------------------------------------------------
# op: "ce" / "kd"; rows x dim hidden states, classes x dim weight; train: loss and gradients, else the loss of each row;
# ignored: share of the rows without a label (ce) or without any teacher entry (kd); short: share of the teacher's entries
# that are missing.

def _ce(name, rows, dim, classes, dtype, train, bias=False, ignored=0.0):
    return {"name": name, "op": "ce", "rows": rows, "dim": dim, "classes": classes, "dtype": dtype, "train": train, "bias": bias,
            "ignored": ignored}


def _kd(name, rows, dim, classes, top, dtype, train, temperature=1.0, bias=False, ignored=0.0, short=0.0):
    return {"name": name, "op": "kd", "rows": rows, "dim": dim, "classes": classes, "top": top, "dtype": dtype, "train": train,
            "temperature": temperature, "bias": bias, "ignored": ignored, "short": short}


def listed():
    return [
        # the score of one answer: one row against the whole vocabulary, the latency of a single call
        _ce("ce score 1", 1, 1024, 32768, "bf16", False),
        # scores of a short ragged list of answers, odd vocabulary
        _ce("ce score 37", 37, 2048, 50021, "bf16", False, bias=True),
        # a step of an ordinary training job, a tenth of the rows padded
        _ce("ce train 2048", 2048, 2048, 32000, "bf16", True, ignored=0.1),
        # the largest: a long batch over a large vocabulary
        _ce("ce train 8192", 8192, 4096, 131072, "bf16", True, ignored=0.02),
        # 32-bit training of a ragged batch, no size a multiple of anything
        _ce("ce train fp32 odd", 1531, 643, 10007, "fp32", True, bias=True, ignored=0.2),
        # per-pixel classes of the segmentation network's own head: 64 channels, 6 classes, a batch of 64 images of 512 x 512
        _ce("ce pixels", 64 * 512 * 512, 64, 6, "bf16", True, bias=True, ignored=0.05),
        # validation loss of a few rows against the teacher
        _kd("kd eval 64", 64, 1024, 32768, 16, "bf16", False, temperature=2.0, ignored=0.05),
        # distillation step, ordinary
        _kd("kd train 2048", 2048, 2048, 32000, 32, "bf16", True, temperature=2.0, ignored=0.05, short=0.1),
        # distillation step, a large vocabulary and many entries
        _kd("kd train 4096", 4096, 4096, 131072, 64, "bf16", True),
        # 32-bit, ragged
        _kd("kd train fp32 odd", 777, 515, 5003, 7, "fp32", True, temperature=4.0, bias=True, ignored=0.1, short=0.3),
        # per-pixel distillation of the segmentation head, three of six classes kept: 8 images of 512 x 512
        _kd("kd pixels", 8 * 512 * 512, 64, 6, 3, "bf16", True, temperature=2.0, bias=True, short=0.1),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def _even(rng, n, step):
    """n as it is, or (twice of three times) the next multiple of step below it."""
    return n if n <= step or rng.random() < 1 / 3 else n // step * step


def draw(rng):
    dtype = "bf16" if rng.random() < 0.75 else "fp32"
    train = rng.random() < 0.7
    bias = rng.random() < 0.4
    ignored = rng.choice([0.0, 0.02, 0.1, 0.3])
    if rng.random() < 0.25:                        # per-pixel heads
        rows, dim, classes = _log_int(rng, 1 << 14, 1 << 23), _even(rng, rng.randint(16, 64), 8), rng.randint(2, 24)
    else:                                          # vocabularies
        dim = _even(rng, _log_int(rng, 48, 4096), 64)
        classes = _even(rng, _log_int(rng, 600, 131072), 64)
        rows = _log_int(rng, 1, 8192)
    if rng.random() < 0.55:
        return {k: v for k, v in _ce("", rows, dim, classes, dtype, train, bias, ignored).items() if k != "name"}
    top = min(_log_int(rng, 1, 64), classes, max(1, (1 << 25) // rows))
    return {k: v for k, v in _kd("", rows, dim, classes, top, dtype, train, rng.choice([1.0, 2.0, 3.5]), bias, ignored,
                                 rng.choice([0.0, 0.2])).items() if k != "name"}


# ---- inputs -------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    rows, dim, classes = case["rows"], case["dim"], case["classes"]
    # a weight that gives logits of a standard deviation near 1.5, labels that thin out with their number, and hidden states
    # that lean towards their label's row: a network some way into its training
    w = torch.randn(classes, dim, generator=g, device=dev) * (1.5 / dim ** 0.5)
    label = (classes * torch.rand(rows, generator=g, device=dev, dtype=torch.float64) ** 2).long().clamp_(max=classes - 1)
    h = torch.randn(rows, dim, generator=g, device=dev)
    lean = torch.rand(rows, 1, generator=g, device=dev) * 3
    part = 1 << 21
    for a in range(0, rows, part):
        h[a:a + part] += lean[a:a + part] * w[label[a:a + part]]
    s = {"case": case, "hidden": h.to(dt), "weight": w.to(dt),
         "bias": torch.randn(classes, generator=g, device=dev) * 0.3 if case["bias"] else None}
    del h, w
    gone = torch.rand(rows, generator=g, device=dev) < case["ignored"]
    if case["op"] == "ce":
        s["target"] = label.masked_fill_(gone, -100)
    else:
        top = case["top"]
        gaps = torch.randint(1, max(1, classes // top) + 1, (rows, top), generator=g, device=dev)
        gaps[:, 0] = label - gaps[:, 1:].sum(1) // 2
        index = torch.cumsum(gaps, 1) % classes                   # distinct: the gaps after the first add up to less than classes
        index = torch.gather(index, 1, torch.rand(rows, top, generator=g, device=dev).argsort(1))
        fall = torch.rand(rows, top, generator=g, device=dev).mul_(1.5 if top < 16 else 0.5).cumsum(1)
        index[torch.rand(rows, top, generator=g, device=dev) < case["short"]] = -1
        index[gone] = -1
        s["teacher_index"], s["teacher_logits"] = index, (9.0 - fall).to(dt)
    if case["train"]:
        for k in ("hidden", "weight", "bias"):
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------

def _own_run(s):
    from fea_amd import functional as F
    c = s["case"]
    how = {"bias": s["bias"], "reduction": "mean" if c["train"] else "none"}
    if c["op"] == "ce":
        loss = F.linear_cross_entropy(s["hidden"], s["weight"], s["target"], **how)
    else:
        loss = F.linear_distillation(s["hidden"], s["weight"], s["teacher_logits"], s["teacher_index"], temperature=c["temperature"], **how)
    if not c["train"]:
        return {"loss": loss}
    names = [k for k in ("hidden", "weight", "bias") if s[k] is not None]
    return {"loss": loss.detach(), **dict(zip(names, torch.autograd.grad(loss, [s[k] for k in names])))}


def run(s):
    if own:
        return _own_run(s)
    c = s["case"]
    h, w = s["hidden"].detach().float(), s["weight"].detach().float()
    t = c.get("temperature", 1.0)
    z = h @ w.t()
    if s["bias"] is not None:
        z += s["bias"].detach()
    if t != 1.0:
        z /= t
    top = z.max(1, keepdim=True).values
    q = torch.exp(z - top)
    total = q.sum(1, keepdim=True)
    lse = torch.log(total) + top
    if c["op"] == "ce":
        counts = s["target"] != -100
        index = s["target"].clamp(min=0)[:, None]
        p = counts[:, None].float()
        rowloss = torch.where(counts, (lse - torch.gather(z, 1, index))[:, 0], 0.0)
    else:
        there = s["teacher_index"] >= 0
        counts = there.any(1)
        index = s["teacher_index"].clamp(min=0)
        a = torch.where(there, s["teacher_logits"].float() / t, -torch.inf)
        a = a - torch.where(counts, a.max(1).values, 0.0)[:, None]
        e = torch.exp(a)
        norm = torch.where(counts, e.sum(1), 1.0)[:, None]
        p = e / norm
        logp = a - torch.log(norm)
        rowloss = t * t * torch.where(there, p * (logp - torch.gather(z, 1, index) + lse), 0.0).sum(1)
    if not c["train"]:
        return {"loss": rowloss}
    n = counts.sum().clamp(min=1)
    dz = q.div_(total)
    dz.scatter_add_(1, index, -p)
    dz *= (counts.float() * t / n)[:, None]
    out = {"loss": (rowloss.double().sum() / n).float(), "hidden": (dz @ w).to(s["hidden"].dtype),
           "weight": (dz.t() @ h).to(s["weight"].dtype)}
    if s["bias"] is not None:
        out["bias"] = dz.double().sum(0).float() if c["rows"] > 100000 else dz.sum(0)
    return out


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    rows, dim, classes = case["rows"], case["dim"], case["classes"]
    once = (rows * dim + classes * dim) * size + (classes * 4 if case["bias"] else 0)
    labels = rows * 8 if case["op"] == "ce" else rows * case["top"] * (8 + size)
    return {"bytes": 2 * once + labels + 4 if case["train"] else once + labels + 4 * rows,
            "flops": (6 if case["train"] else 2) * rows * dim * classes}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    if 6.0 * case["rows"] * case["dim"] * case["classes"] > 2e14:
        return None
    s = prepare(case, seed)
    w = s["weight"].detach().double()
    b = s["bias"].detach().double() if s["bias"] is not None else torch.zeros(case["classes"], dtype=torch.float64, device=w.device)
    t = float(case.get("temperature", 1.0))
    rows = case["rows"]
    part = max(1, min(rows, (1 << 28) // case["classes"], (1 << 26) // case["dim"]))
    if case["op"] == "ce":
        live = s["target"] >= 0
    else:
        live = (s["teacher_index"] >= 0).sum(1) > 0
    n = max(1, int(live.sum()))
    losses, dh, dw, db = [], [], torch.zeros_like(w), torch.zeros_like(b)
    for a in range(0, rows, part):
        x = s["hidden"].detach()[a:a + part].double()
        on = live[a:a + part]
        logq = torch.log_softmax((torch.matmul(x, w.T) + b) / t, dim=-1)
        want = torch.zeros_like(logq)
        if case["op"] == "ce":
            want[on, s["target"][a:a + part][on]] = 1.0
            plogp = 0.0
        else:
            i = s["teacher_index"][a:a + part]
            v = (s["teacher_logits"][a:a + part].double() / t).masked_fill(i < 0, -1e300)
            p = torch.softmax(v, dim=-1).masked_fill(i < 0, 0.0)
            want.scatter_add_(1, i.clamp(min=0), p)
            plogp = torch.special.xlogy(p, p).sum(1)
        losses.append(t * t * on * (plogp - (want * logq).sum(1)))
        if case["train"]:
            want.neg_().add_(logq.exp_()).mul_(on[:, None] * (t / n))
            dh.append(torch.matmul(want, w))
            dw += torch.matmul(want.T, x)
            db += want.sum(0)
    loss = torch.cat(losses)
    if not case["train"]:
        return {"loss": loss}
    out = {"loss": loss.sum() / n, "hidden": torch.cat(dh), "weight": dw}
    if s["bias"] is not None:
        out["bias"] = db
    return out
