"""The loss heads over many classes in 64 bits, with the bounds that their kernels' arithmetic gives.

u = torch.finfo(dtype).eps / 2 (a rounding to the storage type), e = 2^-24 (a rounding in 32 bits), with B = max_v sum_d |h_d w_d| + |b_v|:
  a logit is off by dz <= (D + 4) e B / T (D products and sums, bias, scale), an exponential by 3 e more and e |z - lse| for its argument;
  log-sum-exp by the largest of these and the sum's (16 + V / 64) e;  so a loss by 2 of them, a softmax value q by the same relative to q.
  A teacher's share p = exp(x_k) / sum exp(x_k), x_k = (a_k - max a) / T in 32 bits: a and 1 / T are rounded and multiplied on either side of the
  difference (4 e A with A = max |a| / T), the difference is (2 e A) and its exponential's argument (2 x 2 e A): 10 e A of itself, the sum the
  same, so p is off by 20 e A of itself and log p by 20 e A.
  With bf16 operands the backward takes z from 16 bits that the forward kept (more than 64 rows, no bias gradient): half a step of
  64 / 65535 off, so q by up to exp(32 / 65535) - 1 < 4.89e-4 of itself (and by the e^-64 that counts as 0).
  dz = g (q - p) is rounded once to the storage type; dh and dw add the products' fp32 sums and one rounding to the storage type.
  Where every row has its own upstream gradient, dw's product takes rnd(q - p) and rnd(g h), two operands rounded once each:
  |rnd(x) rnd(y) - x y| <= (2 u + u^2) |x y|, so its terms |dz| |h| are off by u (1 + u) more than with one upstream gradient
  (which meets the fp32 sum). """
import torch

E = 2.0 ** -24


def case(rows, dim, classes, dtype, seed=0, top=0, ignored=0.0, short=0.0, bias=False):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, dim, generator=g).to(dtype)
    w = (torch.randn(classes, dim, generator=g) * (1.5 / dim ** 0.5)).to(dtype)
    b = torch.randn(classes, generator=g) * 0.3 if bias else None
    gone = torch.rand(rows, generator=g) < ignored
    if not top:
        t = torch.randint(0, classes, (rows,), generator=g)
        return h, w, b, t.masked_fill(gone, -100)
    i = torch.randint(0, classes, (rows, top), generator=g)          # the same class twice in a row happens
    i[torch.rand(rows, top, generator=g) < short] = -1
    i[gone] = -1
    return h, w, b, i, (torch.randn(rows, top, generator=g) * 2 + 5).to(dtype)


def evaluate(h, w, b, index, tlog=None, ignore_index=-100, temperature=1.0, reduction="mean", gout=None, kept=None, norms=False):
    """{"loss", "hidden", "weight", "bias"}: values and bounds, as (value, bound) pairs in 64 bits.  gout: upstream gradient of the losses
    (rows) for "none", else of the result.  kept: the
    backward had the forward's logits (None: as a head whose every operand has a gradient would).
    norms: "hidden" and "weight" as (value, bound of the Frobenius norm of all their errors together).  Element by element a bound adds up
    the sizes of a column's errors, and from some hundred rows on one row's whole share fits in.  With E the errors of dz, |E| <= off:
    |E w|_F <= |off|_F |w|_2 and |E^T h|_F <= |off|_F |h|_2 (the largest singular value), the products' own roundings element by element on
    top.  With an upstream gradient for every row dw = (q - p)^T (g h), both rounded: |E^T (g h)|_F + |(q - p)^T (u |g h|)|_F, E of q - p
    alone, the product of both errors u times the first."""
    dtype, t = h.dtype, temperature
    u = torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else E
    hd, wd = h.double().reshape(-1, h.shape[-1]), w.double()
    rows, dim = hd.shape
    v = wd.shape[0]
    bd = torch.zeros(v, dtype=torch.float64) if b is None else b.double()
    z = (hd @ wd.T + bd) / t
    lse = torch.logsumexp(z, 1)
    q = torch.exp(z - lse[:, None])
    p = torch.zeros_like(z)
    if tlog is None:
        ix = index.reshape(-1)
        on = ix != ignore_index
        p[on, ix[on]] = 1.0
        loss = torch.where(on, lse - z.gather(1, torch.where(on, ix, 0)[:, None])[:, 0], 0.0)
        scale = 1.0
        spread, arg = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    else:
        ix, a = index.reshape(rows, -1), tlog.double().reshape(rows, -1) / t
        a = a.masked_fill(ix < 0, -torch.inf)
        on = (a > -torch.inf).any(1)
        pk = torch.softmax(torch.where(on[:, None], a, 0.0), 1) * on[:, None]
        p.scatter_add_(1, ix.clamp(min=0), pk)
        zk = z.gather(1, ix.clamp(min=0))
        loss = t * t * torch.where(pk > 0, pk * (torch.log(pk.clamp(min=1e-300)) - zk + lse[:, None]), 0.0).sum(1)
        scale = t * t
        arg = 20 * E * torch.where(torch.isfinite(a), a, 0.0).abs().amax(1)
        spread = (pk * (torch.log(pk.clamp(min=1e-300)).abs() + zk.abs() + lse.abs()[:, None])).nan_to_num(0.0, 0.0, 0.0).sum(1)
    n = max(1, int(on.sum()))
    big = (hd.abs() @ wd.abs().T + torch.where(bd > -1e30, bd, 0.0).abs()).amax(1)
    dz_log = ((dim + 4) * E * big / t + (16 + v / 64) * E + 3 * E + E * (z - lse[:, None]).masked_fill(z < -1e30, 0).abs().amax(1)).masked_fill(~on, 0.0)
    loss_off = scale * (2 * dz_log + E * lse.abs().masked_fill(~on, 0.0) + ((8 + (0 if tlog is None else index.shape[-1])) * E + arg) * (spread + 1))
    loss = torch.where(on, loss, 0.0)
    if reduction == "none":
        g = torch.ones(rows, dtype=torch.float64) if gout is None else gout.double().reshape(-1)
        out = {"loss": (loss, loss_off + E * loss.abs())}
    else:
        div = n if reduction == "mean" else 1
        g = torch.full((rows,), (1.0 if gout is None else float(gout)) / div, dtype=torch.float64)
        out = {"loss": (loss.sum() / div, loss_off.sum() / div + 2 * E * loss.abs().sum() / div)}
    g = g * t * on
    q, p = q * on[:, None], p * on[:, None]
    q = q.nan_to_num(0.0) if not on.all() else q
    hd = torch.where(on[:, None], hd, 0.0)
    dz = g[:, None] * (q - p)
    kept = kept if kept is not None else rows > 64 and b is None and not (v <= 32 and dim <= 64 and rows >= 4096)
    kept = 4.89e-4 if kept and dtype == torch.bfloat16 else 0.0
    off = g.abs()[:, None] * (q * kept * (1 + u) + (1.7e-28 if kept else 0.0) + q * 2 * dz_log[:, None] + (8 + (0 if tlog is None else index.shape[-1])) * E * (p + q) + p * arg[:, None]) + u * dz.abs() + 2 * E * dz.abs()
    dh, dw = dz @ wd, dz.T @ hd
    if norms:
        def largest(x):                                     # singular value, from the smaller Gram matrix; 1e-9 for its own roundings
            return float(torch.linalg.eigvalsh(x.T @ x if x.shape[0] >= x.shape[1] else x @ x.T)[-1].clamp(min=0).sqrt()) * (1 + 1e-9)
        sums = (v + 8) * E * (dz.abs() @ wd.abs()) + u * dh.abs()
        out["hidden"] = (dh, float(off.norm()) * largest(wd) + float(sums.norm()))
        sums = (rows + 8) * E * (dz.abs().T @ hd.abs()) + u * dw.abs()
        if reduction == "none":
            gh, size = g[:, None] * hd, g.abs()[:, None].clamp(min=1e-300)
            first = float((off / size).norm()) * largest(gh)
            out["weight"] = (dw, first * (1 + u) + u * float(gh.norm()) * largest(q - p) + float(sums.norm()))
        else:
            out["weight"] = (dw, float(off.norm()) * largest(hd) + float(sums.norm()))
        return out
    out["hidden"] = (dh, off @ wd.abs() + (v + 8) * E * (dz.abs() @ wd.abs()) + u * dh.abs() + 1e-37)
    own = u * (1 + u) if reduction == "none" else 0.0
    out["weight"] = (dw, off.T @ hd.abs() + own * (dz.abs().T @ hd.abs()) + (rows + 8) * E * (dz.abs().T @ hd.abs()) + u * dw.abs() + 1e-37)
    offb = g.abs()[:, None] * (q * 2 * dz_log[:, None] + 8 * E * (p + q) + p * arg[:, None]) + 4 * E * g.abs()[:, None] * (q + p)
    out["bias"] = (dz.sum(0), offb.sum(0) + 20 * E * (g.abs()[:, None] * (q + p)).sum(0) + 1e-37)
    return out


def check(name, got, want):
    value, bound = want
    got = got.detach().double().cpu().reshape(value.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{name}: NaN in other places"
    far = (got - value).abs() - bound
    far = far[torch.isfinite(value)]
    same = got[~torch.isfinite(value) & ~torch.isnan(value)] == value[~torch.isfinite(value) & ~torch.isnan(value)]
    assert bool(same.all()), f"{name}: other infinities"
    assert far.numel() == 0 or float(far.max()) <= 0, f"{name}: {float(far.max()):.3e} beyond its bound, worst ratio " \
        f"{float(((got - value).abs() / bound)[torch.isfinite(value)].max()):.2f}"


def check_norm(name, got, want):
    """The Frobenius norm of all errors together."""
    value, bound = want
    off = float((got.detach().double().cpu().reshape(value.shape) - value).norm())
    assert off <= bound, f"{name}: errors of norm {off:.3e}, {off / bound:.2f} of their bound"


# Layouts of a single row [D] (the last position of a long sequence, a column, the start of wider rows, of none that is aligned, every second
# element), as [1, D].
ONE_ROW = ["plain", "last of many", "a column", "of rows that end off a line", "off a line", "every second"]


def one_row(name, x):
    """x [D] in the layout `name`, a tensor of one row."""
    d = x.shape[0]
    if name == "plain":
        return x.clone()[None]
    if name == "last of many":
        n = (1 << 21) // d + 2
        t = torch.zeros(1, n, d, dtype=x.dtype, device=x.device)
        t[:, -1] = x
        return t[:, -1]
    if name == "a column":
        return x.clone()[:, None].t()
    if name == "of rows that end off a line":
        t = torch.zeros(1, d + 3, dtype=x.dtype, device=x.device)
        t[:, :d] = x
        return t[:, :d]
    if name == "off a line":
        t = torch.zeros(3, d + 1, dtype=x.dtype, device=x.device)
        t[1:2, 1:] = x
        return t[1:2, 1:]
    t = torch.zeros(1, 2 * d, dtype=x.dtype, device=x.device)
    t[:, ::2] = x
    return t[:, ::2]
