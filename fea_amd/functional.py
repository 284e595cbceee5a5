"""Segmentation loss, mask binarisation and IoU on the HIP kernels (the reference has none), and the loss heads over many classes:
`linear_cross_entropy`, `linear_distillation`."""
from __future__ import annotations

import os

import torch

from . import _lib as L


class _BceDice(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target):
        n, c, h, w = logits.shape
        lg = logits.detach().contiguous().float()
        tg = target.contiguous()
        if tg.dtype != torch.uint8:
            tg = (tg > 0).to(torch.uint8)
        dev = lg.device
        part = torch.empty(L.call("fea_loss_blocks", n, c, h * w) * 4, dtype=torch.float32, device=dev)
        sums = torch.empty((c, 4), dtype=torch.float64, device=dev)
        loss = torch.empty(1, dtype=torch.float32, device=dev)
        S = L.stream_ptr()
        L.call("fea_bce_dice_sums", lg, tg, sums, part, n, c, h * w, S)
        L.call("fea_bce_dice_grad", lg, tg, sums, loss, None, 1.0, n, c, h * w, S)
        ctx.save_for_backward(lg, tg, sums)
        return loss[0]

    @staticmethod
    def backward(ctx, gout):
        lg, tg, sums = ctx.saved_tensors
        n, c, h, w = lg.shape
        dl = torch.empty_like(lg)
        L.call("fea_bce_dice_grad", lg, tg, sums, None, dl, 1.0, n, c, h * w, L.stream_ptr())
        return dl * gout, None


def bce_dice_loss(logits: torch.Tensor, target: torch.Tensor) -> torch.Tensor:
    """BCEWithLogits(mean) + 1 - mean_c Dice_c  (see oracle/unet_oracle.py:bce_dice_loss)."""
    if not logits.is_cuda:
        raise L.FeaError("fea_amd.functional runs on a ROCm device only")
    return _BceDice.apply(logits, target)


def bce_dice_loss_and_grad(logits: torch.Tensor, target_u8: torch.Tensor, dlogits: torch.Tensor = None, ws=None):
    """Fused fast path for training loops: returns (loss[1], dlogits) without autograd."""
    n, c, h, w = logits.shape
    dev = logits.device
    if ws is None:
        ws = {}
    key = (n, c, h, w)
    if ws.get("key") != key:
        ws["key"] = key
        ws["part"] = torch.empty(L.call("fea_loss_blocks", n, c, h * w) * 4, dtype=torch.float32, device=dev)
        ws["sums"] = torch.empty((c, 4), dtype=torch.float64, device=dev)
        ws["loss"] = torch.empty(1, dtype=torch.float32, device=dev)
        ws["dl"] = torch.empty((n, c, h, w), dtype=torch.float32, device=dev)
    if dlogits is None:
        dlogits = ws["dl"]
    S = L.stream_ptr()
    L.call("fea_bce_dice_sums", logits, target_u8, ws["sums"], ws["part"], n, c, h * w, S)
    L.call("fea_bce_dice_grad", logits, target_u8, ws["sums"], ws["loss"], dlogits, 1.0, n, c, h * w, S)
    return ws["loss"], dlogits


def binarise_mask(grey_u8: torch.Tensor) -> torch.Tensor:
    """target = grey > 127 (uint8 {0,1})."""
    g = grey_u8.contiguous()
    out = torch.empty_like(g)
    L.call("fea_binarise", g, out, g.numel(), L.stream_ptr())
    return out


def mask_iou_counts(logits: torch.Tensor, target_u8: torch.Tensor, want_mask: bool = True, inter=None, union=None):
    """pred = logits > 0; per-class int64 intersection / union counts
    (accumulated into `inter`/`union` when given)."""
    n, c, h, w = logits.shape
    lg = logits.detach().contiguous().float()
    tg = target_u8.contiguous()
    dev = lg.device
    mask = torch.empty((n, c, h, w), dtype=torch.uint8, device=dev) if want_mask else None
    if inter is None:
        inter = torch.zeros(c, dtype=torch.int64, device=dev)
    if union is None:
        union = torch.zeros(c, dtype=torch.int64, device=dev)
    L.call("fea_mask_iou", lg, tg, mask, inter, union, n, c, h * w, L.stream_ptr())
    return mask, inter, union


def threshold_mask(logits: torch.Tensor) -> torch.Tensor:
    """pred = logits > 0 as uint8 {0,1} (inference.py:39-40 without ground truth): fea_mask_iou with no target."""
    n, c, h, w = logits.shape
    lg = logits.detach().contiguous().float()
    mask = torch.empty((n, c, h, w), dtype=torch.uint8, device=lg.device)
    L.call("fea_mask_iou", lg, None, mask, None, None, n, c, h * w, L.stream_ptr())
    return mask


def iou_from_counts(inter: torch.Tensor, union: torch.Tensor):
    iou = torch.where(union > 0, inter.double() / union.clamp(min=1).double(), torch.ones_like(inter, dtype=torch.float64))
    return iou, iou.mean()


# ---- loss heads over many classes ---------------------------------------------------------------------------------------

def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """[..., D] -> [rows, D] as the kernels read it: contiguous rows, 16-byte aligned where D allows it, less than 2^21 elements apart."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    epc = 16 // t.element_size()
    d = t.shape[1]
    if t.shape[0] == 1 and t.stride(0) != d:           # the stride of a single row means nothing, and contiguous() would keep it
        t = t.reshape(-1).contiguous().as_strided((1, d), (d, 1))
    if (t.stride(1) != 1 and d > 1) or t.stride(0) < d or t.stride(0) >= 1 << 21 or (d % epc == 0 and (t.data_ptr() % 16 or t.stride(0) % epc)):
        t = t.contiguous()
        if d % epc == 0 and t.data_ptr() % 16:         # contiguous already, but a view at an odd offset
            t = t.clone()
    return t


def _row_state(row, rows, k, teacher):
    """Addresses of stat [rows, 2], dsel [rows, k] and, with a teacher, psel [rows, k] in the one tensor that holds them."""
    at = row.data_ptr()
    return at, at + rows * 8, at + rows * (8 + 4 * k) if teacher else None


def _linear_loss_fwd(hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits, grads):
    """One forward call.  grads: 0, or what the backward will want (1 hidden, 2 weight, 4 bias).  Returns (loss, saved)."""
    dev = hidden.device
    h, w = _aligned_rows(hidden), _aligned_rows(weight)
    (rows, d), v = h.shape, w.shape[0]
    k = 1 if tlog is None else index.shape[-1]
    ix = index if index.dtype == torch.int64 else index.to(torch.int64)
    ix = ix.contiguous()
    b = None if bias is None else bias.detach().contiguous()
    dt = L.dt_code(h.dtype)
    row = keep = None
    stat = dsel = psel = None
    if grads:
        row = torch.empty(rows * (2 + k * (1 if tlog is None else 2)), dtype=torch.float32, device=dev)
        stat, dsel, psel = _row_state(row, rows, k, tlog is not None)
        n = 0 if keep_logits is False else L.load().fea_linear_loss_keep_bytes(rows, d, v, dt, grads >> 2)
        if n > 0 and (keep_logits or n <= int(os.environ.get("FEA_AMD_LINEAR_KEEP", 1 << 33))):
            try:
                keep = torch.empty(n, dtype=torch.uint8, device=dev)
            except torch.cuda.OutOfMemoryError:
                if keep_logits:
                    raise
                # (left open: the backward recomputes them)
    if reduction == "none":
        loss, count = torch.empty(index.shape if tlog is None else index.shape[:-1], dtype=torch.float32, device=dev), None
        outs = (loss, None, None, 0)
    else:
        loss = torch.empty((), dtype=torch.float32, device=dev)
        count = torch.empty((), dtype=torch.int32, device=dev)
        outs = (None, loss, count, int(reduction == "mean"))
    n = L.load().fea_linear_loss_ws_bytes(rows, d, v, k, dt, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    if tlog is None:
        L.call("fea_linear_ce_fwd", h, h.stride(0), w, w.stride(0), b, ix, ignore_index, stat, dsel, keep, grads >> 2, *outs, ws, n, rows, d, v, dt, L.stream_ptr(dev.index))
    else:
        tl = tlog.detach().contiguous()
        L.call("fea_linear_kd_fwd", h, h.stride(0), w, w.stride(0), b, tl, L.dt_code(tl.dtype), ix, k, temperature, stat, dsel, psel, keep, grads >> 2,
               *outs, ws, n, rows, d, v, dt, L.stream_ptr(dev.index))
    return loss, (ix, row, keep, count)


class _LinearLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits, train):
        grads = sum(bit for bit, want in zip((1, 2, 4), ctx.needs_input_grad) if want) if train else 0
        loss, (ix, row, keep, count) = _linear_loss_fwd(hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits, grads)
        if not grads:
            return loss
        # the operands themselves are saved, so that autograd sees a change in place between forward and backward
        ctx.save_for_backward(hidden, weight, bias, ix, row, keep, count if reduction == "mean" else None)
        ctx.how = (temperature, reduction, 1 if tlog is None else index.shape[-1], tlog is not None, grads)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gout):
        hidden, weight, bias, ix, row, keep, count = ctx.saved_tensors
        temperature, reduction, k, teacher, grads = ctx.how
        # (the autograd engine runs this on the forward's device and stream)
        h, w = _aligned_rows(hidden), _aligned_rows(weight)
        b = None if bias is None else bias.detach().contiguous()
        (rows, d), v = h.shape, w.shape[0]
        dt = L.dt_code(h.dtype)
        stat, dsel, psel = _row_state(row, rows, k, teacher)
        dh = torch.empty(hidden.shape, dtype=h.dtype, device=h.device) if grads & 1 else None
        dw = torch.empty(weight.shape, dtype=w.dtype, device=w.device) if grads & 2 else None
        db = torch.empty(v, dtype=torch.float32, device=h.device) if grads & 4 else None
        go = gout.detach().contiguous()
        n = L.load().fea_linear_loss_ws_bytes(rows, d, v, k, dt, grads | (8 if keep is not None else 0))
        ws = torch.empty(n, dtype=torch.uint8, device=h.device)
        L.call("fea_linear_loss_bwd", h, h.stride(0), w, w.stride(0), b, ix, k, stat, dsel, psel, keep, grads >> 2, count, go, int(reduction == "none"),
               temperature, dh, dw, db, ws, n, rows, d, v, dt, L.stream_ptr(h.device.index))
        return dh, dw, db, None, None, None, None, None, None, None


_LABELS = (torch.int64, torch.int32, torch.int16, torch.int8, torch.uint8)


def _linear_loss(who, hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits):
    if torch.jit.is_tracing():
        raise L.FeaError(f"{who}: a trace (torch.jit) does not record the kernels; capture the call in a graph (torch.cuda.graph)")
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"{who}: reduction {reduction!r} (use 'mean', 'sum' or 'none')")
    if keep_logits is not None and not isinstance(keep_logits, bool):
        raise ValueError(f"{who}: keep_logits {keep_logits!r} (use True, False or None)")
    if not isinstance(hidden, torch.Tensor) or not isinstance(weight, torch.Tensor) or not isinstance(index, torch.Tensor):
        raise ValueError(f"{who}: hidden, weight and the labels are tensors")
    if hidden.dtype != weight.dtype or hidden.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{who}: hidden and weight are both float32 or both bfloat16 (got {hidden.dtype}, {weight.dtype})")
    if hidden.dim() < 1 or weight.dim() != 2 or hidden.shape[-1] != weight.shape[1] or 0 in weight.shape:
        raise ValueError(f"{who}: hidden [..., D] and weight [classes, D] do not fit (got {tuple(hidden.shape)}, {tuple(weight.shape)})")
    if weight.shape[0] > 1 << 24 or weight.shape[1] > 1 << 16 or hidden.numel() // weight.shape[1] >= 1 << 30:
        raise ValueError(f"{who}: up to 2^24 classes of 2^16 features and less than 2^30 rows are served (got {tuple(hidden.shape)}, {tuple(weight.shape)})")
    if index.dtype not in _LABELS:
        raise ValueError(f"{who}: labels are integers (got {index.dtype})")
    lead = index.shape if tlog is None else index.shape[:-1]
    if lead != hidden.shape[:-1]:
        raise ValueError(f"{who}: one label row for each hidden row (got {tuple(index.shape)} for hidden {tuple(hidden.shape)})")
    if bias is not None:
        if bias.dtype not in (torch.float32, weight.dtype) or bias.shape != weight.shape[:1]:
            raise ValueError(f"{who}: bias is [classes] in float32 or the weight's type (got {tuple(bias.shape)}, {bias.dtype})")
        bias = bias.float()
    dev = hidden.device
    for t in (hidden, weight, bias, index, tlog):
        if t is not None and t.device != dev:
            raise ValueError(f"{who}: operands on {dev} and {t.device}")
    if dev.type != "cuda":
        raise L.FeaError(f"{who} runs on a ROCm device only")
    train = torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad))
    if lead.numel() == 0:
        # nothing counts: the loss is 0 and so is every gradient
        zero = (hidden.sum() + weight[:0].sum() + (0 if bias is None else bias[:0].sum())).float() if train else hidden.new_zeros((), dtype=torch.float32)
        return zero if reduction != "none" else zero.expand(lead)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return _linear_loss(who, hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits)
    # Where nothing wants a gradient the call need not become a node (6 of the 20 us that the host takes for a loss), unless forward-mode
    # derivatives may be on the way, which the node refuses
    if train or torch.autograd.forward_ad._current_level >= 0:
        return _LinearLoss.apply(hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits, train)
    return _linear_loss_fwd(hidden, weight, bias, index, tlog, ignore_index, temperature, reduction, keep_logits, 0)[0]


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: torch.Tensor = None,
                         ignore_index: int = -100, reduction: str = "mean", keep_logits: bool = None) -> torch.Tensor:
    """Softmax cross entropy of `hidden @ weight.T + bias` against one label per row.

    hidden [..., D] and weight [classes, D]: both float32 or both bfloat16 (sums, softmax and loss in 32 bits), up to 2^24 classes of
    2^16 features and less than 2^30 rows; target [...] integers; bias [classes], float32 or the weight's type.  Rows whose target is `ignore_index` do not count: loss 0 and
    gradient 0, whatever their hidden state holds.  A target outside [0, classes) makes the loss and the gradients NaN.
    reduction "mean" is over the rows that count (0 if none does), "none" gives a loss for each row.  float32 result.
    Differentiable once, in reverse mode, in hidden, weight and bias.
    keep_logits, in a call that has a backward: True, the forward keeps the logits for it, in 16 bits each (bfloat16; the gradients' shares
    of the softmax are off by 4.9e-4 of themselves, an eighth of their rounding to bfloat16 behind that) or whole in 32 (float32, with a bias
    gradient, up to 64 rows, a split reduction), and an allocation that fails is raised; False, none are kept and the backward computes
    them again in pieces of up to 2^28, which takes a third more products and no memory for all of them; None, they are kept if
    they take 8 GiB or less (FEA_AMD_LINEAR_KEEP: another limit in bytes, 0 for none) and the memory is there.  With True or False the
    gradients are the same from run to run; with None they depend, within these roundings, on whether there was room.
    Few classes of few features (32, 64) are always computed again, which reads no more.
    An NHWC feature map and a 1x1 convolution's weight viewed [classes, channels] are taken as they are."""
    ignore_index = int(ignore_index)
    if not -(1 << 63) <= ignore_index < 1 << 63:
        raise ValueError(f"linear_cross_entropy: ignore_index {ignore_index} is no 64-bit integer")
    return _linear_loss("linear_cross_entropy", hidden, weight, bias, target, None, ignore_index, 1.0, reduction, keep_logits)


def linear_distillation(hidden: torch.Tensor, weight: torch.Tensor, teacher_logits: torch.Tensor, teacher_index: torch.Tensor,
                        bias: torch.Tensor = None, temperature: float = 1.0, reduction: str = "mean", keep_logits: bool = None) -> torch.Tensor:
    """Distillation of `hidden @ weight.T + bias` from a teacher's top logits.

    teacher_logits [..., K] (float32 or bfloat16) and teacher_index [..., K] (integers): the teacher's K (1..256) largest logits of
    a row and their classes; a negative index is no entry.  With p = softmax(teacher_logits / T) over a row's entries and
    q = softmax of all the student's logits / T, the loss of a row is T^2 sum_k p_k (log p_k - log q_{index_k}).  Rows without
    an entry (or with -inf logits alone) do not count.  A class named twice in a row has the sum of both shares; an index
    beyond the classes, a NaN or +inf teacher logit make the loss and the gradients NaN.  The teacher has no gradient.
    hidden, weight, bias, reduction, keep_logits and the result as in `linear_cross_entropy`."""
    who = "linear_distillation"
    if not isinstance(teacher_logits, torch.Tensor) or not isinstance(teacher_index, torch.Tensor):
        raise ValueError(f"{who}: teacher_logits and teacher_index are tensors")
    if teacher_logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{who}: teacher_logits are float32 or bfloat16 (got {teacher_logits.dtype})")
    if teacher_logits.dim() < 1 or teacher_logits.shape != teacher_index.shape or not 1 <= teacher_logits.shape[-1] <= 256:
        raise ValueError(f"{who}: teacher_logits and teacher_index are [..., K] with K from 1 to 256 (got {tuple(teacher_logits.shape)}, "
                         f"{tuple(teacher_index.shape)})")
    temperature = float(temperature)
    if not 1e-3 <= temperature <= 1e3:
        raise ValueError(f"{who}: temperature {temperature} (0.001 to 1000)")
    return _linear_loss(who, hidden, weight, bias, teacher_index, teacher_logits, 0, temperature, reduction, keep_logits)
