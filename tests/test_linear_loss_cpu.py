"""Refusals of the loss heads over many classes, and the oracle's own checks: no GPU is touched."""
import pytest
import torch

from fea_amd import _lib as L
from fea_amd import functional as F
from tests import linear_loss_oracle as O

H, W, T = torch.zeros(4, 8), torch.zeros(5, 8), torch.zeros(4, dtype=torch.int64)
A, I = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)


@pytest.mark.parametrize("bad", [
    {"reduction": "avg"}, {"hidden": H.half(), "weight": W.half()}, {"hidden": H.bfloat16()}, {"weight": W[:, :7]}, {"weight": W[0]},
    {"weight": W[:0]}, {"hidden": H[:, :0], "weight": W[:, :0]}, {"target": T.float()}, {"target": T.bool()}, {"target": T[:3]},
    {"target": T[:, None]}, {"bias": torch.zeros(4)}, {"bias": torch.zeros(5, dtype=torch.float64)}, {"hidden": None}, {"target": None}, {"ignore_index": 1 << 63}])
def test_cross_entropy_refuses(bad):
    kw = {"hidden": H, "weight": W, "target": T} | bad
    with pytest.raises(ValueError, match="linear_cross_entropy"):
        F.linear_cross_entropy(**kw)


@pytest.mark.parametrize("bad", [
    {"temperature": 0.0}, {"temperature": -1.0}, {"temperature": float("nan")}, {"temperature": float("inf")}, {"teacher_logits": A[:, :2]},
    {"teacher_logits": A[:, :0], "teacher_index": I[:, :0]}, {"teacher_logits": A.double()}, {"teacher_index": A},
    {"teacher_logits": A[:3], "teacher_index": I[:3]}, {"teacher_logits": torch.zeros(4, 257), "teacher_index": torch.zeros(4, 257, dtype=torch.int64)},
    {"teacher_logits": None}, {"reduction": "batchmean"}])
def test_distillation_refuses(bad):
    kw = {"hidden": H, "weight": W, "teacher_logits": A, "teacher_index": I} | bad
    with pytest.raises(ValueError, match="linear_distillation"):
        F.linear_distillation(**kw)


def test_no_cpu_path():
    with pytest.raises(L.FeaError, match="ROCm device"):
        F.linear_cross_entropy(H, W, T)
    with pytest.raises(L.FeaError, match="ROCm device"):
        F.linear_distillation(H, W, A, I)


def test_workspace_sizes():
    ws = L.load().fea_linear_loss_ws_bytes
    assert ws(0, 8, 8, 1, 0, 0) == 0 and ws(8, 8, 8, 1, 5, 0) == 0 and ws(8, 8, 8, 0, 0, 7) == 0
    for dt in (L.F32, L.BF16):
        for rows, d, v, k in ((1, 8, 1, 1), (7, 5, 3, 2), (8192, 4096, 131072, 1), (1 << 24, 64, 6, 1), (1 << 20, 64, 100000, 4)):
            assert 0 < ws(rows, d, v, k, dt, 0) < 6 << 30, (rows, d, v)
            sizes = [ws(rows, d, v, k, dt, g) for g in (1, 2, 3, 7)]
            assert sizes[0] <= sizes[2] <= sizes[3] and sizes[1] <= sizes[2], (rows, d, v)
            assert sizes[3] < 24 << 30, (rows, d, v)
            assert 0 < ws(rows, d, v, k, dt, 11) <= max(sizes[3], ws(rows, d, v, k, dt, 3)) * 2


def test_kept_sizes():
    keep = L.load().fea_linear_loss_keep_bytes
    assert keep(0, 8, 8, 0, 0) == 0 and keep(1 << 20, 64, 6, 1, 0) == 0 and keep(100, 64, 1000, 5, 0) == 0
    for wide in (0, 1):
        assert keep(100, 64, 1000, L.F32, wide) == 100 * 1024 * 4
        for dt in (L.F32, L.BF16):
            assert keep(64, 64, 1000, dt, wide) == 64 * 1024 * 4
    assert keep(100, 64, 1000, L.BF16, 1) == 100 * 1024 * 4
    for rows, d, v in ((65, 8, 1), (100, 64, 1000), (8192, 4096, 131072), (1 << 20, 65, 6)):
        ld = (v + 63) // 64 * 64
        assert rows * ld * 4 <= keep(rows, d, v, L.F32, 0) < rows * ld * 4 + 256
        assert rows * ld * 2 < keep(rows, d, v, L.BF16, 0) <= rows * ld * 2 + 256 + rows * ((v + 127) // 128) * 32


@pytest.mark.parametrize("top", [0, 4])
def test_oracle_against_autograd_in_64_bits(top):
    c = O.case(20, 12, 30, torch.float32, seed=1, top=top, ignored=0.2, short=0.3, bias=True)
    got = O.evaluate(*c, temperature=1.0 if not top else 2.0)
    x = [t.double().requires_grad_(True) for t in c[:3]]
    z = x[0] @ x[1].T + x[2]
    if not top:
        loss = torch.nn.functional.cross_entropy(z, c[3])
    else:
        there = c[3] >= 0
        p = torch.softmax(torch.where(there, c[4].double() / 2.0, -1e30), 1) * there
        logq = torch.log_softmax(z / 2.0, 1).gather(1, c[3].clamp(min=0))
        loss = 4.0 * torch.where(there, torch.special.xlogy(p, p) - p * logq, 0.0).sum() / there.any(1).sum()
    for k, g in zip(("hidden", "weight", "bias"), torch.autograd.grad(loss, x)):
        assert torch.allclose(got[k][0], g, rtol=1e-9, atol=1e-12), k
    assert torch.allclose(got["loss"][0], loss, rtol=1e-9)


def test_check_finds_a_planted_error():
    """The comparison the GPU tests rest on: a value beyond its bound, a NaN or an infinity in another place is found."""
    value, bound = torch.tensor([1.0, 2.0], dtype=torch.float64), torch.tensor([1e-3, 1e-3], dtype=torch.float64)
    O.check("x", torch.tensor([1.0005, 2.0]), (value, bound))
    for bad in ([1.002, 2.0], [float("nan"), 2.0], [float("inf"), 2.0]):
        with pytest.raises(AssertionError):
            O.check("x", torch.tensor(bad), (value, bound))


@pytest.mark.parametrize("rows,d,v,db", [(4096, 64, 32, 0), (5000, 8, 2, 0), (100, 64, 1000, 256), (4096, 64, 32, 256)])
def test_entries_without_their_shares_are_refused(rows, d, v, db):
    """A backward over several teacher entries a row that needs the forward's shares and has none.  (The addresses are never used: without
    the refusal the workspace of no bytes is refused.)"""
    at = 1 << 20

    def bwd(k, psel):
        L.call("fea_linear_loss_bwd", at, d, at, d, None, at, k, at, at, psel, None, 1, None, at, 0, 1.0, at, at, db, at, 0, rows, d, v, L.F32, None)
    with pytest.raises(L.FeaError, match="need psel"):
        bwd(3, None)
    for k, psel in ((1, None), (3, at)):
        with pytest.raises(L.FeaError, match="workspace"):
            bwd(k, psel)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", O.ONE_ROW)
def test_one_row_of_any_stride(name, dtype):
    """A single row's stride means nothing (and contiguous() keeps it): the kernels get the features' number, of the same values, without a
    copy where the row lies as they read it."""
    for d in (64, 1024, 5, 1):
        x = torch.randn(d, generator=torch.Generator().manual_seed(1)).to(dtype)
        t = O.one_row(name, x)
        assert t.shape[-1] == d and t.numel() == d
        r = F._aligned_rows(t)
        assert r.shape == (1, d) and r.stride() == (d, 1) and torch.equal(r[0], x)
        if d * x.element_size() % 16 == 0:
            assert r.data_ptr() % 16 == 0
        if t.stride(-1) == 1 and t.data_ptr() % 16 == 0:
            assert r.data_ptr() == t.data_ptr()


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("grad", [True, False])
def test_a_trace_is_refused(grad):
    """torch.jit.trace would record the empty results and no kernel."""
    with torch.set_grad_enabled(grad):
        with pytest.raises(L.FeaError, match="linear_cross_entropy: a trace"):
            torch.jit.trace(lambda h: F.linear_cross_entropy(h, W, T), (H,))
        with pytest.raises(L.FeaError, match="linear_distillation: a trace"):
            torch.jit.trace(lambda h: F.linear_distillation(h, W, A, I), (H,))


@pytest.mark.parametrize("bad", [0, 1, "yes", 1 << 33])
def test_keep_logits_is_a_choice(bad):
    with pytest.raises(ValueError, match="linear_cross_entropy: keep_logits"):
        F.linear_cross_entropy(H, W, T, keep_logits=bad)
    with pytest.raises(ValueError, match="linear_distillation: keep_logits"):
        F.linear_distillation(H, W, A, I, keep_logits=bad)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_norms_find_what_elements_hide(reduction):
    """bfloat16 roundings of dz and of the results alone stay within the norms' bounds; a row lost from the weight's gradient, or dz rounded
    to the bits of an 8-bit type, does not."""
    h, w, _, t = O.case(513, 640, 700, torch.bfloat16, seed=33, ignored=0.1)
    g = torch.randn(513, generator=torch.Generator().manual_seed(1))
    how = {"reduction": reduction, "gout": g if reduction == "none" else None, "kept": False}
    want = O.evaluate(h, w, None, t, norms=True, **how)
    on = t != -100
    p = torch.nn.functional.one_hot(t.clamp(min=0), 700).double()
    g = (g.double() if reduction == "none" else torch.full((513,), 1.0 / int(on.sum()), dtype=torch.float64)) * on
    dz = torch.softmax(h.double() @ w.double().T, 1) - p

    def step(dz):
        dh = g[:, None] * (dz @ w.double())
        dw = dz.T @ (g[:, None] * h.double()).bfloat16().double() if reduction == "none" else (dz * g[:, None]).T @ h.double()
        return dh.bfloat16(), dw.bfloat16()
    dh, dw = step(dz.bfloat16().double())
    O.check_norm("hidden", dh, want["hidden"])
    O.check_norm("weight", dw, want["weight"])
    lost = dz.bfloat16().double()
    lost[int(on.nonzero()[5] if reduction == "mean" else g.abs().argmax())] = 0.0
    with pytest.raises(AssertionError, match="weight"):
        O.check_norm("weight", step(lost)[1], want["weight"])
    m, e = torch.frexp(dz)
    for k, name in enumerate(("hidden", "weight")[:2 if reduction == "mean" else 1]):      # (none: the bound allows for hidden's rounding too)
        with pytest.raises(AssertionError, match=name):
            O.check_norm(name, step(torch.ldexp((m * 4).round() / 4, e))[k], want[name])


@pytest.mark.parametrize("h,w", [((4, 1), ((1 << 24) + 1, 1)), ((4, 1), ((1 << 32) + 5, 1)), ((4, (1 << 16) + 1), (5, (1 << 16) + 1)), ((1 << 30, 1), (5, 1)), ((2, 1 << 30, 3), (5, 3))])
def test_more_than_is_served_is_refused(h, w):
    """Sizes beyond the kernels' (and beyond 32 bits) are refused before anything is allocated, and never cut to 32 bits."""
    x, y = torch.zeros(1).expand(h), torch.zeros(1).expand(w)
    t = torch.zeros(1, dtype=torch.int64).expand(h[:-1])
    with pytest.raises(ValueError, match="linear_cross_entropy: up to"):
        F.linear_cross_entropy(x, y, t)
    with pytest.raises(ValueError, match="linear_distillation: up to"):
        F.linear_distillation(x, y, torch.zeros(1).expand(*h[:-1], 2), t[..., None].expand(*h[:-1], 2))


def test_sizes_that_are_refused_take_no_bytes():
    lib = L.load()
    for rows, d, v, k in ((1 << 30, 8, 8, 1), (8, (1 << 16) + 1, 8, 1), (8, 8, (1 << 24) + 1, 1), (8, 8, (1 << 31) - 1, 1), (8, 8, 8, 257), (-1, 8, 8, 1)):
        for dt in (L.F32, L.BF16):
            assert [lib.fea_linear_loss_ws_bytes(rows, d, v, k, dt, g) for g in (0, 1, 7, 15)] == [0] * 4
            assert k > 1 or lib.fea_linear_loss_keep_bytes(rows, d, v, dt, 0) == 0
    assert lib.fea_linear_loss_ws_bytes(64, 1 << 16, 8, 256, L.F32, 0) > 0 and lib.fea_linear_loss_keep_bytes(64, 8, 1 << 24, L.F32, 0) > 0
