"""linear_cross_entropy and linear_distillation against their definition in 64 bits (tests/linear_loss_oracle.py)."""
import pytest
import torch

from fea_amd import _lib as L
from fea_amd import functional as F
from tests import linear_loss_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16]
SHAPES = [(1, 8, 1), (1, 1, 2), (1, 64, 600), (2, 5, 7), (3, 64, 6), (17, 33, 129), (64, 128, 128), (129, 72, 1000), (5000, 72, 40), (257, 200, 333),
          (300, 96, 5003), (513, 640, 1537), (5000, 64, 6), (4097, 24, 33), (4096, 64, 32), (4100, 33, 13), (6001, 16, 2), (4111, 40, 24), (5003, 7, 1), (33, 515, 1000),
          (48, 1024, 777), (16, 300, 2049), (150, 99, 700), (700, 51, 5000)]


def _leaf(t):
    return None if t is None else t.to(DEV).requires_grad_(True)


def _run(h, w, b, index, tlog=None, gout=None, **how):
    h, w, b = _leaf(h), _leaf(w), _leaf(b)
    if tlog is None:
        loss = F.linear_cross_entropy(h, w, index.to(DEV), bias=b, **how)
    else:
        loss = F.linear_distillation(h, w, tlog.to(DEV), index.to(DEV), bias=b, **how)
    leaves = [t for t in (h, w, b) if t is not None]
    grads = torch.autograd.grad(loss, leaves, None if gout is None else gout.to(DEV))
    return dict(zip(["loss", "hidden", "weight", "bias"], [loss, *grads]))


def _compare(got, want):
    for k, v in got.items():
        O.check(k, v, want[k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_cross_entropy(shape, dtype):
    h, w, b, t = O.case(*shape, dtype, seed=sum(shape), ignored=0.2, bias=shape[0] % 2 == 1)
    _compare(_run(h, w, b, t), O.evaluate(h, w, b, t))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("top", [1, 5, 64])
def test_distillation(shape, dtype, top):
    h, w, b, i, a = O.case(*shape, dtype, seed=sum(shape) + top, top=top, ignored=0.2, short=0.3, bias=shape[0] % 2 == 1)
    _compare(_run(h, w, b, i, a, temperature=2.0), O.evaluate(h, w, b, i, a, temperature=2.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(9, 40, 300), (40, 64, 300), (100, 64, 300), (4200, 16, 30)])
def test_most_entries(shape, dtype):
    """256 teacher entries per row, most classes named more than once."""
    c = O.case(*shape, dtype, seed=31, top=256, ignored=0.1, short=0.2, bias=True)
    _compare(_run(*c, temperature=3.0), O.evaluate(*c, temperature=3.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(100, 2048, 500), (301, 4099, 1000), (200, 6000, 130), (387, 3264, 2112), (65, 3000, 33)])
@pytest.mark.parametrize("top", [0, 3, 256])
def test_few_tiles_split_the_reduction(shape, dtype, top):
    """Long reductions over few tiles of rows and classes, in parts."""
    c = O.case(*shape, dtype, seed=72 + top, top=top, ignored=0.1, short=0.2, bias=shape[0] % 2 == 1)
    _compare(_run(*c), O.evaluate(*c))
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(3))
    _compare(_run(*c, gout=gout, reduction="none"), O.evaluate(*c, gout=gout, reduction="none"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 4096, 5), (17, 1543, 300), (40, 2056, 1000), (64, 20600, 130), (3, 5000, 16000), (30, 3840, 3840)])
@pytest.mark.parametrize("top", [0, 3, 256])
def test_few_rows_and_classes_split_the_reduction(shape, dtype, top):
    """Long reductions over few classes, in parts, with ragged last ones."""
    c = O.case(*shape, dtype, seed=71 + top, top=top, ignored=0.1, short=0.2, bias=shape[0] % 2 == 1)
    _compare(_run(*c), O.evaluate(*c))
    with torch.no_grad():
        x = [None if t is None else t.to(DEV) for t in c]
        loss = F.linear_distillation(x[0], x[1], x[4], x[3], bias=x[2], reduction="none") if top else F.linear_cross_entropy(x[0], x[1], x[3], bias=x[2], reduction="none")
    O.check("loss", loss, O.evaluate(*c, reduction="none")["loss"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,top", [((100, 64, 300), 254), ((100, 64, 300), 255), ((70, 8, 170000), 5), ((300, 72, 2000), 4), ((300, 72, 2000), 40)])
def test_where_the_entries_are(shape, top, dtype):
    """Selected logits out of the product: four entries in a column tile and more, all in one tile, in too many tiles, too many entries."""
    h, w, _, i, a = O.case(*shape, dtype, seed=61, top=top, ignored=0.1, short=0.1)
    i[::3] = i[::3] % 120                                      # all in the first tile
    i[1] = shape[2] - 1                                        # one class, every time
    _compare(_run(h, w, None, i, a, temperature=1.5), O.evaluate(h, w, None, i, a, temperature=1.5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("shape", [(77, 40, 300), (4500, 24, 11)])
def test_reductions(shape, dtype, reduction, top):
    c = O.case(*shape, dtype, seed=5, top=top, ignored=0.2, bias=True)
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(1)) if reduction == "none" else torch.tensor(-3.0)
    kw = {"temperature": 0.5} if top else {}
    _compare(_run(*c, gout=gout, reduction=reduction, **kw), O.evaluate(*c, gout=gout, reduction=reduction, **kw))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 72, 900), (700, 40, 2000)])
@pytest.mark.parametrize("top", [0, 4])
def test_pieces(shape, dtype, top, monkeypatch):
    """Many pieces of the rows (few classes) and of the classes (many): the sums over pieces, in 32 bits."""
    monkeypatch.setenv("FEA_AMD_LINEAR_PIECE", str(1 << 16))
    c = O.case(*shape, dtype, seed=9, top=top, ignored=0.1, short=0.2, bias=True)
    _compare(_run(*c), O.evaluate(*c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(300, 72, 900), (700, 40, 2000), (60, 33, 3000), (513, 643, 1999)])
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("piece", [1 << 16, 1 << 27])
def test_pieces_of_kept_logits(shape, dtype, top, piece, monkeypatch):
    """The same from kept logits, with an upstream gradient for every row."""
    monkeypatch.setenv("FEA_AMD_LINEAR_PIECE", str(piece))
    c = O.case(*shape, dtype, seed=10, top=top, ignored=0.1, short=0.2)
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(2))
    _compare(_run(*c, gout=gout, reduction="none"), O.evaluate(*c, gout=gout, reduction="none"))
    _compare(_run(*c), O.evaluate(*c))


@pytest.mark.parametrize("shape", [(4096, 64, 4096), (4000, 200, 4100), (2049, 1096, 2310), (4097, 72, 8185), (300, 520, 40000), (1300, 643, 2011)])
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("dtype", TYPES)
def test_large_tiles(shape, top, dtype):
    """Sizes that take the 256 x 256 tile (fp32: as planes of bf16) in some or all of their products, with ragged ends in every
    direction."""
    c = O.case(*shape, dtype, seed=3, top=top, ignored=0.1, short=0.2, bias=shape[0] % 2 == 0)
    _compare(_run(*c, reduction="sum"), O.evaluate(*c, reduction="sum"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 64, 600), (33, 515, 1000), (64, 128, 130), (65, 8, 64), (130, 33, 257), (258, 200, 333), (514, 640, 1537), (2050, 1096, 2310)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("keep", [0, 1 << 30])
def test_logits_kept_or_recomputed(shape, dtype, top, keep, bias, monkeypatch):
    """A head keeps its logits for the backward, within a limit; recomputed ones hold the same bounds."""
    monkeypatch.setenv("FEA_AMD_LINEAR_KEEP", str(keep))
    c = O.case(*shape, dtype, seed=sum(shape) + 1, top=top, ignored=0.2, short=0.3, bias=bias)
    _compare(_run(*c), O.evaluate(*c))
    x = [_leaf(t) for t in c[:3] if t is not None]
    b = x[2] if bias else None
    loss = F.linear_distillation(*x[:2], c[4].to(DEV), c[3].to(DEV), bias=b) if top else F.linear_cross_entropy(*x[:2], c[3].to(DEV), bias=b)
    held = [t.numel() for t in loss.grad_fn.saved_tensors if t is not None and t.dtype == torch.uint8]
    assert [n >= shape[0] * shape[2] * (c[0].element_size() if shape[0] > 64 and not bias else 4) for n in held] == [True] * (keep > 0)
    want = torch.autograd.grad(loss, x, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, x), want))


def test_no_room_for_the_logits(monkeypatch):
    """Where the logits find no room the backward recomputes them."""
    c = O.case(300, 64, 700, torch.float32, seed=52, ignored=0.1)
    n = L.load().fea_linear_loss_keep_bytes(300, 64, 700, L.F32, 0)
    empty, asked = torch.empty, []

    def full(*size, **how):
        if size == (n,) and how.get("dtype") == torch.uint8:
            asked.append(n)
            raise torch.cuda.OutOfMemoryError("no room")
        return empty(*size, **how)
    monkeypatch.setattr(torch, "empty", full)
    got = _run(*c)
    assert asked == [n]
    _compare(got, O.evaluate(*c))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.02])
def test_logits_far_apart(dtype, temperature):
    """Logits that lie hundreds below their tile's largest count as a share of 0, others down to e^-64 as they are."""
    h, w, _, i, a = O.case(200, 64, 700, dtype, seed=50, top=4, ignored=0.1, short=0.2)
    h = (h.float() * torch.logspace(0, 1.5, 200)[:, None]).to(dtype)
    _compare(_run(h, w, None, i, a, temperature=temperature), O.evaluate(h, w, None, i, a, temperature=temperature))


def test_far_kept_logits(monkeypatch):
    """More than 2^31 kept logits, from two chunks of the rows, against recomputed ones.  Either side's shares of the softmax are off by 2^-8 and
    4.9e-4 of themselves at most; a row's shares and its label's add up to 2 at most, and the fp32 sums over a million classes to 1e-3 of that."""
    g = torch.Generator().manual_seed(51)
    rows, v, d = 2400, 1000003, 16
    h, w = torch.randn(rows, d, generator=g).bfloat16(), torch.randn(v, d, generator=g).bfloat16()
    t = torch.randint(0, v, (rows,), generator=g)
    assert rows * v > 1 << 31
    kept = _run(h, w, None, t, reduction="sum")
    monkeypatch.setenv("FEA_AMD_LINEAR_KEEP", "0")
    again = _run(h, w, None, t, reduction="sum")
    assert torch.equal(kept["loss"], again["loss"])
    top = float(w.float().abs().max())
    off = (kept["hidden"].float() - again["hidden"].float()).abs()
    assert bool((off <= 2 * (2 * 2.0 ** -8 + 4.9e-4 + 1e-3) * top + 2 * 2.0 ** -8 * again["hidden"].float().abs()).all())
    # a class's gradient: its shares of all rows, at most 2 |h| of its labels' rows in sum; classes that no label names are compared to their own size
    free = torch.ones(v, dtype=torch.bool)
    free[t] = False
    a, b = kept["weight"].float().cpu()[free], again["weight"].float().cpu()[free]
    q = torch.zeros(v, dtype=torch.float64)
    for k in range(0, rows, 240):
        z = h[k:k + 240].float() @ w.float().T
        q += torch.softmax(z, 1).double().sum(0)
    bound = q[free].float()[:, None] * float(h.float().abs().max()) * (2 * 2.0 ** -8 + 4.9e-4 + 1e-3) + 2 * 2.0 ** -8 * b.abs()
    assert bool(((a - b).abs() <= bound).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [9, 4100])
def test_nothing_counts(dtype, rows):
    h, w, b, t = O.case(rows, 16, 20, dtype, bias=True)
    got = _run(h, w, b, torch.full_like(t, -100))
    assert all(float(v.detach().abs().max()) == 0.0 for v in got.values())
    i = torch.full((rows, 3), -1)
    got = _run(h, w, b, i, torch.zeros(rows, 3, dtype=dtype))
    assert all(float(v.detach().abs().max()) == 0.0 for v in got.values())
    got = _run(h, w, b, torch.zeros(rows, 3, dtype=torch.int64), torch.full((rows, 3), -torch.inf, dtype=dtype))
    assert all(float(v.detach().abs().max()) == 0.0 for v in got.values())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("shape", [(70, 64, 200), (4200, 64, 7)])
def test_ignored_rows_may_hold_anything(shape, dtype, top, bad):
    """The hidden state of a row that does not count reaches neither the loss nor any gradient."""
    c = list(O.case(*shape, dtype, seed=3, top=top, ignored=0.4, bias=True))
    want = O.evaluate(*c)
    gone = c[3] == -100 if not top else (c[3] < 0).all(1)
    assert 5 < int(gone.sum()) < shape[0] - 5
    c[0] = c[0].clone()
    c[0][gone] = bad
    _compare(_run(*c), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -1e30])
def test_ignored_rows_of_kept_logits_may_hold_anything(dtype, top, bad):
    c = list(O.case(90, 64, 200, dtype, seed=3, top=top, ignored=0.4))
    want = O.evaluate(*c)
    gone = c[3] == -100 if not top else (c[3] < 0).all(1)
    assert 5 < int(gone.sum()) < 85
    c[0] = c[0].clone()
    c[0][gone] = bad
    _compare(_run(*c), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_classes_of_kept_logits(dtype):
    """A bias without a gradient masks classes: their kept logits are a share of 0, and gradient 0."""
    h, w, b, t = O.case(65, 48, 400, dtype, seed=4, bias=True)
    b[100:228] = -torch.inf
    b[256:384] = torch.finfo(torch.float32).min
    t = t % 100
    want = O.evaluate(h, w, b, t)
    x, y = _leaf(h), _leaf(w)
    loss = F.linear_cross_entropy(x, y, t.to(DEV), bias=b.to(DEV))
    assert any(s is not None and s.dtype == torch.uint8 for s in loss.grad_fn.saved_tensors)
    gh, gw = torch.autograd.grad(loss, [x, y])
    assert float(gw[100:228].abs().max()) == 0.0 and float(gw[256:384].abs().max()) == 0.0
    kept = O.evaluate(h, w, b, t, kept=True)
    _compare({"loss": loss, "hidden": gh, "weight": gw}, kept)
    assert torch.equal(kept["hidden"][0], want["hidden"][0])


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_classes(dtype):
    """Classes masked by a bias of -inf or of the type's lowest value: softmax 0 and gradient 0 there."""
    h, w, b, t = O.case(65, 48, 400, dtype, seed=4, bias=True)
    b[100:228] = -torch.inf                                  # the whole of a column tile and parts of its neighbours
    b[256:384] = torch.finfo(torch.float32).min
    t = t % 100
    got = _run(h, w, b, t)
    _compare(got, O.evaluate(h, w, b, t))
    assert float(got["weight"][100:228].abs().max()) == 0.0 and float(got["bias"][256:384].abs().max()) == 0.0
    h, w, b, t = O.case(4100, 48, 9, dtype, seed=4, bias=True)
    b[3], b[8] = -torch.inf, torch.finfo(torch.float32).min
    t = t % 3
    got = _run(h, w, b, t)
    _compare(got, O.evaluate(h, w, b, t))
    assert float(got["weight"][3].abs().max()) == 0.0 and float(got["bias"][8]) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_teacher_minus_infinity_is_no_share(dtype):
    h, w, b, i, a = O.case(40, 32, 90, dtype, seed=6, top=6)
    a[:, 2] = -torch.inf
    a[7] = -torch.inf
    _compare(_run(h, w, b, i, a), O.evaluate(h, w, b, i, a))


@pytest.mark.parametrize("rows", [10, 4100])
def test_a_label_that_names_no_class_is_nan(rows):
    h, w, b, t = O.case(rows, 32, 20, torch.float32, seed=7)
    for bad in (20, 1 << 40, -5):
        x = t.clone()
        x[4] = bad
        loss = F.linear_cross_entropy(h.to(DEV), w.to(DEV), x.to(DEV), reduction="none")
        want = O.evaluate(h, w, b, t, reduction="none")["loss"][0]
        rest = torch.arange(rows) != 4
        assert torch.isnan(loss[4]) and torch.allclose(loss.cpu().double()[rest], want[rest], rtol=1e-5)
    h, w, b, i, a = O.case(rows, 32, 20, torch.float32, seed=7, top=3)
    i[2, 1] = 20
    a[5, 0] = torch.nan
    a[6, 2] = torch.inf
    got = _run(h, w, b, i, a, reduction="none", gout=torch.ones(rows))
    assert torch.isnan(got["loss"]).nonzero().flatten().tolist() == [2, 5, 6]
    assert torch.isnan(got["hidden"]).all(1).nonzero().flatten().tolist() == [2, 5, 6]


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Strided rows, odd storage offsets, leading dimensions, an expanded hidden state, other integer types, views of a 1x1
    convolution's weight: the same values as contiguous ones."""
    h, w, b, t = O.case(60, 64, 150, dtype, seed=8, ignored=0.1, bias=True)
    want = _run(h, w, b, t)
    wide = torch.zeros(60, 200, dtype=dtype)
    wide[:, 3:67] = h
    tall = torch.zeros(151 * 64 + 1, dtype=dtype)
    tall[1:1 + 150 * 64] = w.reshape(-1)
    for x in (_leaf(wide)[:, 3:67], _leaf(h.t().contiguous()).t(), _leaf(h).reshape(3, 4, 5, 64)):
        y = _leaf(tall)[1:1 + 150 * 64].view(150, 64, 1, 1).view(150, 64)
        for kind in (torch.int64, torch.int32, torch.int16):
            loss = F.linear_cross_entropy(x, y, t.to(DEV).to(kind).reshape(x.shape[:-1]), bias=b.to(DEV))
            gx, gy = torch.autograd.grad(loss, [x, y])
            assert torch.equal(loss, want["loss"]) and torch.equal(gx.reshape(60, 64), want["hidden"]) and torch.equal(gy, want["weight"])
    u8 = t.clamp(min=0)
    loss = F.linear_cross_entropy(h.to(DEV), w.to(DEV), u8.to(torch.uint8).to(DEV), ignore_index=0, reduction="sum")
    O.check("loss", loss, O.evaluate(h, w, None, u8, ignore_index=0, reduction="sum")["loss"])
    one = _leaf(h[:1])
    loss = F.linear_cross_entropy(one.expand(60, 64), w.to(DEV), t.to(DEV), reduction="sum")
    ref = O.evaluate(h[:1].expand(60, 64), w, None, t, reduction="sum")
    O.check("loss", loss, ref["loss"])
    g = torch.autograd.grad(loss, one)[0].double().cpu()
    tol = ref["hidden"][1].sum(0) + 60 * torch.finfo(dtype).eps / 2 * ref["hidden"][0].abs().sum(0)
    assert bool(((g - ref["hidden"][0].sum(0)).abs() <= tol).all())
    bare = F.linear_cross_entropy(h[0].to(DEV), w.to(DEV), t[0].to(DEV))
    assert bare.shape == () and torch.equal(bare, F.linear_cross_entropy(h[:1].to(DEV), w.to(DEV), t[:1].to(DEV)))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_something_very_wide(dtype):
    """Rows further apart than a buffer load's 32-bit offsets reach over a tile."""
    h, w, b, t = O.case(70, 64, 300, dtype, seed=8, ignored=0.1, bias=True)
    want = O.evaluate(h, w, b, t)
    for n in range(2):
        rows = [h, w]
        wide = torch.zeros(rows[n].shape[0], (1 << 21) + 8, dtype=dtype, device=DEV)
        wide[:, 8:72] = rows[n].to(DEV)
        rows = [x.to(DEV) for x in rows]
        rows[n] = wide[:, 8:72]
        rows = [x.detach().requires_grad_(True) for x in rows]
        loss = F.linear_cross_entropy(rows[0], rows[1], t.to(DEV), bias=b.to(DEV))
        _compare(dict(zip(("loss", "hidden", "weight"), [loss, *torch.autograd.grad(loss, rows)])), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 65536, 50), (70, 65536, 40), (2, 1, 1 << 24), (66, 2, 1 << 20)])
def test_longest_and_widest(shape, dtype):
    """The most features, the most classes."""
    c = O.case(*shape, dtype, seed=80, ignored=0.1)
    _compare(_run(*c), O.evaluate(*c))


def test_far_rows():
    """More than 2^31 elements of hidden states: 8,300 copies of a batch, whose rows do not depend on each other."""
    h, w, b, t = O.case(4096, 64, 6, torch.bfloat16, seed=40, ignored=0.1, bias=True)
    base = _run(h, w, b, t, reduction="sum")
    n = 8300
    assert n * h.numel() > 1 << 31
    far = _run(h.to(DEV).repeat(n, 1), w, b, t.to(DEV).repeat(n), reduction="sum")
    assert torch.equal(far["hidden"].view(n, 4096, 64)[-1], base["hidden"]) and torch.equal(far["hidden"].view(n, 4096, 64)[n // 2], base["hidden"])
    # sums of n equal parts: in 32 bits per workgroup, in 64 across, rounded once
    for k, u in (("loss", 1e-5), ("weight", 2.0 ** -8 + 1e-5), ("bias", 1e-5)):
        want = O.evaluate(h, w, b, t, reduction="sum")[k]
        O.check(k, far[k] / n, (want[0], want[1] + u * want[0].abs() + 1e-5 * want[0].abs().max()))


def test_far_classes():
    """More than 2^31 elements of weight: 100 copies of 5,300 classes, labels among the last copy.  Each copy has a hundredth of the softmax."""
    h, w, _, t = O.case(70, 4096, 5300, torch.bfloat16, seed=41)
    n = 100
    assert n * w.numel() > 1 << 31
    base = O.evaluate(h, w, None, t, reduction="none")
    x, y = _leaf(h), w.to(DEV).repeat(n, 1).requires_grad_(True)
    loss = F.linear_cross_entropy(x, y, (t + (n - 1) * 5300).to(DEV), reduction="none")
    gh, gw = torch.autograd.grad(loss.sum(), [x, y])
    import math
    O.check("loss", loss, (base["loss"][0] + math.log(n), base["loss"][1] + 4e-6))
    # the copies' weights are equal, so dh is the base's; its sum runs over n times as many terms
    O.check("hidden", gh, (base["hidden"][0], base["hidden"][1] * 1.5 + n * 5300 * O.E * base["hidden"][0].abs().mean()))
    q = torch.softmax(h.double() @ w.double().T, 1)
    free = q.T @ h.double() / n
    bound = (q.T @ h.double().abs()) / n * 2.0 ** -6 + free.abs() * 2.0 ** -8
    for k in (0, n // 2, n - 2):
        O.check(f"copy {k}", gw[k * 5300:(k + 1) * 5300], (free, bound))
    last = free.clone()
    last.index_add_(0, t, -h.double())
    hot = torch.zeros_like(bound).index_add_(0, t, h.double().abs())
    O.check("the labels' copy", gw[(n - 1) * 5300:], (last, bound + 2.0 ** -6 * hot))


def test_only_the_gradients_that_are_wanted():
    c = O.case(50, 64, 200, torch.bfloat16, seed=2, bias=True)
    want = _run(*c)
    for names in (["hidden"], ["weight"], ["bias"], ["weight", "bias"]):
        x = {k: v.to(DEV).requires_grad_(k in names) for k, v in zip(("hidden", "weight", "bias"), c)}
        loss = F.linear_cross_entropy(x["hidden"], x["weight"], c[3].to(DEV), bias=x["bias"])
        for k, g in zip(names, torch.autograd.grad(loss, [x[k] for k in names])):
            assert torch.equal(g, want[k]), (names, k)
    with torch.no_grad():
        loss = F.linear_cross_entropy(x["hidden"], x["weight"], c[3].to(DEV), bias=x["bias"])
    assert not loss.requires_grad and torch.equal(loss, want["loss"])


def test_bf16_bias_and_empty_batch():
    h, w, b, t = O.case(20, 32, 64, torch.bfloat16, seed=2, bias=True)
    b = b.bfloat16()
    x = _leaf(b)
    loss = F.linear_cross_entropy(h.to(DEV), w.to(DEV), t.to(DEV), bias=x)
    g = torch.autograd.grad(loss, x)[0]
    ref = O.evaluate(h, w, b, t)
    assert g.dtype == torch.bfloat16
    O.check("bias", g, (ref["bias"][0], ref["bias"][1] + 2.0 ** -8 * ref["bias"][0].abs()))
    e, w = _leaf(h[:0]), _leaf(w)
    for loss in (F.linear_cross_entropy(e, w, t[:0].to(DEV)), F.linear_distillation(e, w, h[:0, :4].to(DEV), t[:0, None].expand(0, 4).to(DEV))):
        gh, gw = torch.autograd.grad(loss, [e, w])
        assert float(loss.detach()) == 0.0 and gh.shape == (0, 32) and float(gw.abs().max()) == 0.0
    assert F.linear_cross_entropy(e, w, t[:0].to(DEV), reduction="none").shape == (0,)


@pytest.mark.parametrize("top", [0, 2])
def test_gradient_against_differences(top):
    """Central differences of the fp32 loss along a direction.  The step's cubic term is below (0.02)^2 of the slope; the two losses
    are off by 1e-6 each, over 2 x 0.02."""
    c = O.case(30, 24, 70, torch.float32, seed=11, top=top, ignored=0.1, bias=True)
    kw = {"temperature": 1.5} if top else {}
    got = _run(*c, **kw)
    g = torch.Generator().manual_seed(3)
    for k, name in enumerate(["hidden", "weight", "bias"]):
        d = torch.randn(c[k].shape, generator=g)
        d /= d.norm()
        step = 0.02
        pair = []
        for sign in (1, -1):
            x = list(c)
            x[k] = x[k] + sign * step * d
            pair.append(float(_run(*x, **kw)["loss"].detach()))
        slope = float((got[name].cpu() * d).sum())
        curve = float(O.evaluate(*c, **kw)[name][0].norm())
        assert abs((pair[0] - pair[1]) / (2 * step) - slope) <= 2e-6 / (2 * step) + 4e-4 * max(curve, 1.0), name


def test_same_result_every_time_and_on_another_stream():
    c = O.case(700, 64, 1200, torch.bfloat16, seed=12, top=4, bias=True)
    want = _run(*c)
    s = torch.cuda.Stream()
    for _ in range(3):
        got = _run(*c)
        with torch.cuda.stream(s):
            other = _run(*c)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]) and torch.equal(other[k], want[k]), k


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [0, 3])
def test_kept_logits_captured_and_on_other_streams(dtype, top):
    """Two steps at once on two streams, and a captured one replayed with other inputs, each with its own kept logits."""
    cases = [O.case(300, 64, 700, dtype, seed=s, top=top, ignored=0.1) for s in (1, 2, 3)]
    kw = {"temperature": 2.0} if top else {}
    wants = [_run(*c, **kw) for c in cases]
    torch.cuda.synchronize()
    streams, gots = [torch.cuda.Stream() for _ in cases], []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            gots.append(_run(*c, **kw))
    torch.cuda.synchronize()
    for got, want in zip(gots, wants):
        assert all(torch.equal(got[k], want[k]) for k in want)
    x = [None if t is None else t.to(DEV) for t in cases[0]]
    for t in x[:2]:
        t.requires_grad_(True)

    def step():
        loss = F.linear_distillation(x[0], x[1], x[4], x[3], **kw) if top else F.linear_cross_entropy(x[0], x[1], x[3])
        assert any(t is not None and t.dtype == torch.uint8 for t in loss.grad_fn.saved_tensors)
        return [loss.detach(), *torch.autograd.grad(loss, x[:2])]

    with torch.cuda.stream(streams[0]):
        step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for c, want in list(zip(cases, wants))[::-1] + [(cases[0], wants[0])]:
        with torch.no_grad():
            for dst, src in zip(x, c):
                if dst is not None:
                    dst.copy_(src.to(DEV))
        g.replay()
        other = _run(*cases[1], **kw)                       # the program's own work in between
        torch.cuda.synchronize()
        assert all(torch.equal(a, want[k]) for a, k in zip(out, ("loss", "hidden", "weight")))
        assert all(torch.equal(other[k], wants[1][k]) for k in other)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_logits_kept_or_not(dtype, monkeypatch):
    """A class at +inf has no softmax (inf - inf): the loss and the gradients it reaches are NaN, kept or recomputed."""
    h, w, b, t = O.case(130, 64, 300, dtype, seed=5, bias=True)
    b[200] = torch.inf
    got = []
    for keep in ("0", str(1 << 30)):
        monkeypatch.setenv("FEA_AMD_LINEAR_KEEP", keep)
        x, y = _leaf(h), _leaf(w)
        loss = F.linear_cross_entropy(x, y, t.to(DEV), bias=b.to(DEV), reduction="sum")
        got.append([loss.detach(), *torch.autograd.grad(loss, [x, y])])
    assert bool(torch.isnan(got[0][0]))
    for a, c in zip(*got):
        assert torch.equal(torch.isnan(a), torch.isnan(c))


@pytest.mark.parametrize("top", [0, 3])
def test_captured_and_replayed(top):
    """Forward and backward in one captured graph, replayed with other inputs, the program's own work in between; a second graph
    of the same operator keeps its own workspaces."""
    cases = [O.case(130, 64, 500, torch.bfloat16, seed=s, top=top, ignored=0.1, bias=True) for s in (1, 2, 3)]
    graphs = []
    for n in range(2):
        x = [t.to(DEV) for t in cases[0]]
        for t in x[:3]:
            t.requires_grad_(True)

        def step():
            loss = F.linear_distillation(x[0], x[1], x[4], x[3], bias=x[2]) if top else F.linear_cross_entropy(x[0], x[1], x[3], bias=x[2])
            return [loss.detach(), *torch.autograd.grad(loss, x[:3])]

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, x, out))
    for c in cases + cases[:1]:
        want = _run(*c)
        for g, x, out in graphs:
            with torch.no_grad():
                for dst, src in zip(x, c):
                    dst.copy_(src.to(DEV))
        for g, x, out in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, x, out in graphs:
            for k, v in zip(("loss", "hidden", "weight", "bias"), out):
                assert torch.equal(v, want[k]), k


def test_together_in_a_training_loop():
    """Labels and a teacher together on one head, as a distillation step uses them: both losses, one backward, an optimizer step;
    against the same step from the definition's gradients."""
    h, w, b, t = O.case(200, 64, 300, torch.float32, seed=21, ignored=0.2, bias=True)
    i, a = O.case(200, 64, 300, torch.float32, seed=22, top=8, short=0.2)[3:]
    head = torch.nn.Linear(64, 300).to(DEV)
    with torch.no_grad():
        head.weight.copy_(w)
        head.bias.copy_(b)
    opt = torch.optim.SGD(head.parameters(), lr=0.5)
    x = h.to(DEV).requires_grad_(True)
    loss = 0.3 * F.linear_cross_entropy(x, head.weight, t.to(DEV), bias=head.bias) \
        + 0.7 * F.linear_distillation(x, head.weight, a.to(DEV), i.to(DEV), bias=head.bias, temperature=2.0)
    loss.backward()
    opt.step()
    p, q = O.evaluate(h, w, b, t), O.evaluate(h, w, b, i, a, temperature=2.0)

    def both(k):
        return 0.3 * p[k][0] + 0.7 * q[k][0], 0.3 * p[k][1] + 0.7 * q[k][1] + 4 * O.E * (p[k][0].abs() + q[k][0].abs())
    O.check("loss", loss, both("loss"))
    O.check("hidden", x.grad, both("hidden"))
    for name, now, start in (("weight", head.weight, w), ("bias", head.bias, b)):
        value, bound = both(name)
        O.check(name, now, (start.double() - 0.5 * value, 0.5 * bound + 2 * O.E * (start.double().abs() + value.abs())))


def test_double_backward_is_refused():
    h, w, b, t = O.case(5, 16, 9, torch.float32)
    x = _leaf(h)
    g = torch.autograd.grad(F.linear_cross_entropy(x, w.to(DEV), t.to(DEV)), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_change_in_place_between_forward_and_backward_is_refused():
    h, w, b, t = O.case(5, 16, 9, torch.float32)
    x, y = _leaf(h), _leaf(w)
    loss = F.linear_cross_entropy(x, y, t.to(DEV))
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_workspace_and_operands_are_checked():
    """The C entry points refuse what they cannot serve, before any launch."""
    h, w, _, t = O.case(16, 32, 40, torch.float32)
    h, w, t = h.to(DEV), w.to(DEV), t.to(DEV)
    n = L.load().fea_linear_loss_ws_bytes(16, 32, 40, 1, L.F32, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    out = torch.empty(16, device=DEV)

    def fwd(h=h, ldh=32, ws=ws, n=n, rows=16, d=32, v=40, dt=L.F32, keep=None):
        L.call("fea_linear_ce_fwd", h, ldh, w, 32, None, t, -100, None, None, keep, 0, out, None, None, 0, ws, n, rows, d, v, dt, L.stream_ptr())
    fwd()
    for bad in ({"n": n - 1}, {"ws": None}, {"ldh": 31}, {"ldh": 33}, {"h": None}, {"dt": 7}, {"rows": 0}, {"v": 0}, {"d": 0}, {"h": h.data_ptr() + 4},
                {"ws": ws.data_ptr() + 16}, {"d": 1 << 17, "ldh": 1 << 17}, {"keep": ws.data_ptr() + 64}):
        with pytest.raises(L.FeaError):
            fwd(**bad)
    far = torch.zeros(1, device=DEV)                        # (refused before anything is read)
    with pytest.raises(L.FeaError, match="strides"):
        fwd(h=far, ldh=1 << 21, dt=L.BF16)
    n = L.load().fea_linear_loss_keep_bytes(80, 32, 40, L.BF16, 0)
    keep, back = torch.empty(n, dtype=torch.uint8, device=DEV), torch.empty(1 << 24, dtype=torch.uint8, device=DEV)
    x = torch.zeros(80, 32, dtype=torch.bfloat16, device=DEV)
    f = torch.zeros(160, device=DEV)
    for kp, db in ((keep, f), (keep.data_ptr() + 64, None)):
        with pytest.raises(L.FeaError, match="kept"):
            L.call("fea_linear_loss_bwd", x, 32, x, 32, None, t.repeat(5), 1, f, f, None, kp, 0, None, f, 0, 1.0, x, None, db, back, back.numel(), 80, 32, 40,
                   L.BF16, L.stream_ptr())
    torch.cuda.synchronize()


def _entry_step(h, w, b, index, tlog=None, gout=None, temperature=1.0, kept=True, shares=True):
    """A step through the C entry points: mean loss and count out of the forward, then the backward with both a count and an upstream
    gradient for every row.  {"loss", "count", "hidden", "weight", "bias"}."""
    (rows, d), v, k, dt = h.shape, w.shape[0], 1 if tlog is None else index.shape[1], L.dt_code(h.dtype)
    h, w, index, gout = h.to(DEV), w.to(DEV), index.to(DEV), gout.to(DEV)
    b = None if b is None else b.to(DEV)
    wide = int(b is not None)
    stat, dsel, psel = (torch.empty(rows, n, device=DEV) for n in (2, k, k))
    n = L.load().fea_linear_loss_keep_bytes(rows, d, v, dt, wide) if kept else 0
    keep = torch.empty(n, dtype=torch.uint8, device=DEV) if n else None
    loss, count = torch.empty((), device=DEV), torch.empty((), dtype=torch.int32, device=DEV)
    n = L.load().fea_linear_loss_ws_bytes(rows, d, v, k, dt, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    rest = (keep, wide, None, loss, count, 1, ws, n, rows, d, v, dt, L.stream_ptr())
    if tlog is None:
        L.call("fea_linear_ce_fwd", h, d, w, d, b, index, -100, stat, dsel, *rest)
    else:
        tlog = tlog.to(DEV)
        L.call("fea_linear_kd_fwd", h, d, w, d, b, tlog, L.dt_code(tlog.dtype), index, k, temperature, stat, dsel, psel, *rest)
    dh, dw, db = torch.empty_like(h), torch.empty_like(w), None if b is None else torch.empty(v, device=DEV)
    n = L.load().fea_linear_loss_ws_bytes(rows, d, v, k, dt, 3 + 4 * wide + 8 * (keep is not None))
    ws = torch.empty(n, dtype=torch.uint8, device=DEV)
    L.call("fea_linear_loss_bwd", h, d, w, d, b, index, k, stat, dsel, psel if shares and tlog is not None else None, keep, wide, count, gout, 1, temperature, dh, dw, db,
           ws, n, rows, d, v, dt, L.stream_ptr())
    torch.cuda.synchronize()
    return {"loss": loss, "count": count, "hidden": dh, "weight": dw} | ({} if b is None else {"bias": db})


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(40, 64, 300), (200, 72, 500), (200, 51, 500), (1300, 643, 2011), (4100, 24, 9)])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("kept", [True, False])
def test_count_divides_every_gradient(shape, dtype, top, kept):
    """A count beside an upstream gradient for every row: hidden's, weight's and bias's gradients are all divided by it."""
    c = O.case(*shape, dtype, seed=91 + top, top=top, ignored=0.2, bias=shape[0] % 2 == 0 and not (kept and shape[0] == 200))
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(4))
    got = _entry_step(*c, gout=gout, temperature=2.0 if top else 1.0, kept=kept)
    on = int((c[3] != -100).sum()) if not top else int((c[3] >= 0).any(1).sum())
    assert int(got.pop("count")) == on
    kw = {"temperature": 2.0} if top else {}
    mean = O.evaluate(*c, **kw)
    want = O.evaluate(*c, gout=gout / on, reduction="none", kept=None if kept else False, **kw)        # (T is a power of two: the order of T and the division is free)
    want["loss"] = mean["loss"]
    _compare(got, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(40, 64, 300), (200, 51, 500), (4095, 64, 32)])
@pytest.mark.parametrize("kept", [True, False])
def test_entries_without_their_shares(shape, dtype, kept):
    """Without a bias gradient and with more than a few classes the backward takes the selected entries from dsel alone."""
    c = O.case(*shape, dtype, seed=95, top=5, ignored=0.2, short=0.2)
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(5))
    want, got = (_entry_step(*c, gout=gout, kept=kept, shares=s) for s in (True, False))
    assert all(torch.equal(got[k], want[k]) for k in want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(70, 64, 200), (4200, 64, 7)])
@pytest.mark.parametrize("temperature", [0.02, 0.5, 1.0, 4.0])
def test_teacher_logits_at_the_ends_of_the_type(shape, dtype, temperature):
    """Entries masked by the type's lowest value have no share beside others; alone in a row they are equals and it counts, as are equal
    ones at the largest value.  The definition does not change when a row's logits move together: the bounds are those of zeros."""
    h, w, b, i, a = O.case(*shape, dtype, seed=17, top=4, ignored=0.1, short=0.1, bias=True)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    mask = torch.rand(a.shape, generator=torch.Generator().manual_seed(18)) < 0.3
    mask[5], mask[6] = True, False
    i[5:8] = torch.tensor([[1, 2, -1, 4], [0, 2, 3, -1], [3, 1, 2, 0]])
    a[6], mask[7] = high, torch.tensor([True, True, True, False])
    same = a.masked_fill(mask, -torch.inf)
    alone = (mask | (i < 0)).all(1) & (i >= 0).any(1)               # only masked entries
    assert bool(alone[5]) and not bool(alone[7])
    same[alone], same[6] = 0.0, 0.0
    a = a.masked_fill(mask, low).masked_fill(i < 0, torch.nan)      # (no entry, whatever the logit holds)
    same = same.masked_fill(i < 0, 0.0)
    want = O.evaluate(h, w, b, i, same, temperature=temperature, reduction="none")
    gout = torch.ones(shape[0])
    _compare(_run(h, w, b, i, a, temperature=temperature, reduction="none", gout=gout), want)
    _compare(_run(h, w, b, i, a, temperature=temperature), O.evaluate(h, w, b, i, same, temperature=temperature))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", O.ONE_ROW)
@pytest.mark.parametrize("dim", [64, 51])
def test_one_row_or_one_class_of_any_stride(name, dim, dtype):
    """The score and the gradients of one hidden state, and of many over one class, whatever the single row's stride."""
    for rows, classes in ((1, 300), (70, 1), (1, 1)):
        h, w, b, t = O.case(rows, dim, classes, dtype, seed=24, bias=True)
        want = O.evaluate(h, w, b, t)
        x, y, b = h.to(DEV), w.to(DEV), b.to(DEV)
        x = O.one_row(name, x[0]) if rows == 1 else x
        y = O.one_row(name, y[0]) if classes == 1 else y
        O.check("loss", F.linear_cross_entropy(x, y, t.to(DEV), bias=b), want["loss"])
        leaves = [v.detach().requires_grad_(True) for v in (x, y, b)]
        assert leaves[0].stride() == x.stride() and leaves[1].stride() == y.stride()
        loss = F.linear_cross_entropy(*leaves[:2], t.to(DEV), bias=leaves[2])
        _compare(dict(zip(("loss", "hidden", "weight", "bias"), [loss, *torch.autograd.grad(loss, leaves)])), want)
        i, a = t[:, None].to(DEV), torch.zeros(rows, 1, device=DEV)
        assert torch.equal(F.linear_distillation(x, y, a, i, bias=b), loss.detach())


@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(top, grad):
    """A tangent of hidden, weight or bias is refused, not dropped, whether gradients are recorded or not; a call without one is served."""
    c = [t.to(DEV) for t in O.case(9, 16, 30, torch.float32, top=top, bias=True)]

    def loss(h, w, b):
        return F.linear_distillation(h, w, c[4], c[3], bias=b) if top else F.linear_cross_entropy(h, w, c[3], bias=b)
    want = loss(*c[:3])
    with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
        assert torch.equal(loss(*c[:3]), want)
        for k in range(3):
            x = list(c[:3])
            x[k] = torch.autograd.forward_ad.make_dual(x[k], torch.ones_like(x[k]))
            with pytest.raises(NotImplementedError):
                loss(*x)


def _kept(loss):
    return any(t is not None and t.dtype == torch.uint8 for t in loss.grad_fn.saved_tensors)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(33, 64, 500), (300, 72, 700), (200, 51, 500)])
@pytest.mark.parametrize("top", [0, 3])
def test_keep_logits_decides(shape, dtype, top, monkeypatch):
    """keep_logits = True and False whatever the limit is, with the gradients of a limit that allows them and of none, and either within the
    bounds."""
    c = O.case(*shape, dtype, seed=28, top=top, ignored=0.1)
    x = [t.to(DEV).requires_grad_(True) for t in c[:2]]

    def step(**how):
        loss = F.linear_distillation(*x, c[4].to(DEV), c[3].to(DEV), **how) if top else F.linear_cross_entropy(*x, c[3].to(DEV), **how)
        return _kept(loss), dict(zip(("loss", "hidden", "weight"), [loss.detach(), *torch.autograd.grad(loss, x)]))
    for choice in (True, False):
        monkeypatch.setenv("FEA_AMD_LINEAR_KEEP", "0" if choice else str(1 << 40))
        kept, got = step(keep_logits=choice)
        assert kept == choice
        _compare(got, O.evaluate(*c, kept=None if choice else False))
        monkeypatch.setenv("FEA_AMD_LINEAR_KEEP", str(1 << 40) if choice else "0")
        kept, same = step()
        assert kept == choice and all(torch.equal(got[k], same[k]) for k in got)
    monkeypatch.undo()
    with torch.no_grad():
        assert torch.equal(F.linear_distillation(*x, c[4].to(DEV), c[3].to(DEV), keep_logits=True) if top else
                           F.linear_cross_entropy(*x, c[3].to(DEV), keep_logits=True), got["loss"])


def test_keep_logits_raises_where_there_is_no_room(monkeypatch):
    """Asked for, a failed allocation is the caller's; not wanted, none is tried."""
    c = O.case(300, 64, 700, torch.bfloat16, seed=52, ignored=0.1)
    n = L.load().fea_linear_loss_keep_bytes(300, 64, 700, L.BF16, 0)
    want = _run(*c, keep_logits=False)
    empty = torch.empty

    def full(*size, **how):
        if size == (n,) and how.get("dtype") == torch.uint8:
            raise torch.cuda.OutOfMemoryError("no room")
        return empty(*size, **how)
    monkeypatch.setattr(torch, "empty", full)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        _run(*c, keep_logits=True)
    for choice in (False, None):
        got = _run(*c, keep_logits=choice)
        assert all(torch.equal(got[k], want[k]) for k in want)


def test_without_kept_logits_memory_is_bounded_by_a_piece():
    """3.3e9 logits (6.6 GB in 16 bits): the step takes its gradients, a piece of 2^28 in 16 bits and as much again for partial sums."""
    g = torch.Generator(device=DEV).manual_seed(6)
    h = torch.randn(16384, 64, generator=g, device=DEV).bfloat16().requires_grad_(True)
    w = torch.randn(200000, 64, generator=g, device=DEV).bfloat16().requires_grad_(True)
    t = torch.randint(0, 200000, (16384,), generator=g, device=DEV)
    peaks = []
    for choice in (False, True):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        start = torch.cuda.memory_allocated()
        loss = F.linear_cross_entropy(h, w, t, keep_logits=choice)
        torch.autograd.grad(loss, [h, w])
        del loss
        torch.cuda.synchronize()
        peaks.append(torch.cuda.max_memory_allocated() - start)
    assert peaks[0] < 2 * (1 << 29) and peaks[1] > 16384 * 200000 * 2, peaks


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(64, 128, 500), (200, 72, 500), (513, 640, 1537), (1300, 643, 2011), (2049, 1096, 2310), (300, 520, 20000), (4100, 64, 6), (4200, 33, 30)])
@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("keep", [True, False])
def test_norms_of_the_errors(shape, dtype, top, keep):
    """All errors of a gradient together, with one upstream gradient and with one for every row, logits kept and recomputed."""
    c = O.case(*shape, dtype, seed=34 + top, top=top, ignored=0.1, short=0.2)
    kw = {"temperature": 2.0} if top else {}
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(8))
    for how in ({}, {"reduction": "none", "gout": gout}):
        want = O.evaluate(*c, norms=True, kept=None if keep else False, **kw, **how)
        got = _run(*c, keep_logits=keep, **kw, **how)
        O.check("loss", got["loss"], want["loss"])
        for k in ("hidden", "weight"):
            O.check_norm(k, got[k], want[k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("shape", [(40, 64, 300), (130, 51, 500), (4100, 24, 9)])
def test_saved_on_the_host_checkpointed_and_in_threads(shape, dtype, top):
    """What the forward saves may go to the host and back, be made again in the backward, and belong to steps of several threads at once."""
    import threading
    from torch.utils.checkpoint import checkpoint
    cases = [[None if t is None else t.to(DEV) for t in O.case(*shape, dtype, seed=s, top=top, ignored=0.1, bias=shape[0] == 40)] for s in (1, 2, 3, 4)]

    def loss(h, w, b, i, a=None):
        return F.linear_distillation(h, w, a, i, bias=b, temperature=2.0) if top else F.linear_cross_entropy(h, w, i, bias=b)

    def step(c, call=loss):
        x = [None if t is None else t.detach().requires_grad_(True) for t in c[:3]]
        out = call(*x, *c[3:])
        return [out.detach(), *torch.autograd.grad(out, [t for t in x if t is not None])]
    wants = [step(c) for c in cases]
    with torch.autograd.graph.save_on_cpu():
        got = step(cases[0])
    assert all(torch.equal(a, b) for a, b in zip(got, wants[0]))
    got = step(cases[1], lambda *x: checkpoint(loss, *x, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, wants[1]))
    torch.cuda.synchronize()
    gots = [None] * len(cases)

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(3):
                gots[k] = step(cases[k])
            torch.cuda.current_stream().synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for got, want in zip(gots, wants):
        assert got is not None and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(24, 64, 300), (120, 72, 500), (4200, 24, 9)])
def test_teacher_of_another_type_and_layout(shape, dtype):
    """A teacher's logits in the other type, int32 classes, both cut from wider rows, in a batch of sequences."""
    h, w, b, i, a = O.case(*shape, dtype, seed=36, top=5, ignored=0.1, short=0.2, bias=True)
    a = a.to(torch.float32 if dtype == torch.bfloat16 else torch.bfloat16)
    lead = (shape[0] // 12, 12)
    wide_a, wide_i = torch.full((*lead, 9), torch.nan, dtype=a.dtype, device=DEV), torch.full((*lead, 9), 1 << 20, dtype=torch.int32, device=DEV)
    wide_a[..., 2:7], wide_i[..., 3:8] = a.to(DEV).view(*lead, 5), i.to(DEV).view(*lead, 5).int()
    x, y, z = _leaf(h), _leaf(w), _leaf(b)
    loss = F.linear_distillation(x.view(*lead, -1), y, wide_a[..., 2:7], wide_i[..., 3:8], bias=z, temperature=2.0, reduction="none")
    assert loss.shape == lead
    gout = torch.randn(shape[0], generator=torch.Generator().manual_seed(9))
    grads = torch.autograd.grad(loss, [x, y, z], gout.to(DEV).view(lead))
    _compare(dict(zip(("loss", "hidden", "weight", "bias"), [loss, *grads])), O.evaluate(h, w, b, i, a, temperature=2.0, reduction="none", gout=gout))
