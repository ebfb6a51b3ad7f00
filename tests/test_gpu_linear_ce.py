"""linear_cross_entropy on the GPU against the definition in float64.

Tolerances, from the arithmetic (u = 2^-24, half a float32 step):
  a logit        l: operand pairs hold 22 bits and the lo*lo term is dropped: 3 u |x||w| per product; an accumulator
                 takes 16 adds that round toward zero (2 u each) before it is added in fp32 (u): with
                 S = sum |x||w|: |dl| <= (35 + K/128) u S + 4 u |l|. (Up to 16 rows without a
                 gradient: fp32 chains, K/8 + 8 adds.)
  a probability  p = 2^(l - lse): |dp| <= p (2 max|dl| + 8 u (1 + |lse|) + (128 + V/128) u)
  d = p - y      held as a pair: 2^-22 |d| + 2^-39 more
  a gradient     a product of d: (11 + n/64) u sum |d||w|, and dd carried through
Where rows are left out, or the incoming gradient is not one, the same bounds scale with it."""
import numpy as np
import pytest
import torch

from conftest import rng

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def formula(x, w, t, b=None, g=None):
    """Row losses and gradients in float64 (torch, on the GPU); g: the gradient of every row's loss."""
    x, w = torch.as_tensor(x, device="cuda").double(), torch.as_tensor(w, device="cuda").double()
    t = torch.as_tensor(t, device="cuda").double()
    live = t >= 0
    x = torch.where(live[:, None], x, torch.zeros_like(x))
    l = x @ w
    if b is not None:
        l = l + torch.as_tensor(b, device="cuda").double()
    lse = torch.logsumexp(l, 1)
    idx = t.clamp(min=0).long()
    rows = torch.where(live, lse - l.gather(1, idx[:, None])[:, 0], torch.zeros_like(lse))
    g = torch.ones_like(rows) if g is None else torch.as_tensor(g, device="cuda").double()
    g = torch.where(live, g, torch.zeros_like(g))
    p = torch.exp(l - lse[:, None])
    d = p.clone()
    d[torch.arange(len(t), device=d.device), idx] -= 1
    d = d * g[:, None]
    # bounds
    K, V, M = x.shape[1], w.shape[1], len(t)
    adds = 35 + K / 128 if M > 16 else max(35 + K / 128, 2 * (K / 8 + 9))
    finite_l = torch.where(torch.isfinite(l), l.abs(), torch.zeros_like(l))
    dl = (adds * U * (x.abs() @ w.abs()) + 4 * U * finite_l).amax(1)
    if K > 0 and M > 0:
        dl = dl + 2.0 ** -39 * x.abs().max() * w.abs().max() * K      # (elements far below the largest one)
    rel_p = 2 * dl + 8 * U * (1 + lse.abs()) + (128 + V / 128) * U
    dd = (rel_p[:, None] * p + 2.0 ** -39) * g.abs().amax() + 2.0 ** -22 * d.abs()
    dd = torch.where(live[:, None], dd, torch.zeros_like(dd))
    tol = {"rows": 2 * dl + 8 * U * (1 + lse.abs()),
           "dx": dd @ w.abs().t() + (11 + V / 64) * U * (d.abs() @ w.abs().t()),
           "dw": x.abs().t() @ dd + (11 + M / 64) * U * (x.abs().t() @ d.abs()),
           "db": dd.sum(0) + (8 + M / 32) * U * d.abs().sum(0)}
    return {"rows": rows, "dx": d @ w.t(), "dw": x.t() @ d, "db": d.sum(0), "live": live}, tol


def within(got, ref, tol, what):
    got = torch.as_tensor(np.asarray(got), device="cuda").double().reshape(ref.shape)
    bad = ~((got - ref).abs() <= tol)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g of tolerance" % (
        what, int(bad.sum()), bad.numel(), float(((got - ref).abs() / tol.clamp(min=1e-300))[bad].max()))


def near(got, ref, what, most=2e-6):
    """The 2-norm, where errors of random sign average out: at most the expected loss to truncation of the
    logits and of the gradient product (4e-7 each, times a spread of a few in l) and the pairs' 2^-22."""
    got = torch.as_tensor(np.asarray(got), device="cuda").double().reshape(ref.shape)
    if float(ref.norm()) > 0:
        assert float((got - ref).norm() / ref.norm()) <= most, (what, float((got - ref).norm() / ref.norm()))


def inputs(M, K, V, seed=0, ignored=0.0, scale=2.0):
    r = rng(seed)
    x = r.standard_normal((M, K)).astype(np.float32)
    w = (r.standard_normal((K, V)) * (scale / np.sqrt(K))).astype(np.float32)
    b = r.standard_normal(V).astype(np.float32)
    t = r.integers(0, V, M).astype(np.float32)
    if ignored:
        t[r.random(M) < ignored] = -1
    return x, w, b, t


def step(nd, x, w, t, b, reduction):
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    B = None if b is None else nd.Array(b, requires_grad=True)
    loss = nd.linear_cross_entropy(X, W, nd.Array(t), bias=B, reduction=reduction)
    if reduction != "none":
        loss.backward()
    return loss, X, W, B


SIZES = [(1, 1, 1), (1, 16, 2), (3, 7, 5), (2, 513, 130), (5, 1030, 131), (16, 64, 128), (17, 65, 129), (33, 40, 257), (128, 64, 256),
         (130, 100, 1000), (257, 129, 511), (300, 64, 4099), (64, 520, 3001), (255, 63, 8191), (513, 8, 300), (1000, 1, 77)]


@pytest.mark.parametrize("M,K,V", SIZES)
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_loss_and_gradients(nd, M, K, V, reduction):
    x, w, b, t = inputs(M, K, V, seed=M + K + V, ignored=0.2 if M > 4 else 0.0)
    b = b if reduction == "mean" else None
    live = (t >= 0).sum()
    c = 1.0 / live if reduction == "mean" else 1.0
    loss, X, W, B = step(nd, x, w, t, b, reduction)
    ref, tol = formula(x, w, t, b, np.full(M, c))
    assert loss.shape() == [1]
    total = float(ref["rows"].sum()) * (c if reduction == "mean" else 1.0)
    # the sum over the rows: ceil(M/512) + 25 adds of fp32
    bound = (float(tol["rows"].sum()) + (M / 512 + 25) * U * float(ref["rows"].abs().sum())) * c
    assert abs(float(loss.to_numpy()[0]) - total) <= bound + 4 * U * abs(total)
    assert X.grad().shape() == [M, K] and W.grad().shape() == [K, V]
    for name, arr in (("dx", X), ("dw", W)) + ((("db", B),) if B is not None else ()):
        within(arr.grad().to_numpy(), ref[name], tol[name], name)
        near(arr.grad().to_numpy(), ref[name], name)
    if B is not None:
        assert B.grad().shape() == [1, V]
    assert nd._lib.lib.endia_b200_device_status(None) == 0


@pytest.mark.parametrize("M,K,V", [(1, 16, 2), (7, 33, 1001), (16, 64, 128), (40, 65, 129), (300, 64, 4099)])
def test_row_losses_and_row_gradients(nd, M, K, V):
    """reduction="none": a loss per row, and a gradient that differs from row to row (of both signs and
    sizes apart by 2^20)."""
    x, w, b, t = inputs(M, K, V, seed=3, ignored=0.3 if M > 4 else 0.0)
    g = (rng(5).standard_normal(M) * 2.0 ** rng(6).integers(-10, 10, M)).astype(np.float32)
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    rows = nd.linear_cross_entropy(X, W, nd.Array(t), bias=B, reduction="none")
    assert rows.shape() == [M]
    ref, tol = formula(x, w, t, b, g)
    within(rows.to_numpy(), ref["rows"], tol["rows"], "rows")
    assert (rows.to_numpy()[t < 0] == 0).all()
    nd.sum(rows * nd.Array(g)).backward()
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        within(arr.grad().to_numpy(), ref[name], tol[name], name)


@pytest.mark.parametrize("M,K,V", [(8, 3584, 640), (16, 4096, 200), (17, 3000, 300)])
def test_few_rows_with_many_features(nd, M, K, V):
    """A logit's error (4e-7 of it, towards zero) is common to a row's logits and its log-sum-exp when both
    passes form them alike, and cancels: what is left of a gradient's error is that of its products."""
    x, w, b, t = inputs(M, K, V, seed=5, ignored=0.3)
    _, X, W, B = step(nd, x, w, t, b, "sum")
    ref, _ = formula(x, w, t, b)
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        near(arr.grad().to_numpy(), ref[name], name, most=8e-7)


@pytest.mark.parametrize("M,K,V", [(1, 16, 2), (3, 700, 333), (16, 1030, 131), (40, 65, 129)])
def test_losses_without_a_gradient(nd, M, K, V):
    """Nothing requires a gradient: the forward pass alone, one pass over the weight for up to 16 rows."""
    x, w, b, t = inputs(M, K, V, seed=6, ignored=0.2 if M > 4 else 0.0)
    rows = nd.linear_cross_entropy(nd.Array(x), nd.Array(w), nd.Array(t), bias=nd.Array(b), reduction="none")
    assert not rows.requires_grad()
    ref, tol = formula(x, w, t, b)
    within(rows.to_numpy(), ref["rows"], tol["rows"], "rows")
    mean = nd.linear_cross_entropy(nd.Array(x), nd.Array(w), nd.Array(t), bias=nd.Array(b))
    assert abs(float(mean.to_numpy()[0]) - float(ref["rows"].sum() / (t >= 0).sum())) <= float(tol["rows"].max()) + 1e-6


@pytest.mark.parametrize("M,K,V", [(70000, 8, 2500), (24, 70000, 2100)])
def test_several_pieces(nd, M, K, V):
    """Sizes at which the vocabulary is walked in several pieces, backward (many rows) and forward (many
    features), the last piece shorter than the others."""
    x, w, b, t = inputs(M, K, V, seed=1, ignored=0.1)
    loss, X, W, B = step(nd, x, w, t, b, "mean")
    c = 1.0 / (t >= 0).sum()
    ref, tol = formula(x, w, t, b, np.full(M, c))
    assert abs(float(loss.to_numpy()[0]) - float(ref["rows"].sum()) * c) <= float(tol["rows"].max()) + 1e-5
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        within(arr.grad().to_numpy(), ref[name], tol[name], name)
        near(arr.grad().to_numpy(), ref[name], name)


@pytest.mark.parametrize("M", [6, 40, 300])
def test_rows_left_out_may_hold_anything(nd, M):
    """NaN, infinities and the lowest float in rows whose target is negative: their loss and gradient are
    exactly zero and nothing else changes, to the bit."""
    K, V = 48, 700
    x, w, b, t = inputs(M, K, V, seed=9)
    t[1::2] = -1
    t[3] = -7.5
    outs = []
    for junk in (0.0, 1.0):
        xx = x.copy()
        if junk:
            xx[1] = np.nan
            xx[3] = np.inf
            xx[5, ::2] = np.finfo(np.float32).min
            xx[5, 1] = -np.inf
        else:
            xx[1::2] = 0
        loss, X, W, B = step(nd, xx, w, t, b, "mean")
        outs.append([a.to_numpy() for a in (loss, X.grad(), W.grad(), B.grad())])
        assert (X.grad().to_numpy()[1::2] == 0).all()
    for a, c in zip(*outs):
        assert np.array_equal(a, c)


@pytest.mark.parametrize("M", [3, 50])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_no_row_counts(nd, M, reduction):
    x, w, b, t = inputs(M, 20, 60)
    x[0] = np.nan
    loss, X, W, B = step(nd, x, w, np.full(M, -1, np.float32), b, reduction)
    assert loss.to_numpy()[0] == 0
    for a in (X, W, B):
        assert (a.grad().to_numpy() == 0).all()


def test_no_rows(nd):
    x, w, b, t = inputs(1, 12, 30)
    loss, X, W, B = step(nd, x[:0], w, t[:0], b, "mean")
    assert loss.to_numpy()[0] == 0 and X.grad().shape() == [0, 12]
    assert (W.grad().to_numpy() == 0).all() and (B.grad().to_numpy() == 0).all()
    rows = nd.linear_cross_entropy(nd.Array(x[:0]), nd.Array(w), nd.Array(t[:0]), reduction="none")
    assert rows.shape() == [0]


@pytest.mark.parametrize("M", [4, 60])
@pytest.mark.parametrize("bad", [30.0, 2.5, 1e9, np.nan, np.inf])
def test_a_target_that_names_no_class(nd, M, bad):
    x, w, b, t = inputs(M, 12, 30)
    t[2] = bad
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    rows = nd.linear_cross_entropy(X, W, nd.Array(t), reduction="none").to_numpy()
    assert np.isnan(rows[2]) and np.isfinite(np.delete(rows, 2)).all()
    loss = nd.linear_cross_entropy(X, W, nd.Array(t))
    loss.backward()
    assert np.isnan(loss.to_numpy()[0]) and np.isnan(W.grad().to_numpy()).all()
    dx = X.grad().to_numpy()
    assert np.isnan(dx[2]).all() and np.isfinite(np.delete(dx, 2, 0)).all()


@pytest.mark.parametrize("M", [5, 70])
def test_banned_classes(nd, M):
    """A bias of -inf or of the lowest float bans a class: probability 0 and no gradient through it."""
    K, V = 24, 400
    x, w, b, t = inputs(M, K, V, seed=4)
    b[7::3] = -np.inf
    b[8::3] = np.finfo(np.float32).min
    b[256:384] = -np.inf                       # a whole group of 128 classes
    t = (np.floor(t) % 7).astype(np.float32)
    loss, X, W, B = step(nd, x, w, t, b, "mean")
    ref, tol = formula(x, w, t, b, np.full(M, 1.0 / M))
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        within(arr.grad().to_numpy(), ref[name], tol[name], name)
    banned = ~np.isfinite(b) | (b < -1e30)
    assert (W.grad().to_numpy()[:, banned] == 0).all() and (B.grad().to_numpy()[0, banned] == 0).all()
    # a target that is banned: an infinite loss; no class left: NaN
    t2 = t.copy()
    t2[0] = 7
    rows = nd.linear_cross_entropy(nd.Array(x), nd.Array(w), nd.Array(t2), bias=nd.Array(b), reduction="none").to_numpy()
    assert np.isposinf(rows[0]) and np.isfinite(rows[1:]).all()
    rows = nd.linear_cross_entropy(nd.Array(x), nd.Array(w), nd.Array(t), bias=nd.Array(np.full(V, -np.inf)), reduction="none")
    assert np.isnan(rows.to_numpy()).all()


@pytest.mark.parametrize("M", [8, 80])
@pytest.mark.parametrize("sx,sw", [(1e18, 1e-18), (1e-25, 1e25), (3e-20, 1.0), (1.0, 1e-38)])
def test_scales_far_from_one(nd, M, sx, sw):
    x, w, b, t = inputs(M, 32, 300, seed=11)
    x, w = (x * sx).astype(np.float32), (w * sw).astype(np.float32)
    loss, X, W, _ = step(nd, x, w, t, None, "mean")
    ref, tol = formula(x, w, t, None, np.full(M, 1.0 / M))
    within(X.grad().to_numpy(), ref["dx"], tol["dx"] + 1e-44, "dx")
    within(W.grad().to_numpy(), ref["dw"], tol["dw"] + 1e-44, "dw")


@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e30])
def test_incoming_gradients_far_from_one(nd, scale):
    x, w, b, t = inputs(60, 32, 300, seed=12)
    g = (rng(1).standard_normal(60) * scale).astype(np.float32)
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    nd.sum(nd.linear_cross_entropy(X, W, nd.Array(t), bias=B, reduction="none") * nd.Array(g)).backward()
    ref, tol = formula(x, w, t, b, g)
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        within(arr.grad().to_numpy(), ref[name], tol[name] + 1e-44, name)
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    (nd.linear_cross_entropy(X, W, nd.Array(t), bias=B) * scale).backward()
    ref, tol = formula(x, w, t, b, np.full(60, float(np.float32(scale)) / 60))
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        within(arr.grad().to_numpy(), ref[name], tol[name] + 1e-44, name)


@pytest.mark.parametrize("M", [8, 80])
def test_one_element_far_above_the_others(nd, M):
    """An outlier sets the scale of its operand: the others keep 2^-40 of it."""
    x, w, b, t = inputs(M, 32, 300, seed=12)
    x[1, 3] = 2.0 ** 12
    w[3, :] *= 2.0 ** -10
    loss, X, W, B = step(nd, x, w, t, b, "mean")
    ref, tol = formula(x, w, t, b, np.full(M, 1.0 / M))
    for name, arr in (("dx", X), ("dw", W), ("db", B)):
        within(arr.grad().to_numpy(), ref[name], tol[name], name)


@pytest.mark.parametrize("M", [9, 64])
def test_large_logits(nd, M):
    """Logits of some hundreds: the maximum is taken out before any exponential."""
    x, w, b, t = inputs(M, 64, 513, seed=13, scale=200.0)
    loss, X, W, B = step(nd, x, w, t, b, "mean")
    assert np.isfinite(loss.to_numpy()[0])
    ref, tol = formula(x, w, t, b, np.full(M, 1.0 / M))
    assert abs(float(loss.to_numpy()[0]) - float(ref["rows"].mean())) <= float(tol["rows"].max())
    within(X.grad().to_numpy(), ref["dx"], tol["dx"], "dx")


@pytest.mark.parametrize("M", [7, 90])
def test_layouts(nd, M):
    """x as a strided view, with leading dims, transposed; the weight as the transposed view of an
    embedding and inside a wider matrix: the same result as from contiguous copies, to the bit."""
    from endia_b200._array import Array, ArrayShape
    K, V = 40, 333
    x, w, b, t = inputs(M, K, V, seed=14)

    def view_of(a, rows, cols, ld, offset):
        wide = np.full(offset + rows * ld, np.nan, np.float32)
        for i in range(rows):
            wide[offset + i * ld:offset + i * ld + cols] = a[i]
        base = nd.Array(wide)
        v = Array(ArrayShape([rows, cols], [ld, 1], offset))
        v.buf, v.base_, v.is_view = base.buf, base, True
        return v.requires_grad_(True)
    _, X0, W0, _ = step(nd, x, w, t, b, "mean")
    want = X0.grad().to_numpy(), W0.grad().to_numpy()
    for xv, wv in ((view_of(x, M, K, K + 5, 3), view_of(w, K, V, V + 7, 9)), (view_of(x, M, K, K + 8, 8), view_of(w, K, V, 340, 4))):
        nd.linear_cross_entropy(xv, wv, nd.Array(t), bias=nd.Array(b)).backward()
        assert np.array_equal(xv.grad().to_numpy(), want[0]) and np.array_equal(wv.grad().to_numpy(), want[1])
    # tied embedding: rows of E are the classes
    E, XT = nd.Array(np.ascontiguousarray(w.T), requires_grad=True), nd.Array(np.ascontiguousarray(x.T), requires_grad=True)
    nd.linear_cross_entropy(XT.T(), E.T(), nd.Array(t), bias=nd.Array(b)).backward()
    assert np.array_equal(E.grad().to_numpy(), want[1].T) and np.array_equal(XT.grad().to_numpy(), want[0].T)
    # leading dims
    if M % 3 == 0:
        X3 = nd.Array(x.reshape(3, M // 3, K), requires_grad=True)
        W3 = nd.Array(w, requires_grad=True)
        rows = nd.linear_cross_entropy(X3, W3, nd.Array(t.reshape(3, M // 3)), bias=nd.Array(b), reduction="none")
        assert rows.shape() == [3, M // 3]
        nd.linear_cross_entropy(X3, W3, nd.Array(t.reshape(3, M // 3)), bias=nd.Array(b)).backward()
        assert X3.grad().shape() == [3, M // 3, K]
        assert np.array_equal(X3.grad().to_numpy().reshape(M, K), want[0]) and np.array_equal(W3.grad().to_numpy(), want[1])


def test_the_same_array_twice(nd):
    """Weight and input from one array, and a target used twice: gradients add up."""
    r = rng(2)
    a = r.standard_normal((24, 24)).astype(np.float32)
    t = r.integers(0, 24, 24).astype(np.float32)
    A = nd.Array(a, requires_grad=True)
    nd.linear_cross_entropy(A, A, nd.Array(t)).backward()
    ref, tol = formula(a, a, t, None, np.full(24, 1 / 24))
    within(A.grad().to_numpy(), ref["dx"] + ref["dw"], tol["dx"] + tol["dw"] + U * (ref["dx"] + ref["dw"]).abs(), "sum")
    W = nd.Array(a, requires_grad=True)
    T = nd.Array(t)
    l1, l2 = nd.linear_cross_entropy(nd.Array(a), W, T), nd.linear_cross_entropy(nd.Array(2 * a), W, T)
    (l1 + l2).backward()
    r1, t1 = formula(a, a, t, None, np.full(24, 1 / 24))
    r2, t2 = formula(2 * a, a, t, None, np.full(24, 1 / 24))
    within(W.grad().to_numpy(), r1["dw"] + r2["dw"], t1["dw"] + t2["dw"] + U * (r1["dw"] + r2["dw"]).abs(), "two losses")


def test_only_the_gradients_that_are_asked_for(nd):
    x, w, b, t = inputs(40, 32, 500, seed=21)
    full = step(nd, x, w, t, b, "mean")
    for which in (0, 1, 2):
        arrs = [nd.Array(a, requires_grad=i == which) for i, a in enumerate((x, w, b))]
        nd.linear_cross_entropy(arrs[0], arrs[1], nd.Array(t), bias=arrs[2]).backward()
        assert np.array_equal(arrs[which].grad().to_numpy(), full[1 + which].grad().to_numpy())
        assert not any(a.has_grad() for i, a in enumerate(arrs) if i != which)
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    g = nd.grad(outs=[nd.linear_cross_entropy(X, W, nd.Array(t), bias=nd.Array(b))], inputs=[X])[0]
    assert np.array_equal(g.to_numpy(), full[1].grad().to_numpy()) and not W.has_grad()


@pytest.mark.parametrize("M,K,V", [(12, 30, 200), (600, 130, 5000)])
def test_the_same_bits_every_time(nd, M, K, V):
    x, w, b, t = inputs(M, K, V, seed=22, ignored=0.1)
    a, c = (step(nd, x, w, t, b, "mean") for _ in range(2))
    for u, v in ((a[0], c[0]), (a[1].grad(), c[1].grad()), (a[2].grad(), c[2].grad()), (a[3].grad(), c[3].grad())):
        assert np.array_equal(u.to_numpy(), v.to_numpy())


@pytest.mark.parametrize("M", [10, 40])
def test_gradient_against_differences(nd, M):
    """The directional derivative of the float64 loss by central differences (h = 1e-4: error h^2 of the
    third derivative, 1e-7 of the value here)."""
    K, V = 30, 150
    x, w, b, t = inputs(M, K, V, seed=23, ignored=0.2)
    loss, X, W, B = step(nd, x, w, t, b, "mean")
    r = rng(24)
    for arr, at in ((X, 0), (W, 1), (B, 2)):
        v = r.standard_normal((x, w, b)[at].shape)

        def value(h):
            args = [x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)]
            args[at] = args[at] + h * v
            l = args[0] @ args[1] + args[2]
            keep = t >= 0
            m = l.max(1, keepdims=True)
            lse = (m + np.log(np.exp(l - m).sum(1, keepdims=True)))[:, 0]
            return (lse - l[np.arange(M), np.maximum(t, 0).astype(int)])[keep].mean()
        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        got = float((arr.grad().to_numpy().reshape(v.shape).astype(np.float64) * v).sum())
        assert abs(got - slope) <= 1e-5 * max(1.0, abs(slope)), (got, slope)


def test_second_order_and_forward_mode(nd):
    """create_graph=True and jvp use the differentiable composition: gradients of gradients against torch in
    float64 (1e-4, the bound of the framework's second-order tests)."""
    M, K, V = 6, 8, 11
    x, w, b, t = inputs(M, K, V, seed=25)
    t[2] = -1
    v = rng(26).standard_normal((M, K)).astype(np.float32)
    for reduction in ("mean", "sum"):
        X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
        loss = nd.linear_cross_entropy(X, W, nd.Array(t), bias=B, reduction=reduction)
        gx = nd.grad(outs=[loss], inputs=[X], create_graph=True)[0]
        gw = nd.grad(outs=[nd.sum(gx * nd.Array(v))], inputs=[W])[0].to_numpy()
        tx, tw, tb = (torch.tensor(a, dtype=torch.float64, requires_grad=True) for a in (x, w, b))
        tl = torch.nn.functional.cross_entropy(tx @ tw + tb, torch.tensor(np.where(t < 0, -100, t)).long(), reduction=reduction)
        tg = torch.autograd.grad(tl, tx, create_graph=True)[0]
        want = torch.autograd.grad((tg * torch.tensor(v).double()).sum(), tw)[0].numpy()
        assert np.abs(gw - want).max() <= 1e-4 * np.abs(want).max()
        assert np.abs(gx.to_numpy() - tg.detach().numpy()).max() <= 1e-5
        X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
        loss = nd.linear_cross_entropy(X, W, nd.Array(t), bias=B, reduction=reduction)
        tangent = nd.jvp(loss, [X], [nd.Array(v)]).to_numpy()
        assert tangent.shape == (1,) and abs(tangent[0] - float((tg.detach() * torch.tensor(v)).sum())) <= 1e-5
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    rows = nd.linear_cross_entropy(X, W, nd.Array(t), reduction="none")
    tan = nd.jvp(rows, [X], [nd.Array(v)])
    assert tan.shape() == [M] and tan.to_numpy()[2] == 0


def test_jacobian_of_the_row_losses(nd):
    M, K, V = 5, 6, 9
    x, w, b, t = inputs(M, K, V, seed=28)
    t[1] = -1
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    rows = nd.linear_cross_entropy(X, W, nd.Array(t), bias=B, reduction="none")
    rows.backward()
    assert X.grad().shape() == [M, M, K] and W.grad().shape() == [M, K, V]
    for i in range(M):
        ref, _ = formula(x, w, t, b, np.eye(M)[i])
        assert np.abs(X.grad().to_numpy()[i] - ref["dx"].cpu().numpy()).max() <= 1e-5
        assert np.abs(W.grad().to_numpy()[i] - ref["dw"].cpu().numpy()).max() <= 1e-5
        assert np.abs(B.grad().to_numpy()[i, 0] - ref["db"].cpu().numpy()).max() <= 1e-5


def test_on_another_stream(nd):
    x, w, b, t = inputs(200, 64, 3000, seed=27)
    want = step(nd, x, w, t, b, "mean")
    want = [a.to_numpy() for a in (want[0], want[1].grad(), want[2].grad(), want[3].grad())]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            got = step(nd, x, w, t, b, "mean")
        got = [a.to_numpy() for a in (got[0], got[1].grad(), got[2].grad(), got[3].grad())]
    for a, c in zip(got, want):
        assert np.array_equal(a, c)


def test_two_streams_at_once(nd):
    """Two steps in flight on two streams: no work space is shared."""
    cases = [inputs(300, 64, 5000, seed=s) for s in (31, 32)]
    want = []
    for x, w, b, t in cases:
        r = step(nd, x, w, t, b, "mean")
        want.append([a.to_numpy() for a in (r[0], r[1].grad(), r[2].grad())])
    arrs = [[nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True), nd.Array(b), nd.Array(t)] for x, w, b, t in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    losses = [None, None]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                X, W, B, T = arrs[i]
                X.remove_grad()
                W.remove_grad()
                losses[i] = nd.linear_cross_entropy(X, W, T, bias=B)
                losses[i].backward()
    torch.cuda.synchronize()
    for i in range(2):
        for a, c in zip((losses[i], arrs[i][0].grad(), arrs[i][1].grad()), want[i]):
            assert np.array_equal(a.to_numpy(), c)


def test_captured_step_with_refilled_inputs(nd):
    """A training step captured as a graph and replayed on new inputs (another share of rows left out)
    gives the bits of the step run op by op; two captured steps do not share anything."""
    from endia_b200.utils.general import CapturedStep
    M, K, V = 96, 48, 900
    sets = [inputs(M, K, V, seed=s, ignored=i) for s, i in ((41, 0.0), (42, 0.4), (43, 0.1))]
    w0, b0 = sets[0][1], sets[0][2]

    def make():
        X, T = nd.Array(sets[0][0]), nd.Array(sets[0][3])
        W, B = nd.Array(w0.copy(), requires_grad=True), nd.Array(b0.copy(), requires_grad=True)
        opt = nd.optim.Adam([W, B], lr=1e-2)

        def fn():
            loss = nd.linear_cross_entropy(X, W, T, bias=B)
            loss.backward()
            opt.step()
            loss.zero_grad()
            return loss
        return X, T, W, B, opt, fn
    results = []
    runs = [make(), make(), make()]
    cap = [CapturedStep(r[5], warmup=1, optimizers=[r[4]]) for r in runs[:2]]
    for r in runs:      # back to the start
        torch.cuda.synchronize()
        r[2].buf.copy_(torch.from_numpy(w0.reshape(-1)))
        r[3].buf.copy_(torch.from_numpy(b0))
        r[4].reset_state()
        nd._array.drop_operand_parts(r[2])
    for x, _, _, t in sets:
        for i, r in enumerate(runs):
            r[0].buf.copy_(torch.from_numpy(x.reshape(-1)))
            r[1].buf.copy_(torch.from_numpy(t))
        losses = [cap[0](), cap[1](), runs[2][5]()]
        torch.cuda.synchronize()
        results.append([l.to_numpy() for l in losses])
        assert np.array_equal(results[-1][0], results[-1][1]) and np.array_equal(results[-1][0], results[-1][2])
    # (the captured optimizer forms its bias corrections on the device: parameters agree to its rounding)
    assert np.array_equal(runs[0][2].to_numpy(), runs[1][2].to_numpy())
    assert np.abs(runs[0][2].to_numpy() - runs[2][2].to_numpy()).max() <= 1e-6
    for c in cap:
        c.release()


def test_c_abi_refusals(nd):
    """Bad arguments of the C entry points become a status and a message; nothing is launched."""
    L = nd._lib.lib
    buf = torch.zeros(4096, device="cuda")
    p = buf.data_ptr()
    big = torch.zeros(L.endia_b200_linear_ce_scratch_bytes(4, 8, 16, 1) // 4 + 64, device="cuda").data_ptr()
    before = L.endia_b200_launch_count()
    ok = (p, 8, p, 16, None, p, 4, 8, 16, 0)
    bad = [(p, 7, p, 16, None, p, 4, 8, 16, 0), (p, 8, p, 15, None, p, 4, 8, 16, 0), (None, 8, p, 16, None, p, 4, 8, 16, 0),
           (p, 8, None, 16, None, p, 4, 8, 16, 0), (p, 8, p, 16, None, None, 4, 8, 16, 0), (p, 8, p, 16, None, p, -1, 8, 16, 0),
           (p, 8, p, 16, None, p, 4, 0, 16, 0), (p, 8, p, 16, None, p, 4, 8, 0, 0), (p, 8, p, 16, None, p, 4, 8, 16, 3)]
    for a in bad:
        assert L.endia_b200_linear_ce_fwd(*a, p, p, big, None) == nd._lib.EINVAL
        assert L.endia_b200_linear_ce_bwd(*a, p, p, p, p, p, big, None) == nd._lib.EINVAL
        assert b"linear_ce" in L.endia_b200_last_error()
    assert L.endia_b200_linear_ce_fwd(p, 8, p, 1 << 25, None, p, 4, 8, (1 << 24) + 1, 0, p, p, big, None) == nd._lib.ELIMIT
    assert L.endia_b200_linear_ce_fwd(*ok, None, p, big, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_ce_bwd(*ok, p, None, p, p, p, big, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_ce_fwd(*ok, p, p, None, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_ce_fwd(*ok, p, p, big + 16, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_ce_bwd(*ok, None, p, p, p, p, big, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_ce_bwd(*ok, p, p, None, None, None, big, None) == nd._lib.OK      # nothing asked for
    assert L.endia_b200_launch_count() == before
