"""Activations held in 8 bits (keep8) and the layers that read them (linear(checkpoint=True), MLP(checkpoint=True)).

The 8-bit form is exact arithmetic: it is compared bit by bit with its definition in numpy. The layer's
products are compared with float64 under the bounds of products of 22-bit pairs (u = 2^-24):
(11 + n/64) u sum |a||b| (pairs 3 u, four adds that round toward zero 2 u each, one fp32 add per 64), and
(27 + n/128) u for the product with the 8-bit operand (twelve such adds, one fp32 add per 128)."""
import numpy as np
import pytest
import torch

from conftest import rng, max_rel

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = {None: (lambda z: z, lambda y: np.ones_like(y)), "relu": (lambda z: np.maximum(z, 0), lambda y: (y > 0) * 1.0),
        "tanh": (np.tanh, lambda y: 1 - y * y), "sigmoid": (lambda z: 1 / (1 + np.exp(-z)), lambda y: y * (1 - y))}


def kept_values(x, keep_sign):
    """What the 8-bit form of a float32 array [rows, cols] stands for, by its definition, in float64."""
    rows, cols = x.shape
    pad = (-cols) % 32
    b = np.concatenate([x.astype(np.float64), np.zeros((rows, pad))], 1).reshape(rows, -1, 32)
    finite = np.isfinite(b)
    top = np.where(finite, np.abs(b), 0).max(2, keepdims=True)
    e = np.full(top.shape, -126, np.int64)
    f, k = np.frexp(top)
    e = np.where(top > 0, np.clip(k - 7 + (f * 128 >= 127.5), -126, 121), e)
    unit = np.ldexp(1.0, e)
    v = np.where(finite, b, 0) / unit
    q = np.rint(v)
    if keep_sign:
        q = np.where((q == 0) & (v != 0), np.sign(v), q)
    assert np.abs(q[e[..., 0] < 121]).max(initial=0) <= 127
    q = np.clip(q, -127, 127)
    return np.where(finite, q * unit, np.nan).reshape(rows, -1)[:, :cols]


def read_back(nd, x, keep_sign):
    a = nd.Array(x)
    a.name = "relu" if keep_sign else "arg"
    h = nd.keep8(a)
    assert h is a and a.held()
    return a.to_numpy()


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 64), (7, 100), (33, 257), (1, 5000), (400, 1), (129, 1023), (64, 4096)])
@pytest.mark.parametrize("keep_sign", [False, True])
def test_form_bit_by_bit(nd, rows, cols, keep_sign):
    r = rng(rows * 10007 + cols)
    x = (r.standard_normal((rows, cols)) * np.exp(r.standard_normal((rows, cols)) * 2)).astype(np.float32)
    x[r.random(x.shape) < 0.2] = 0
    assert np.array_equal(read_back(nd, x, keep_sign), kept_values(x, keep_sign).astype(np.float32))


def test_form_at_its_edges(nd):
    """Blocks of zeros, of one value, next to the limits of rounding to 127, denormals, the largest
    floats, NaN and infinities."""
    f = np.finfo(np.float32)
    rows = []
    for top in (1.0, 127.0, 127.49, 127.5, np.nextafter(np.float32(127.5), np.float32(0)), 127.51, 128.0, 255.0, 2.0 ** -100, f.tiny, f.tiny / 8, f.max,
                2.0 ** -149, 0.0):
        row = np.linspace(-1, 1, 32) * top
        row[0], row[1], row[2] = top, -top, 1e-7 * top
        rows.append(row)
    x = np.array(rows, np.float32)
    x = np.concatenate([x, x[:, ::-1] * np.float32(0.37)], 1)
    for keep_sign in (False, True):
        got = read_back(nd, x, keep_sign)
        assert np.isfinite(got).all()
        assert np.array_equal(got, kept_values(x, keep_sign).astype(np.float32))
    y = rng(1).standard_normal((4, 96)).astype(np.float32)
    y[0, 3], y[1, 40], y[2, 95], y[3, :32] = np.nan, np.inf, -np.inf, np.nan
    assert np.array_equal(read_back(nd, y, True), kept_values(y, True).astype(np.float32), equal_nan=True)


def test_error_bound_and_size(nd):
    """At most half a unit, and a unit is at most max / 63.75; 8.25 bits per value."""
    x = rng(2).standard_normal((256, 512)).astype(np.float32)
    got = read_back(nd, x, False)
    top = np.abs(x).reshape(256, 16, 32).max(2, keepdims=True)
    assert (np.abs(got - x).reshape(256, 16, 32) <= top / 63.75 / 2).all()
    assert nd._lib.lib.endia_b200_keep8_bytes(256, 512) == 256 * 512 * 33 // 32


def test_keep8_releases_and_reads_back(nd):
    """The float32 storage goes; an op that reads the array afterwards gets the values of the form; an
    in-place update works on them."""
    x = rng(3).standard_normal((1000, 1024)).astype(np.float32)
    z = nd.Array(x, requires_grad=True)
    h = z * 2.0
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    nd.keep8(h)
    freed = before - torch.cuda.memory_allocated()
    assert freed >= 1000 * 1024 * 4 - (1000 * 1024 * 33 // 32 + 1024)
    want = kept_values(2 * x, False).astype(np.float32)
    assert h.held() and h.shape() == [1000, 1024]
    assert nd.keep8(h) is h and h.held()
    s = nd.sum(h * h)
    assert not h.held()
    assert np.array_equal(h.to_numpy(), want)
    s.backward()        # d sum(h^2) = 2 h, from the form; the graph below is whole
    assert max_rel(z.grad().to_numpy(), 4 * want) <= 4 * U
    h += 1.0
    assert np.array_equal(h.to_numpy(), want + np.float32(1))
    nd.keep8(h)
    assert np.array_equal(h.to_numpy(), kept_values(want + np.float32(1), False).astype(np.float32))


def layer_case(M, K, N, seed):
    r = rng(seed)
    x = (r.standard_normal((M, K)) * np.exp(0.7 * r.standard_normal(K))).astype(np.float32)
    w = (r.standard_normal((K, N)) / np.sqrt(K)).astype(np.float32)
    b = (r.standard_normal(N) * 0.1).astype(np.float32)
    g = r.standard_normal((M, N)).astype(np.float32)
    return x, w, b, g


@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 40, 3), (3, 33, 65), (32, 64, 64), (130, 257, 129), (300, 512, 520), (1001, 77, 333), (2000, 16, 16), (20, 3000, 40)])
@pytest.mark.parametrize("act", [None, "relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("hold", [False, True])
def test_layer_against_the_formula(nd, M, K, N, act, hold):
    """out = act(x W + b) from x; dx, dW, db from the 8-bit forms of x and (hold) of out, relative to the
    values that the forward pass really produced."""
    x, w, b, g = layer_case(M, K, N, M + K + N)
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    out = nd.nn.linear(X, W, B, act, checkpoint=True)
    y = out.to_numpy()
    f, df = ACTS[act]
    x64, w64, b64 = (a.astype(np.float64) for a in (x, w, b))
    zz = x64 @ w64 + b64
    size = np.abs(x64) @ np.abs(w64) + np.abs(b64)
    # (no activation here has a slope above 1; tanhf and the sigmoid's expf: 4 u)
    assert (np.abs(y - f(zz)) <= (12 + K / 64) * U * size + 4 * U * np.abs(f(zz)) + 2.0 ** -38 * np.abs(x).max() * np.abs(w).max() * K).all()
    loss = nd.sum(out * nd.Array(g))
    if hold:
        nd.keep8(out)
    loss.backward()
    yk = kept_values(y, act == "relu") if hold else y.astype(np.float64)
    ds = g.astype(np.float64) * df(yk)
    xk = kept_values(x, False)
    grads = {"dx": (ds @ w64.T, np.abs(ds) @ np.abs(w64).T, N, X), "dw": (xk.T @ ds, np.abs(xk).T @ np.abs(ds), M, W)}
    for name, (ref, mag, n, arr) in grads.items():
        got = arr.grad().to_numpy()
        tiny = 2.0 ** -38 * np.abs(ds).max() * (np.abs(w).max() if name == "dx" else np.abs(xk).max()) * n
        c = 11 + n / 64 if name == "dx" else 27 + n / 128
        assert (np.abs(got - ref) <= (c + 8) * U * mag + tiny).all(), name     # (8 u: act' in fp32)
        assert np.linalg.norm(got - ref) <= 2e-6 * np.linalg.norm(ref) + 1e-30, name
    db = B.grad().to_numpy()
    assert db.shape == (1, N)
    assert (np.abs(db[0] - ds.sum(0)) <= (8 + 8 + M / 64) * U * np.abs(ds).sum(0) + 1e-30).all()
    assert nd._lib.lib.endia_b200_device_status(None) == 0


def test_layer_without_bias_and_parts_of_the_gradient(nd):
    x, w, b, g = layer_case(70, 50, 90, 5)
    whole = None
    for grads in ((1, 1), (1, 0), (0, 1)):
        X, W = nd.Array(x, requires_grad=bool(grads[0])), nd.Array(w, requires_grad=bool(grads[1]))
        nd.sum(nd.nn.linear(X, W, checkpoint=True) * nd.Array(g)).backward()
        got = [a.grad().to_numpy() if a.has_grad() else None for a in (X, W)]
        if whole is None:
            whole = got
        for a, c, k in zip(got, whole, grads):
            assert (a is None) == (k == 0) and (a is None or np.array_equal(a, c))
    # no gradient at all: nothing is kept
    y = nd.nn.linear(nd.Array(x), nd.Array(w), checkpoint=True)
    assert not y.requires_grad() and y.args() == []


def test_empty_and_strided_layers(nd):
    from endia_b200._array import Array, ArrayShape
    X, W, B = nd.Array(np.zeros((0, 5), np.float32), requires_grad=True), nd.Array(np.ones((5, 3), np.float32), requires_grad=True), nd.Array(np.ones(3, np.float32), requires_grad=True)
    out = nd.nn.linear(X, W, B, "relu", checkpoint=True)
    assert out.shape() == [0, 3]
    nd.sum(out).backward()
    assert (W.grad().to_numpy() == 0).all() and (B.grad().to_numpy() == 0).all() and X.grad().shape() == [0, 5]
    x, w, b, g = layer_case(60, 40, 52, 6)
    A, C = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    nd.sum(nd.nn.linear(A, C, nd.Array(b), "tanh", checkpoint=True) * nd.Array(g)).backward()
    wide = np.zeros((60, 47), np.float32)
    wide[:, 3:43] = x
    base = nd.Array(wide)
    V = Array(ArrayShape([60, 40], [47, 1], 3))
    V.buf, V.base_, V.is_view = base.buf, base, True
    V.requires_grad_(True)
    Wt = nd.Array(np.ascontiguousarray(w.T), requires_grad=True)
    nd.sum(nd.nn.linear(V, Wt.T(), nd.Array(b), "tanh", checkpoint=True) * nd.Array(g)).backward()
    assert np.array_equal(V.grad().to_numpy(), A.grad().to_numpy())
    assert np.array_equal(Wt.grad().to_numpy(), C.grad().to_numpy().T)


def mlp_reference(Ws, bs, x, act, dloss, hidden):
    """The gradients of a stack whose layers keep 8-bit forms, in float64, from the hidden activations that
    the forward pass produced (hidden[i]: the float32 output of layer i)."""
    f, df = ACTS[act]
    n = len(Ws)
    g = dloss.astype(np.float64)
    grads = []
    for i in range(n - 1, -1, -1):
        below = kept_values(x if i == 0 else hidden[i - 1], i > 0 and act == "relu")
        ds = g if i == n - 1 else g * df(kept_values(hidden[i], act == "relu"))
        grads = [below.T @ ds, ds.sum(0)] + grads
        g = ds @ Ws[i].astype(np.float64).T
    return grads, g


@pytest.mark.parametrize("act", ["relu", "tanh", "sigmoid"])
@pytest.mark.parametrize("dims,batch", [([8, 64, 64, 4], 256), ([20, 70, 130, 40, 10], 33)])
def test_mlp_against_the_formula(nd, act, dims, batch):
    r = rng(7)
    net = nd.nn.MLP(dims, compute_backward=True, activation=act, checkpoint=True)
    x = r.standard_normal((batch, dims[0])).astype(np.float32)
    y = r.standard_normal((batch, dims[-1])).astype(np.float32)
    Ws, bs = [w.to_numpy() for w in net.weights], [b.to_numpy() for b in net.biases]
    # the activations of the forward pass, from a stack whose arrays stay in float32
    hidden, h = [], nd.Array(x)
    for i, (w, b) in enumerate(zip(net.weights, net.biases)):
        h = nd.nn.linear(h, w, b, act if i < len(dims) - 2 else None, checkpoint=True)
        hidden.append(h.to_numpy())
    X = nd.Array(x, requires_grad=True)
    pred = net.forward(X)
    assert np.array_equal(pred.to_numpy(), hidden[-1])          # the forward values do not depend on it
    loss = nd.mse(pred, nd.Array(y))
    loss.backward()
    dloss = 2.0 * (hidden[-1].astype(np.float64) - y) / y.size
    grads, gx = mlp_reference(Ws, bs, x, act, dloss, hidden)
    # products of pairs and act' in fp32, layer by layer: 2e-6 of the norm per layer
    for got, ref in zip([p.grad().to_numpy() for p in net.params()] + [X.grad().to_numpy()], grads + [gx]):
        assert np.linalg.norm(got.reshape(ref.shape) - ref) <= 2e-6 * len(dims) * np.linalg.norm(ref)
    # every hidden activation is in 8 bits until something reads it
    node, held = pred, []
    while node.args_:
        node = node.args_[0]
        held.append(type(node).__name__ == "Kept8" and node.held())
    assert held == [True] * (len(dims) - 2) + [False]


def test_mlp_memory(nd):
    """What a forward pass leaves behind for the backward pass: a quarter of it per hidden activation."""
    dims, batch = [256, 2048, 2048, 2048, 2048, 64], 4096

    def held(checkpoint):
        net = nd.nn.MLP(dims, compute_backward=True, activation="tanh", checkpoint=checkpoint)
        x = nd.Array(np.ones((batch, dims[0]), np.float32))
        net.forward(x)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = net.forward(x)
        torch.cuda.synchronize()
        return torch.cuda.memory_allocated() - before, out
    full, _a = held(False)
    kept, _b = held(True)
    hidden = 4 * batch * 2048 * 4
    assert full >= hidden
    assert kept <= hidden * 33 / 128 + batch * (dims[0] * 33 // 32 + dims[-1] * 4) + (4 << 20)


def test_activation_with_another_use(nd):
    """An activation that a second op uses keeps its exact values in the forward pass as long as it is not
    handed to keep8, and both paths' gradients arrive."""
    x, w, b, g = layer_case(40, 32, 32, 8)
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    h = nd.relu(X)
    out = nd.nn.linear(h, W, nd.Array(b), checkpoint=True) + h          # a skip connection
    want = np.maximum(x, 0).astype(np.float64) @ w + b + np.maximum(x, 0)
    assert max_rel(out.to_numpy(), want) <= 2e-6
    loss = nd.sum(out * nd.Array(g))
    nd.keep8(h)
    loss.backward()
    ref = (g.astype(np.float64) @ w.astype(np.float64).T + g) * (x > 0)
    assert np.linalg.norm(X.grad().to_numpy() - ref) <= 2e-6 * np.linalg.norm(ref)
    hk = kept_values(np.maximum(x, 0), True)
    assert np.linalg.norm(W.grad().to_numpy() - hk.T @ g) <= 2e-6 * np.linalg.norm(hk.T @ g)


def test_layer_gradient_against_differences(nd):
    """dx of a layer does not depend on the 8-bit form of x: it is the slope of the float64 layer."""
    x, w, b, g = layer_case(12, 20, 24, 9)
    X = nd.Array(x, requires_grad=True)
    nd.sum(nd.nn.linear(X, nd.Array(w), nd.Array(b), "tanh", checkpoint=True) * nd.Array(g)).backward()
    v = rng(10).standard_normal(x.shape)

    def value(h):
        return (np.tanh((x.astype(np.float64) + h * v) @ w.astype(np.float64) + b) * g).sum()
    slope = (value(1e-4) - value(-1e-4)) / 2e-4
    got = float((X.grad().to_numpy().astype(np.float64) * v).sum())
    assert abs(got - slope) <= 1e-5 * max(1.0, abs(slope))


def test_second_order_through_a_checkpointed_layer(nd):
    """create_graph=True: the first gradient is the composition of differentiable ops, as for a layer without
    a checkpoint. Differentiating it again goes back through the layer, whose weight gradient reads the
    8-bit x: S = sum(v gx), gx = ds W^T, ds = g (1 - y^2): dS/dW = v^T ds + x8^T q, q = -2 y (1 - y^2) g (v W)."""
    x, w, b, g = layer_case(10, 12, 14, 11)
    v = rng(12).standard_normal(x.shape).astype(np.float32)
    got = []
    for checkpoint in (False, True):
        X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
        out = nd.nn.linear(X, W, B, "tanh", checkpoint=checkpoint)
        gx = nd.grad(outs=[nd.sum(out * nd.Array(g))], inputs=[X], create_graph=True)[0]
        got.append([gx.to_numpy(), nd.grad(outs=[nd.sum(gx * nd.Array(v))], inputs=[X])[0].to_numpy()])
        X2 = nd.Array(x, requires_grad=True)
        got[-1].append(nd.jvp(nd.nn.linear(X2, nd.Array(w), nd.Array(b), "tanh", checkpoint=checkpoint), [X2], [nd.Array(v)]).to_numpy())
    for a, c in zip(*got):
        assert np.abs(a - c).max() <= 1e-4 * np.abs(a).max()
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    gx = nd.grad(outs=[nd.sum(nd.nn.linear(X, W, B, "tanh", checkpoint=True) * nd.Array(g))], inputs=[X], create_graph=True)[0]
    dw = nd.grad(outs=[nd.sum(gx * nd.Array(v))], inputs=[W])[0].to_numpy()
    w64 = w.astype(np.float64)
    y = np.tanh(x.astype(np.float64) @ w64 + b)
    q = -2 * y * (1 - y * y) * g * (v.astype(np.float64) @ w64)
    want = v.astype(np.float64).T @ (g * (1 - y * y)) + kept_values(x, False).T @ q
    assert np.abs(dw - want).max() <= 1e-4 * np.abs(want).max()


@pytest.mark.parametrize("sx,sw", [(1e-19, 1e-18), (1e-37, 1.0), (1e18, 1e-18), (1e25, 1e-30)])
def test_blocks_of_zeros_beside_tiny_and_large_ones(nd, sx, sw):
    """The operands have a scale per block of 128 x 128; one that is all zeros says nothing about the others,
    and products across blocks of far-apart scales keep the bounds."""
    x, w, b, g = layer_case(300, 390, 260, 31)
    x, w = (x * sx).astype(np.float32), (w * sw).astype(np.float32)
    x[:, :128] = 0
    w[128:256] = 0
    x[130:256, 256:] *= np.float32(2.0 ** -20)
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    out = nd.nn.linear(X, W, checkpoint=True)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    size = np.abs(x64) @ np.abs(w64)
    floor = 2.0 ** -38 * np.abs(x).max() * np.abs(w).max() * 390 + 1e-44
    assert (np.abs(out.to_numpy() - x64 @ w64) <= (12 + 390 / 64) * U * size + floor).all()
    assert np.abs(out.to_numpy()).max() > 0
    nd.sum(out * nd.Array(g)).backward()
    xk = kept_values(x, False)
    for got, ref, mag, n in ((X.grad(), g @ w64.T, np.abs(g) @ np.abs(w64).T, 260), (W.grad(), xk.T @ g, np.abs(xk).T @ np.abs(g), 300)):
        tiny = 2.0 ** -38 * np.abs(g).max() * (np.abs(w).max() if n == 260 else np.abs(xk).max()) * n + 1e-44
        assert (np.abs(got.to_numpy() - ref) <= (27 + n / 64) * U * mag + tiny).all()


def test_jacobian_of_a_checkpointed_layer(nd):
    x, w, b, _ = layer_case(3, 5, 4, 21)
    X, W, B = (nd.Array(a, requires_grad=True) for a in (x, w, b))
    nd.nn.linear(X, W, B, "tanh", checkpoint=True).backward()
    y = np.tanh(x.astype(np.float64) @ w + b)
    jx = np.einsum("in,kn,ij->injk", 1 - y * y, w, np.eye(3))
    jw = np.einsum("in,ik,nm->inkm", 1 - y * y, x, np.eye(4))
    jb = np.einsum("in,nm->inm", 1 - y * y, np.eye(4))
    assert np.abs(X.grad().to_numpy() - jx).max() <= 1e-5
    assert np.abs(W.grad().to_numpy() - jw).max() <= 1e-5
    assert np.abs(B.grad().to_numpy()[:, :, 0] - jb).max() <= 1e-5


def test_an_input_batch_is_not_remembered(nd):
    """The layer's 8-bit copy of a leaf goes with the graph: the leaf holds nothing of it."""
    x, w, b, g = layer_case(2000, 512, 16, 22)
    X, W = nd.Array(x), nd.Array(w, requires_grad=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    out = nd.nn.linear(X, W, checkpoint=True)
    held = torch.cuda.memory_allocated() - before
    assert held >= 2000 * 512
    del out
    import gc
    gc.collect()
    assert torch.cuda.memory_allocated() - before < 2000 * 512


def test_nan_and_infinite_activations(nd):
    """A row with a NaN or an infinity spoils the weight gradient's rows that it reaches and no other row of dx."""
    x, w, b, g = layer_case(40, 33, 34, 13)
    x[3, 5], x[7, 6] = np.nan, np.inf
    X, W = nd.Array(x, requires_grad=True), nd.Array(w, requires_grad=True)
    out = nd.nn.linear(X, W, nd.Array(b), checkpoint=True)
    y = out.to_numpy()
    assert np.isnan(y[3]).all() and not np.isfinite(y[7]).any() and np.isfinite(np.delete(y, [3, 7], 0)).all()
    nd.sum(out * nd.Array(g)).backward()
    dw = W.grad().to_numpy()
    assert np.isnan(dw[[5, 6]]).all() and np.isfinite(np.delete(dw, [5, 6], 0)).all()
    assert np.isfinite(X.grad().to_numpy()).all()


def test_trunk_and_head_together(nd):
    """A network whose activations are held in 8 bits and whose loss never holds the logits, trained with
    Adam: one step's gradients against the formula, and a captured step that replays with the bits of
    the step run op by op."""
    from endia_b200.utils.general import CapturedStep
    r = rng(15)
    dims, V, batch = [24, 96, 96, 48], 1500, 200
    x = r.standard_normal((batch, dims[0])).astype(np.float32)
    t = r.integers(0, V, batch).astype(np.float32)
    t[::7] = -1
    Ws = [(r.standard_normal((dims[i], dims[i + 1])) / np.sqrt(dims[i])).astype(np.float32) for i in range(3)]
    bs = [(r.standard_normal(dims[i + 1]) * 0.1).astype(np.float32) for i in range(3)]
    H = (r.standard_normal((dims[-1], V)) * (2 / np.sqrt(dims[-1]))).astype(np.float32)

    def make():
        W, B = [nd.Array(w.copy(), requires_grad=True) for w in Ws], [nd.Array(b.copy(), requires_grad=True) for b in bs]
        head = nd.Array(H.copy(), requires_grad=True)
        X, T = nd.Array(x), nd.Array(t)
        args = [X, None] + [p for wb in zip(W, B) for p in wb]
        opt = nd.optim.Adam(args[2:] + [head], lr=1e-2)

        def fn(update=True):
            z = nd.nn.mlp(args, activation="relu", checkpoint=True)
            loss = nd.linear_cross_entropy(z, head, T)
            loss.backward()
            if update:
                opt.step()
                loss.zero_grad()
            return loss, z
        return args[2:] + [head], opt, fn
    params, opt, fn = make()
    # the float32 activations of the forward pass
    hidden, h = [], nd.Array(x)
    for i in range(3):
        h = nd.nn.linear(h, params[2 * i], params[2 * i + 1], "relu" if i < 2 else None, checkpoint=True)
        hidden.append(h.to_numpy())
    fn(update=False)
    got = [p.grad().to_numpy() for p in params]
    z, live = hidden[-1].astype(np.float64), t >= 0
    l = z @ H.astype(np.float64)
    p = np.exp(l - l.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    p[np.arange(batch), np.maximum(t, 0).astype(int)] -= 1
    d = p * (live / live.sum())[:, None]
    grads, _ = mlp_reference(Ws, bs, x, "relu", d @ H.astype(np.float64).T, hidden)
    for a, ref in zip(got, grads + [z.T @ d]):
        assert np.linalg.norm(a.reshape(ref.shape) - ref) <= 1e-5 * np.linalg.norm(ref)
    # replayed against op by op
    pa, oa, fa = make()
    pb, ob, fb = make()
    step = CapturedStep(lambda: fa()[0], warmup=1, optimizers=[oa])
    for q, o in ((pa, oa), (pb, ob)):
        src = [v for wb in zip(Ws, bs) for v in wb] + [H]
        for arr, v in zip(q, src):
            arr.buf.copy_(torch.from_numpy(v.reshape(-1)))
            nd._array.drop_operand_parts(arr)
        o.reset_state()
    a, c = step().to_numpy(), fb()[0].to_numpy()
    assert np.array_equal(a, c)
    for _ in range(3):
        a, c = step().to_numpy(), fb()[0].to_numpy()
    assert abs(a[0] - c[0]) <= 1e-5 * abs(c[0])      # (Adam's bias corrections: device against host rounding)
    for u, v in zip(pa, pb):
        assert np.abs(u.to_numpy() - v.to_numpy()).max() <= 1e-5
    step.release()


def test_from_torch_without_a_copy(nd):
    from endia_b200.utils.array_conversions import from_torch, to_torch
    t = torch.arange(12, dtype=torch.float32, device="cuda").reshape(3, 4)
    a = from_torch(t, copy=False)
    assert a.shape() == [3, 4] and not a.requires_grad() and a.data_ptr() == t.data_ptr()
    t += 1
    assert np.array_equal(a.to_numpy(), np.arange(12, dtype=np.float32).reshape(3, 4) + 1)
    assert to_torch(a, copy=False).data_ptr() == t.data_ptr()
    z = torch.ones(3, dtype=torch.complex64, device="cuda")
    assert from_torch(z, requires_grad=True, copy=False).is_complex()
    for bad in (t.t(), t.double(), t.cpu(), t[:, ::2]):
        with pytest.raises(nd.EndiaError):
            from_torch(bad, copy=False)
    assert from_torch(t.t()).to_numpy().shape == (4, 3)


def test_c_abi_refusals(nd):
    L = nd._lib.lib
    buf = torch.zeros(1 << 16, device="cuda")
    p = buf.data_ptr()
    before = L.endia_b200_launch_count()
    assert L.endia_b200_keep8(p, 3, 2, 4, 0, p, None) == nd._lib.EINVAL          # leading dimension
    assert L.endia_b200_keep8(None, 4, 2, 4, 0, p, None) == nd._lib.EINVAL
    assert L.endia_b200_keep8(p, 4, 2, 4, 0, p + 16, None) == nd._lib.EINVAL      # alignment
    assert L.endia_b200_keep8(p, 4, -2, 4, 0, p, None) == nd._lib.EINVAL
    assert L.endia_b200_keep8_read(None, 2, 4, p, None) == nd._lib.EINVAL
    for a in ((p, 3, p, 8, None, 0, 2, 8, 4), (p, 4, p, 7, None, 0, 2, 8, 4), (None, 4, p, 8, None, 0, 2, 8, 4), (p, 4, None, 8, None, 0, 2, 8, 4),
              (p, 4, p, 8, None, 9, 2, 8, 4), (p, 4, p, 8, None, 0, -2, 8, 4), (p, 4, p, 8, None, 0, 2, 8, 0)):
        assert L.endia_b200_linear_keep_fwd(*a, p, p, 0, p, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_keep_fwd(p, 4, p, 8, None, 0, 2, 8, 4, p, p, 0, None, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_keep_fwd(p, 4, p, 8, None, 0, 1 << 28, 8, 4, p, p, 0, p, None) == nd._lib.ELIMIT
    assert L.endia_b200_linear_keep_bwd(None, p, 8, None, None, 0, p, 2, 8, 4, p, p, p, p, None) == nd._lib.EINVAL
    assert L.endia_b200_linear_keep_bwd(p, p, 8, None, None, 2, p, 2, 8, 4, p, p, p, p, None) == nd._lib.EINVAL     # act without out
    assert L.endia_b200_linear_keep_bwd(p, p, 8, None, None, 0, None, 2, 8, 4, p, p, p, p, None) == nd._lib.EINVAL
    assert L.endia_b200_launch_count() == before
