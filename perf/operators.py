"""The operators that train a network with a large output vocabulary in little memory, as they are measured.

linear_cross_entropy: softmax cross entropy of x @ W + b against class numbers, with the gradients of x, W and b,
computed in pieces of the vocabulary (no array of all the logits is kept).

checkpointed linear layer: a layer that keeps its input for the backward pass in 8 bits (signed integers with one
power-of-two scale per 32 features) and forms its weight gradient from them.

`run` computes the plain form with elementary operations in float32, or, where `own` is set, makes the framework's
calls. `exact` gives the same outputs in float64."""
import math

import torch

own = False

IGNORED = -1.0     # a target below zero: the row takes no part (padding)
BLOCK = 32         # features that share a scale in the 8-bit form


def listed():
    def lce(name, rows, features, classes, mode, ignored=0.0, bias=True):
        return {"name": name, "op": "linear_cross_entropy", "rows": rows, "features": features, "classes": classes,
                "mode": mode, "ignored": ignored, "bias": bias}

    def kept(name, rows, features, outputs):
        return {"name": name, "op": "checkpointed_linear", "rows": rows, "features": features, "outputs": outputs}

    return [
        # the batch and the width of the smallest network of the tests: launches and host work count
        lce("lce step 32x64x512", 32, 64, 512, "mean"),
        # scores of a few rows (one candidate each), no gradient: one pass over the weights
        lce("lce score 8x1024x32768", 8, 1024, 32768, "rows", bias=False),
        # an ordinary training step
        lce("lce step 2048x1024x32768", 2048, 1024, 32768, "mean"),
        # odd sizes, a tenth of the rows is padding
        lce("lce step 1537x1000x50001", 1537, 1000, 50001, "mean", ignored=0.1),
        # evaluation of a large batch: the loss alone
        lce("lce loss 8192x1024x65536", 8192, 1024, 65536, "loss", ignored=0.1),
        # a very large vocabulary
        lce("lce step 4096x1024x131072", 4096, 1024, 131072, "mean", bias=False),
        # the batch and the width of the benchmark's network
        lce("lce step 8192x4096x32768", 8192, 4096, 32768, "sum"),
        # the smallest layer of the tests
        kept("kept layer 32x64x64", 32, 64, 64),
        # odd sizes
        kept("kept layer 1001x777x333", 1001, 777, 333),
        # one rank's share of the benchmark's batch at 8 ranks
        kept("kept layer 1024x4096x4096", 1024, 4096, 4096),
        # the benchmark's first and middle layers
        kept("kept layer 8192x1024x4096", 8192, 1024, 4096),
        kept("kept layer 8192x4096x4096", 8192, 4096, 4096),
    ]


def _log_size(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:      # half of the sizes are round, as widths and batches often are
        step = 8 if n < 256 else 64 if n < 4096 else 256
        n = max(step, n // step * step)
    return max(low, min(high, n))


def draw(rng):
    if rng.random() < 0.6:
        while True:
            rows, features, classes = _log_size(rng, 1, 8192), _log_size(rng, 16, 4096), _log_size(rng, 64, 131072)
            if rows * features * classes <= 8192 * 4096 * 32768 and features * classes <= 4096 * 65536 and \
                    rows * classes <= 4096 * 131072:
                break
        return {"op": "linear_cross_entropy", "rows": rows, "features": features, "classes": classes,
                "mode": rng.choice(["mean", "mean", "sum", "loss", "rows"]),
                "ignored": rng.choice([0.0, 0.1, 0.5]) if rows > 4 else 0.0, "bias": rng.random() < 0.6}
    return {"op": "checkpointed_linear", "rows": _log_size(rng, 1, 16384), "features": _log_size(rng, 16, 4096),
            "outputs": _log_size(rng, 16, 4096)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * scale

    rows, features = case["rows"], case["features"]
    if case["op"] == "linear_cross_entropy":
        classes = case["classes"]
        # hidden states of unit size; weights that give logits of a few units, as in a network half trained
        x = normal(rows, features)
        weight = normal(features, classes, scale=2.0 / math.sqrt(features))
        bias = normal(classes, scale=0.5) if case["bias"] else None
        # frequent classes have low numbers
        u = torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)
        target = torch.floor(classes * u ** 3).clamp_(0, classes - 1).to(torch.float32)
        if case["ignored"]:
            drop = torch.rand(rows, generator=g, device="cuda") < case["ignored"]
            drop[0] = False
            target = torch.where(drop, torch.full_like(target, IGNORED), target)
        return {"case": case, "x": x, "weight": weight, "bias": bias, "target": target}
    outputs = case["outputs"]
    # the layer below ends in a ReLU: z is its sum before it; some features are larger than others
    spread = torch.exp(normal(features, scale=0.7))
    return {"case": case, "z": normal(rows, features) * spread,
            "weight": normal(features, outputs, scale=1.0 / math.sqrt(features)),
            "bias": normal(outputs, scale=0.1), "target": normal(rows, outputs)}


def run(state):
    lce = state["case"]["op"] == "linear_cross_entropy"
    if own:
        return _own_cross_entropy(state) if lce else _own_checkpointed(state)
    return _plain_cross_entropy(state) if lce else _plain_checkpointed(state)


# ------------------------------------------------------------------------------------- the framework's calls
def _own_cross_entropy(state):
    import endia_b200 as nd
    from endia_b200.utils.array_conversions import from_torch, to_torch
    mode = state["case"]["mode"]
    train = mode in ("mean", "sum")
    x = from_torch(state["x"], requires_grad=train, copy=False)
    weight = from_torch(state["weight"], requires_grad=train, copy=False)
    bias = None if state["bias"] is None else from_torch(state["bias"], requires_grad=train, copy=False)
    target = from_torch(state["target"], requires_grad=False, copy=False)
    reduction = {"mean": "mean", "sum": "sum", "loss": "mean", "rows": "none"}[mode]
    loss = nd.linear_cross_entropy(x, weight, target, bias=bias, reduction=reduction)
    if not train:
        return [to_torch(loss, copy=False)]
    loss.backward()
    params = [x, weight] + ([] if bias is None else [bias])
    return [to_torch(loss, copy=False)] + [to_torch(p.grad(), copy=False) for p in params]


def _own_checkpointed(state):
    import endia_b200 as nd
    from endia_b200.utils.array_conversions import from_torch, to_torch
    z = from_torch(state["z"], requires_grad=True, copy=False)
    weight = from_torch(state["weight"], requires_grad=True, copy=False)
    bias = from_torch(state["bias"], requires_grad=True, copy=False)
    target = from_torch(state["target"], requires_grad=False, copy=False)
    h = nd.relu(z)
    out = nd.nn.linear(h, weight, bias, checkpoint=True)
    nd.keep8(h)          # from here on the activations are held in 8 bits
    loss = nd.mse(out, target)
    loss.backward()
    return [to_torch(a, copy=False) for a in (loss, z.grad(), weight.grad())] + \
        [to_torch(bias.grad(), copy=False).reshape(-1)]


# ------------------------------------------------------------------------------------------- the plain forms
def _plain_cross_entropy(state):
    x, weight, bias, target = state["x"], state["weight"], state["bias"], state["target"]
    mode = state["case"]["mode"]
    counted = target >= 0
    index = target.clamp(min=0).to(torch.int64).unsqueeze(1)
    logits = torch.matmul(x, weight)
    if bias is not None:
        logits = logits + bias
    top = logits.amax(dim=1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    rows = (top + torch.log(total) - logits.gather(1, index)).squeeze(1)
    rows = torch.where(counted, rows, torch.zeros_like(rows))
    if mode == "rows":
        return [rows]
    count = counted.sum().to(torch.float32)
    loss = (rows.sum() if mode == "sum" else rows.sum() / count).reshape(1)
    if mode == "loss":
        return [loss]
    weight_of_row = counted.to(torch.float32)
    if mode == "mean":
        weight_of_row = weight_of_row / count
    d = e / total
    d.scatter_add_(1, index, torch.full_like(rows, -1.0).unsqueeze(1))
    d = d * weight_of_row.unsqueeze(1)
    out = [loss, torch.matmul(d, weight.t()), torch.matmul(x.t(), d)]
    return out if bias is None else out + [d.sum(dim=0).reshape(1, -1)]


def _blocks_of(h):
    """[rows, blocks, BLOCK], the last block filled up with zeros."""
    rows, features = h.shape
    n = -(-features // BLOCK)
    return torch.nn.functional.pad(h, (0, n * BLOCK - features)).reshape(rows, n, BLOCK)


def _plain_checkpointed(state):
    z, weight, bias, target = state["z"], state["weight"], state["bias"], state["target"]
    h = torch.where(z > 0, z, torch.zeros_like(z))
    out = torch.matmul(h, weight) + bias
    diff = out - target
    loss = (diff * diff).sum().reshape(1) / diff.numel()
    g = diff * (2.0 / diff.numel())
    # 8 bits: the smallest power of two with which no value of the block rounds beyond 127; a value that is not
    # zero does not become zero
    b = _blocks_of(h)
    fraction, exponent = torch.frexp(b.abs().amax(dim=2, keepdim=True))
    exponent = exponent - 7 + (fraction * 128.0 >= 127.5).to(torch.int32)
    v = torch.ldexp(b, -exponent)
    q = torch.round(v)
    q = torch.where((q == 0) & (v != 0), torch.sign(v), q)
    kept = torch.ldexp(q, exponent).reshape(h.shape[0], -1)[:, :h.shape[1]]
    dh = torch.matmul(g, weight.t())
    return [loss, torch.where(z > 0, dh, torch.zeros_like(dh)), torch.matmul(kept.t(), g), g.sum(dim=0)]


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear_cross_entropy":
        return _exact_cross_entropy(s, case["mode"])
    return _exact_checkpointed(s)


def _exact_cross_entropy(s, mode):
    keep = torch.nonzero(s["target"] >= 0).squeeze(1)
    x, weight = s["x"].double()[keep], s["weight"].double()
    t = s["target"][keep].long()
    logits = x @ weight
    if s["bias"] is not None:
        logits += s["bias"].double()
    logp = torch.log_softmax(logits, dim=1)
    del logits
    each = torch.arange(t.numel(), device=t.device)
    nll = -logp[each, t]
    if mode == "rows":
        full = torch.zeros(s["target"].numel(), dtype=torch.float64, device=t.device)
        full[keep] = nll
        return [full]
    scale = 1.0 if mode == "sum" else 1.0 / t.numel()
    loss = (nll.sum() * scale).reshape(1)
    if mode == "loss":
        return [loss]
    d = logp.exp_()
    d[each, t] -= 1.0
    d *= scale
    dx = torch.zeros(s["x"].shape, dtype=torch.float64, device=t.device)
    dx[keep] = d @ weight.t()
    out = [loss, dx, x.t() @ d]
    return out if s["bias"] is None else out + [d.sum(0, keepdim=True)]


def _exact_checkpointed(s):
    z, weight, bias, target = (s[k].double() for k in ("z", "weight", "bias", "target"))
    h = z.clamp(min=0)
    diff = h @ weight + bias - target
    g = diff * 2 / diff.numel()
    rows, features = h.shape
    pad = (-features) % BLOCK
    b = torch.cat([h, h.new_zeros(rows, pad)], dim=1).view(rows, -1, BLOCK)
    top = b.amax(dim=2, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=1e-300))) - 6
    e = torch.where(top / torch.exp2(e) >= 128, e + 1, e)       # (log2 next to a power of two)
    e = torch.where(top / torch.exp2(e) < 64, e - 1, e)
    e = torch.where(top / torch.exp2(e) >= 127.5, e + 1, e)
    unit = torch.where(top > 0, torch.exp2(e), torch.ones_like(e))
    q = torch.round(b / unit)
    q[(q == 0) & (b > 0)] = 1.0
    kept = (q * unit).view(rows, -1)[:, :features]
    return [(diff * diff).mean().reshape(1), (g @ weight.t()) * (z > 0), kept.t() @ g, g.sum(0)]


# ------------------------------------------------------------------------------------------- what it must do
def work(case):
    rows, features = case["rows"], case["features"]
    if case["op"] == "linear_cross_entropy":
        classes = case["classes"]
        product = 2.0 * rows * features * classes
        inputs = rows * features + features * classes + (classes if case["bias"] else 0) + rows
        if case["mode"] in ("loss", "rows"):
            return {"bytes": 4.0 * (inputs + (rows if case["mode"] == "rows" else 1)), "flops": product}
        return {"bytes": 4.0 * (2 * inputs - rows + 1), "flops": 3.0 * product}
    outputs = case["outputs"]
    return {"bytes": 4.0 * (2 * rows * features + 2 * features * outputs + rows * outputs + 2 * outputs + 1),
            "flops": 6.0 * rows * features * outputs}
