"""Losses (endia/functional/loss_ops/): mse, and the cross entropy of a linear layer over a large
vocabulary."""
from .. import _lib
from .._array import Array, ArrayShape, alloc, stream
from ..autograd import state as _state
from ._utils import op_array, setup_shape_and_data, contiguous
from .binary_ops import sub, mul, add, fused_binary, _matrix_layout
from .reduce_ops import sum


def _mse_composed(pred, target):
    diff = sub(pred, target)
    return sum(mul(diff, diff)) / float(pred.size())


def mse(pred, target):
    """sum((pred - target) * (pred - target)) / pred.size(), shape [1] (loss_ops/mse_op.mojo:18-20).

    Two real contiguous arrays of one shape run as ONE fused kernel (endia_b200_mse_fwd_bwd) that
    also writes d loss / d pred = 2 (pred - target) / n, which the VJP hands on as it is: the
    reference's chain of sub, mul, reduce, div and their five VJP passes become two launches. With
    create_graph=True the VJP is the differentiable composition of the same formula. Any other
    operands use the op composition."""
    if (pred.is_complex() or target.is_complex() or pred.shape() != target.shape() or pred.size() == 0
            or not pred.is_contiguous() or not target.is_contiguous()):
        return _mse_composed(pred, target)
    n = pred.size()

    def call(curr, args):
        setup_shape_and_data(curr)
        p, t = args
        dpred = None
        if curr.requires_grad_flag:
            dpred = Array(ArrayShape(p.shape()))
            dpred.name = "mse_vjp"
            setup_shape_and_data(dpred)
        scratch = alloc((_lib.lib.endia_b200_mse_scratch_bytes(n) + 3) // 4)
        _lib.call("endia_b200_mse_fwd_bwd", p.data_ptr(), t.data_ptr(), n, 1.0, curr.data_ptr(),
                  dpred.data_ptr() if dpred is not None else None, scratch.data_ptr(), stream())
        curr._dpred = dpred

    def vjp(primals, grad, out):
        p, t = primals
        zero = Array(0)
        if _state.create_graph:
            # d/dp sum(d*d)/n = (d + d) * (grad/n): mul_op.mojo:125-128 applied to both operands of d*d
            d = sub(p, t)
            gp = mul(add(d, d), grad / float(n))
        elif getattr(grad, "_is_ones_seed", False):
            gp = out._dpred            # the seed of backward() is ones(1): nothing to multiply
        else:
            gp = fused_binary(_lib.BIN_MUL, out._dpred, grad)
        gt = zero
        if t.requires_grad():
            from .unary_ops import neg
            gt = neg(gp)
        return [gp if p.requires_grad() else zero, gt]
    return op_array(ArrayShape([1]), [pred, target], "mse", call, vjp=vjp)


_REDUCTIONS = {"mean": _lib.LOSS_MEAN, "sum": _lib.LOSS_SUM, "none": _lib.LOSS_NONE}


def _row_major(a):
    """`a` (2-D) itself when its rows are contiguous runs, else a contiguous copy, and its leading dimension."""
    if a.is_contiguous():
        return a, max(a.shape()[1], 1)
    layout = _matrix_layout(a)
    if layout is None or layout[0] != 0:
        a = contiguous(a)
        return a, max(a.shape()[1], 1)
    return a, layout[1]


_CLASS_NUMBERS = {}   # V -> [0, 1, ..., V - 1], for the composed form (never written after it is made)


def _class_numbers(V):
    from .init_ops import arange
    if V not in _CLASS_NUMBERS:
        if len(_CLASS_NUMBERS) >= 8:
            _CLASS_NUMBERS.clear()
        _CLASS_NUMBERS[V] = arange(0, V)
    return _CLASS_NUMBERS[V]


def _scratch(nbytes):
    return alloc((nbytes + 3) // 4)


def linear_cross_entropy(x, weight, target, bias=None, reduction="mean"):
    """Softmax cross entropy of the logits x @ weight + bias against class numbers:

        loss_m = log(sum_v exp(l[m, v])) - l[m, target_m]

    x (..., K), weight (K, V) as nn.linear takes it, bias (V) or None, target (...): class numbers as
    floats (the arrays here are float32, so V is at most 2^24). `reduction`: "mean" over the rows that
    count (shape [1], like mse), "sum" (shape [1]) or "none" (target's shape).

    The logits are never held: forward and backward walk the vocabulary in pieces
    (endia_b200_linear_ce_fwd / _bwd), and the backward pass forms each piece's logits again.

    A negative target leaves its row out: loss 0, no gradient, whatever x holds there; a mean over no
    rows is 0. A target that is not an integer below V makes its row's loss NaN, and with it the
    gradients. The target takes no gradient. With create_graph=True (and in forward mode, and for the
    Jacobian of the row losses) the VJP is the differentiable composition of the same formula, which does hold logits, and wants finite x and
    valid targets in every row. The reference has mse only (loss_ops/mse_op.mojo:18-20)."""
    if reduction not in _REDUCTIONS:
        raise _lib.EndiaError(_lib.EINVAL, "linear_cross_entropy: unknown reduction %r" % (reduction,))
    arrays = [x, weight, target] + ([bias] if bias is not None else [])
    if any(a.is_complex() for a in arrays):
        raise _lib.EndiaError(_lib.EINVAL, "linear_cross_entropy: real arrays only")
    if target.requires_grad():
        raise _lib.EndiaError(_lib.EINVAL, "linear_cross_entropy: the target takes no gradient")
    if x.ndim() < 2 or weight.ndim() != 2 or x.shape()[-1] != weight.shape()[0] or x.shape()[:-1] != target.shape() \
            or (bias is not None and bias.shape() != [weight.shape()[1]]):
        raise _lib.EndiaError(_lib.ESHAPE, "linear_cross_entropy: incompatible shapes x %s, weight %s, target %s, bias %s" % (
            x.shape(), weight.shape(), target.shape(), bias.shape() if bias is not None else None))
    K, V = weight.shape()
    if K == 0 or V == 0:
        raise _lib.EndiaError(_lib.ESHAPE, "linear_cross_entropy: needs at least one feature and one class")
    if V > 1 << 24:
        raise _lib.EndiaError(_lib.ELIMIT, "linear_cross_entropy: at most 2^24 classes (class numbers are float32 values)")
    M = target.size()
    if x.ndim() != 2:
        from .view_ops import reshape
        x = reshape(x, [M, K])
    args = [x, weight] + ([bias] if bias is not None else [])
    mode = _REDUCTIONS[reduction]
    labels = contiguous(target)
    saved = {}

    def operands(a):
        xr, ldx = _row_major(a[0])
        wr, ldw = _row_major(a[1])
        b = contiguous(a[2]) if bias is not None else None
        # (the arrays go along so that copies live until their kernels are enqueued)
        return (xr, wr, b), (xr.data_ptr(), ldx, wr.data_ptr(), ldw, b.data_ptr() if b is not None else None,
                             labels.data_ptr(), M, K, V, mode)

    def call(curr, a):
        setup_shape_and_data(curr)
        hold, ops = operands(a)
        state = None
        if curr.requires_grad_flag:
            state = saved["state"] = alloc(_lib.lib.endia_b200_linear_ce_state_bytes(M) // 4)
        scratch = _scratch(_lib.lib.endia_b200_linear_ce_scratch_bytes(M, K, V, 0 if state is not None else 2))
        _lib.call("endia_b200_linear_ce_fwd", *ops, curr.data_ptr(), state.data_ptr() if state is not None else None,
                  scratch.data_ptr(), stream())

    def state_array(shape, offset):
        arr = Array(ArrayShape(shape, None, offset))
        arr.buf = saved["state"]
        return arr

    def row_weights(grad):
        """The incoming gradient per row, [M, 1], in differentiable ops."""
        from .comparison_ops import greater_equal, equal
        from .view_ops import reshape
        counted = greater_equal(reshape(labels, [M, 1]), Array([1]))
        if mode == _lib.LOSS_NONE:      # (leading dims of a Jacobian's seed stay in front)
            lead = grad.shape()[:grad.ndim() - target.ndim()]
            return mul(counted, reshape(contiguous(grad), lead + [M, 1]))
        if mode == _lib.LOSS_MEAN:
            from .binary_ops import div
            count = state_array([1], 0)
            grad = div(grad, add(count, equal(count, Array([1]))))
        return mul(counted, grad)

    def errors(p):
        """softmax(logits) - onehot(target), [M, V], in differentiable ops: exp(l - lse) has rows of sum
        one, and dividing by that sum carries the derivative of lse."""
        from .binary_ops import matmul, div
        from .comparison_ops import equal
        from .reduce_ops import reduce_add
        from .unary_ops import exp
        from .view_ops import reshape
        logits = matmul(p[0], p[1])
        if bias is not None:
            logits = add(logits, p[2])
        e = exp(sub(logits, state_array([M, 1], 4)))
        return sub(div(e, reduce_add(e, [1])), equal(reshape(labels, [M, 1]), _class_numbers(V)))

    def vjp(primals, grad, out):
        want = [_state.wants_grad(p) for p in primals]
        if _state.create_graph or grad.shape() != out.shape():
            from .binary_ops import matmul
            from .reduce_ops import reduce_add
            d = mul(errors(primals), row_weights(grad))
            res = [matmul(d, primals[1].T()) if want[0] else None, matmul(primals[0].T(), d) if want[1] else None]
            if bias is not None:
                res.append(reduce_add(d, [-2]) if want[2] else None)
            return res
        res = []
        for w, shape in zip(want, ([M, K], [K, V], [1, V])):
            res.append(None)
            if w:
                res[-1] = Array(ArrayShape(shape))
                setup_shape_and_data(res[-1])
        if any(want):
            g = contiguous(grad)
            hold, ops = operands(primals)
            scratch = _scratch(_lib.lib.endia_b200_linear_ce_scratch_bytes(M, K, V, 1))
            ptrs = [r.data_ptr() if w else None for r, w in zip(res, want)] + [None]
            _lib.call("endia_b200_linear_ce_bwd", *ops, g.data_ptr(), saved["state"].data_ptr(), *ptrs[:3],
                      scratch.data_ptr(), stream())
        return res

    def jvp(p, t):
        from .binary_ops import matmul
        from .init_ops import ones
        from .reduce_ops import reduce_add
        dl = add(matmul(t[0], p[1]), matmul(p[0], t[1]))
        if bias is not None:
            dl = add(dl, t[2])
        g = row_weights(ones([M]) if mode == _lib.LOSS_NONE else ones([1]))
        rows = mul(reduce_add(mul(errors(p), dl), [1]), g)
        if mode == _lib.LOSS_NONE:
            from .view_ops import reshape
            return reshape(rows, target.shape())
        return sum(rows)
    return op_array(ArrayShape(target.shape() if mode == _lib.LOSS_NONE else [1]), args, "linear_cross_entropy", call,
                    vjp=vjp, jvp=jvp)
