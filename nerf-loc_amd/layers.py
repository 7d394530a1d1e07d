"""Layers of networks of any shape as single kernels, with gradients: what NeRF evaluates layer by layer when the fused
renderer kernels do not cover it (other depths and widths, residual trunks), usable on their own.

  linear(x, weight, bias, activation, residual)   act(x W^T + b) + r; x may be two pieces side by side (a skip connection)
  add_rms_norm(x, weight, residual)               the residual addition and the root-mean-square norm behind it
  add_rms_norm_q8(x, weight, residual)            the same with an 8-bit output and one scale a row
  linear_q8(xq, x_scale, wq, w_scale, ...)        the linear layer on such operands
  quantize_weight(weight)                         a weight matrix as (wq, w_scale)

Tensors live on one GPU and share one type (float32, bfloat16, float16); sums, norms and scales are float32.  Leading
dimensions are free.  The kernels run on the current stream of the tensors' device, allocate nothing but their results
and scratch through torch, and can be captured in a graph (a training step only once the results of eager steps on the
same parameters are gone: torch accumulates a leaf's gradient on the stream of its first living graph).  Gradients are
computed once (no second derivatives), and torch.autocast does not change the types here.
"""
import torch

from . import hip


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _tensors(**named):
    for name, t in named.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))


def _flat(t, name):
    """[..., n] -> [m, n] without a copy where the layout allows it."""
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch.Tensor, got %s" % (name, type(t).__name__))
    if t.dim() < 1:
        raise ValueError("%s must have at least one dimension" % name)
    return t if t.dim() == 2 else t.reshape(t.shape[:-1].numel(), t.shape[-1])


def _once(what):
    # create_graph=True would take the gradients for constants
    if torch.is_grad_enabled():
        raise NotImplementedError("%s: the kernels give first derivatives only (create_graph=True asks for the second)" % what)


class _LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x0, x1, weight, bias, residual, activation):
        operands = hip._layer_input(x0, x1, weight)
        act = hip.activation_code(activation)
        n0, n1, nw, nb, _, _ = ctx.needs_input_grad
        inner = n0 or n1 or nw or nb
        # relu without a residual: y > 0 is where its argument is, so y stands in for it
        own = act == 1 and residual is None
        y, z = hip._linear(operands, act, bias, residual, inner and act != 0 and not own)
        if inner:
            x0, ld0, k0, x1, ld1, k1, w, ldw, M, N, dt, dev = operands
            ctx.save_for_backward(x0, x1, w, y if own else z)
            ctx.plan = (ld0, k0, ld1, k1, ldw, M, N, dt, dev, act)
        return y

    @staticmethod
    def backward(ctx, gy):
        _once("linear")
        n0, n1, nw, nb, nr, _ = ctx.needs_input_grad
        dx0 = dx1 = dw = db = None
        if n0 or n1 or nw or nb:
            x0, x1, w, z = ctx.saved_tensors
            ld0, k0, ld1, k1, ldw, M, N, dt, dev, act = ctx.plan
            dx0, dx1, dw, db = hip._linear_backward((x0, ld0, k0, x1, ld1, k1, w, ldw, M, N, dt, dev), act, gy, z, n0, n1, nw, nb)
        return dx0, dx1, dw, db, gy if nr else None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual in one launch, differentiable in every tensor.

    x [..., K], or a pair ([..., K0], [..., K1]) that stands for their concatenation; weight [N, K] as nn.Linear holds it;
    bias [N]; residual [..., N] (exactly the result's shape); activation None, "relu", "gelu" (the exact one) or "silu"."""
    x0, x1 = x if isinstance(x, (tuple, list)) and len(x) == 2 else (x, None)
    a = _flat(x0, "x")
    lead = None if a is x0 else x0.shape[:-1]          # None: matrices all along
    b = r = None
    if x1 is not None:
        b = _flat(x1, "the second piece of x")
        if x1.shape[:-1] != x0.shape[:-1]:
            raise ValueError("the pieces of x have leading shapes %s and %s" % (tuple(x0.shape[:-1]), tuple(x1.shape[:-1])))
    if residual is not None:
        r = _flat(residual, "residual")
        if residual.shape[:-1] != x0.shape[:-1]:
            raise ValueError("residual has leading shape %s, x %s" % (tuple(residual.shape[:-1]), tuple(x0.shape[:-1])))
    _tensors(weight=weight, bias=bias)
    if _wants_grad(a, b, weight, bias, r):
        y = _LinearFn.apply(a, b, weight, bias, r, "none" if activation is None else activation)
    else:
        y, _ = hip.linear(a, weight, bias, activation, r, b)
    return y if lead is None else y.reshape(lead + y.shape[-1:])


class _AddNormFn(torch.autograd.Function):
    """(y, h) with a residual, y alone without one (h is x then, and its gradient reaches x by itself)."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        inner = any(ctx.needs_input_grad[:3])
        y, h, rstd = hip.add_rms_norm(x, weight, residual, eps, want_h=residual is not None, want_rstd=inner)
        ctx.two = residual is not None
        if inner:
            ctx.save_for_backward(h if ctx.two else x, weight, rstd)
        ctx.set_materialize_grads(False)
        return (y, h) if ctx.two else y

    @staticmethod
    def backward(ctx, gy, gh=None):
        _once("add_rms_norm")
        nx, nw, nr, _ = ctx.needs_input_grad
        if gy is None:
            zero = None
            if nw and gh is not None:
                zero = torch.zeros_like(ctx.saved_tensors[1])
            return gh if nx else None, zero, gh if nr else None, None
        h, weight, rstd = ctx.saved_tensors
        dx, dw = hip.add_rms_norm_backward(gy, h, weight, rstd, gh, want_x=nx or nr, want_w=nw)
        return dx if nx else None, dw, dx if nr else None, None


def add_rms_norm(x, weight, residual=None, eps=1e-6):
    """h = x + residual and y = weight h / sqrt(mean(h^2) + eps) over the last dimension, in one pass.  Returns (y, h);
    without a residual h is x itself.  Differentiable in x, weight and residual; at most 32768 columns.

    In 16-bit types y comes from the float32 sum, h is that sum rounded, and the backward starts from the rounded h."""
    _tensors(x=x, weight=weight, residual=residual)
    a = _flat(x, "x")
    r = None
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("residual %s does not match x %s" % (tuple(residual.shape), tuple(x.shape)))
        r = _flat(residual, "residual")
    if _wants_grad(a, weight, r):
        out = _AddNormFn.apply(a, weight, r, float(eps))
        y, h = out if r is not None else (out, x)
    else:
        y, h, _ = hip.add_rms_norm(a, weight, r, eps, want_h=r is not None)
        h = x if h is None else h
    return (y, h) if x.dim() == 2 else (y.reshape(x.shape), h.reshape(x.shape))


def _no_grad(what, *tensors):
    if _wants_grad(*tensors):
        raise NotImplementedError("%s has no gradient (8-bit numbers are for inference): call it under torch.no_grad()" % what)


def add_rms_norm_q8(x, weight, residual=None, eps=1e-6):
    """add_rms_norm with y in 8 bits: returns (q, scale, h), q float8_e4m3fn like x and scale float32 [...], y = scale q.
    scale = max(max|y| / 448, 2^-126) of its row; a row with an infinity or NaN reads back as NaN."""
    _tensors(x=x, weight=weight, residual=residual)
    _no_grad("add_rms_norm_q8", x, weight, residual)
    a = _flat(x, "x")
    r = None
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError("residual %s does not match x %s" % (tuple(residual.shape), tuple(x.shape)))
        r = _flat(residual, "residual")
    q, scale, h = hip.add_rms_norm(a, weight, r, eps, want_h=r is not None, q8=True)
    if h is None:
        h = a
    return (q, scale, h) if a is x else (q.reshape(x.shape), scale.reshape(x.shape[:-1]), h.reshape(x.shape))


def linear_q8(xq, x_scale, wq, w_scale, bias=None, activation=None, residual=None, out_dtype=torch.bfloat16):
    """act(x W^T + bias) + residual with x = x_scale xq (xq float8_e4m3fn [..., K], x_scale float32 [...]) and
    W = w_scale wq ([N, K], [N]); bias, residual and the result are of out_dtype.  No gradient.

    Above 64 rows a 16-bit result's products are added by the 8-bit matrix instruction, eight at a time at 2^-13 of the
    eight's largest, the eights in float32; a float32 result, and few rows, add every product in float32."""
    _tensors(xq=xq, x_scale=x_scale, wq=wq, w_scale=w_scale, bias=bias, residual=residual)
    _no_grad("linear_q8", x_scale, w_scale, bias, residual)
    a = _flat(xq, "xq")
    lead = xq.shape[:-1]
    if x_scale.shape != lead:
        raise ValueError("x_scale must be of shape %s, got %s" % (tuple(lead), tuple(x_scale.shape)))
    if residual is not None and residual.shape[:-1] != lead:
        raise ValueError("residual has leading shape %s, xq %s" % (tuple(residual.shape[:-1]), tuple(lead)))
    y = hip.linear_q8(a, x_scale if a is xq else x_scale.reshape(-1), wq, w_scale, bias, activation,
                      None if residual is None else _flat(residual, "residual"), out_dtype)
    return y if a is xq else y.reshape(lead + y.shape[-1:])


@torch.no_grad()
def quantize_weight(weight):
    """(wq float8_e4m3fn [N, K], w_scale float32 [N]) for linear_q8, made once per weight version with torch."""
    _tensors(weight=weight)
    if weight.dim() != 2 or weight.shape[1] < 1:
        raise ValueError("weight must be a matrix with columns, got %s" % (tuple(weight.shape),))
    w = weight.float()
    scale = (w.abs().amax(-1) / 448.0).clamp_min(2.0 ** -126)
    return (w / scale[:, None]).to(torch.float8_e4m3fn), scale
