"""reference ``tensorcircuit/torchnn.py:16-138``: ``QuantumNet`` (alias ``TorchLayer``), a ``torch.nn.Module``
around a quantum function ``f(inputs, *weights)``; the batch axis of the inputs is vmapped through the
hip backend (one batched plan execution, not a Python loop).

Next to it, what a hybrid model needs to be trained on measured bitstrings: ``LinearCrossEntropy`` /
``linear_cross_entropy`` (a linear head over many classes and its loss, the logits never stored) and ``Muon`` /
``muon_step`` (an optimiser for matrix-shaped weights, the circuit's ``[layers, qubits]`` angles among them)."""

import math
from typing import Any, Callable, Optional, Sequence, Tuple, Union

import torch

from . import _lib, cons, linalg
from .interfaces.torch import torch_interface

Tensor = Any


class QuantumNet(torch.nn.Module):
    def __init__(self, f: Callable[..., Any], weights_shape: Sequence[Any], initializer: Union[Any, Sequence[Any]] = None,
                 use_vmap: bool = True, vectorized_argnums: Union[int, Sequence[int]] = 0, use_interface: bool = True,
                 use_jit: bool = True, enable_dlpack: bool = False):
        super().__init__()
        if use_vmap:
            f = cons.backend.vmap(f, vectorized_argnums=vectorized_argnums)
        if use_interface:
            f = torch_interface(f, jit=use_jit, enable_dlpack=enable_dlpack)
        self.f = f
        if len(weights_shape) > 0 and isinstance(weights_shape[0], int):
            weights_shape = [tuple(weights_shape)]
        if initializer is not None and not isinstance(initializer, (list, tuple)):
            initializer = [initializer]
        self.q_weights = torch.nn.ParameterList()
        for k, ws in enumerate(weights_shape):
            init = torch.randn(tuple(ws)) if initializer is None else torch.as_tensor(initializer[k]).clone()
            self.q_weights.append(torch.nn.Parameter(init.to(torch.float32 if cons.rdtypestr == "float32" else torch.float64)))

    def forward(self, *inputs: Tensor) -> Tensor:
        return self.f(*inputs, *self.q_weights)


TorchLayer = QuantumNet


# ----------------------------------------------------------------------------- linear head with its loss
_REDUCTIONS = ("none", "sum", "mean")


def _row_stride(x):
    """elements between the rows of an operand; one row may carry any number there (an expanded one: 0)"""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _lce_raw(h, w, target, bias, ignore_index, reduction, for_grad):
    """(loss, stat): h [T, D], w [V, D], target [T]; loss is per row for reduction "none".  stat, what the gradient needs: the
    rows' log sums in two floats, how many rows count, and (not "none") the rows' losses"""
    t, d = h.shape
    v = w.shape[0]
    code = linalg._train_code(h)
    per_row = reduction == "none"
    loss = torch.empty(t if per_row else (), dtype=torch.float32, device=h.device)
    if t == 0:
        stat = torch.empty(1, dtype=torch.float32, device=h.device)
        if not per_row:
            loss.fill_(math.nan if reduction == "mean" else 0.0)
        return loss, stat.zero_()
    L = _lib.lib()
    hp, hs, wp, ws = h.data_ptr(), _row_stride(h), w.data_ptr(), _row_stride(w)
    nbytes = L.tcmi_lce_work_bytes(hp, hs, wp, ws, t, d, v, code, _lib.LCE_FOR_GRAD if for_grad else _lib.LCE_ALONE)
    if nbytes < 0:
        raise ValueError(f"linear_cross_entropy: {t} rows, {d} features, {v} classes are out of range")
    floats = 2 * t + 2 if per_row else 3 * t + 1 + (t + 1) % 2        # even: vmap cuts stacks of them, and the log sums need 8 bytes
    if for_grad:
        stat = torch.empty(floats, dtype=torch.float32, device=h.device)
        work = torch.empty(nbytes, dtype=torch.uint8, device=h.device)
        lse = stat.data_ptr()
    else:                            # nobody needs them after the call: the workspace's tail
        stat, work = None, torch.empty(nbytes + 4 * floats, dtype=torch.uint8, device=h.device)
        lse = work.data_ptr() + nbytes
    with linalg._on(h.device):
        _lib.check(L.tcmi_linear_cross_entropy(
            hp, hs, wp, ws, None if bias is None else bias.data_ptr(), target.data_ptr(), ignore_index, t, d, v, lse,
            loss.data_ptr() if per_row else lse + 4 * (2 * t + 1), None if per_row else loss.data_ptr(), lse + 8 * t,
            int(reduction == "mean"), int(for_grad), work.data_ptr(), nbytes, code, linalg._raw_stream(h.device)),
            "tcmi_linear_cross_entropy")
    return loss, stat


def _lce_grad_raw(h, w, target, bias, stat, dloss, ignore_index, reduction, need):
    t, d = h.shape
    v = w.shape[0]
    dev = h.device
    outs = [torch.empty(x.shape, dtype=x.dtype, device=dev) if n else None for x, n in zip((h, w, bias), need)]
    if t == 0:
        return tuple(torch.empty(0, device=dev) if o is None else o.zero_() for o in outs)
    code = linalg._train_code(h)
    dloss = dloss.to(torch.float32).resolve_neg().contiguous()        # a view that only carries its sign (of an imaginary part)
    L = _lib.lib()
    hp, hs, wp, ws, lse = h.data_ptr(), _row_stride(h), w.data_ptr(), _row_stride(w), stat.data_ptr()
    nbytes = L.tcmi_lce_work_bytes(hp, hs, wp, ws, t, d, v, code, _lib.LCE_GRAD)
    work = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    ptrs = [None if o is None else o.data_ptr() for o in outs]
    with linalg._on(dev):
        _lib.check(L.tcmi_linear_cross_entropy_grad(
            hp, hs, wp, ws, None if bias is None else bias.data_ptr(), target.data_ptr(), ignore_index, t, d, v, lse,
            dloss.data_ptr(), int(reduction == "none"), lse + 8 * t if reduction == "mean" else None, *ptrs, work.data_ptr(),
            nbytes, code, linalg._raw_stream(dev)), "tcmi_linear_cross_entropy_grad")
    return tuple(torch.empty(0, device=dev) if o is None else o for o in outs)


def _vmap_loop(fn, info, in_dims, args):
    """one call per batch element: the operators take one head a call"""
    outs = [fn(*[a.select(d, i) if d is not None else a for a, d in zip(args, in_dims)]) for i in range(info.batch_size)]
    return tuple(torch.stack([o[k] for o in outs]) for k in range(len(outs[0]))), tuple(0 for _ in outs[0])


class _LinearCrossEntropyEager(torch.autograd.Function):
    """the same outside torch.func, whose calling convention costs two signature look-ups a call (60 us)"""

    @staticmethod
    def forward(ctx, h, w, target, bias, ignore_index, reduction):
        loss, stat = _lce_raw(h, w, target, bias, ignore_index, reduction, True)
        ctx.ignore_index, ctx.reduction = ignore_index, reduction
        ctx.save_for_backward(h, w, target, bias, stat)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        h, w, target, bias, stat = ctx.saved_tensors
        need = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3])
        grad = _LinearCrossEntropyGrad.apply if torch.is_grad_enabled() else _lce_grad_raw
        dh, dw, db = grad(h, w, target, bias, stat, dloss, ctx.ignore_index, ctx.reduction, need)
        return dh if need[0] else None, dw if need[1] else None, None, db if need[2] else None, None, None


class _LinearCrossEntropy(torch.autograd.Function):
    generate_vmap_rule = False

    @staticmethod
    def forward(h, w, target, bias, ignore_index, reduction):
        return _lce_raw(h, w, target, bias, ignore_index, reduction, True)

    @staticmethod
    def vmap(info, in_dims, *args):
        return _vmap_loop(_LinearCrossEntropy.apply, info, in_dims, args)

    @staticmethod
    def setup_context(ctx, inputs, output):
        h, w, target, bias, ctx.ignore_index, ctx.reduction = inputs
        ctx.mark_non_differentiable(output[1])
        ctx.save_for_backward(h, w, target, bias, output[1])

    @staticmethod
    def backward(ctx, dloss, _):
        h, w, target, bias, stat = ctx.saved_tensors
        need = (ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.needs_input_grad[3] and bias is not None)
        dh, dw, db = _LinearCrossEntropyGrad.apply(h, w, target, bias, stat, dloss, ctx.ignore_index, ctx.reduction, need)
        return dh if need[0] else None, dw if need[1] else None, None, db if need[2] else None, None, None


class _LinearCrossEntropyGrad(torch.autograd.Function):
    generate_vmap_rule = False

    @staticmethod
    def forward(h, w, target, bias, stat, dloss, ignore_index, reduction, need):
        return _lce_grad_raw(h, w, target, bias, stat, dloss, ignore_index, reduction, need)

    @staticmethod
    def vmap(info, in_dims, *args):
        return _vmap_loop(_LinearCrossEntropyGrad.apply, info, in_dims[:6] + (None,) * 3, args)

    @staticmethod
    def setup_context(ctx, inputs, output):
        pass

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError("linear_cross_entropy is differentiable once")


def linear_cross_entropy(input: Tensor, weight: Tensor, target: Tensor, bias: Optional[Tensor] = None, ignore_index: int = -100,
                         reduction: str = "mean") -> Tensor:
    """``cross_entropy(input @ weight.T + bias, target)`` without the logits: input ``[..., features]``, weight
    ``[classes, features]``, bias ``[classes]``, one dtype of float32, bfloat16, float16; target ``[...]`` int64 class numbers
    (the ``sample_int`` format of ``Circuit.sample`` for a head over bitstrings).  The loss is float32, per row of ``target``
    for ``reduction="none"``; gradients for input, weight and bias, once.

    Rows whose target is ``ignore_index`` have loss 0 and contribute nothing to any gradient, whatever they hold; the mean
    over no rows is NaN (its gradients are zero).  Any other target outside ``0 .. classes - 1`` gives NaN, in the loss and
    in the gradients (checked where the targets live, nothing is read out of range).  Classes may be masked by a bias
    of ``-inf``.  A non-finite feature or weight of a row that counts gives NaN, or where the logits it makes are ``-inf`` a
    class without probability and gradients of NaN.  float64 (``tc.set_dtype("complex128")``) is refused, and so are
    forward-mode tangents.

    The loss stores no logits.  Its gradient stores the probabilities of as many classes as 1 GiB holds, twice (a training step
    with few rows takes more than its logits would), and copies of operands that are float32 or whose rows are no whole
    number of 64 features.  ``vmap`` runs one call per element.

    A logit of a float32 head is held to ``2 ** -22`` of its terms, ``2 ** -39`` of its row's largest feature times largest weight:
    features that are ``2 ** 17`` and more apart and weighted the other way round should be brought to like sizes.  Gradients
    are held by class and feature, whatever their sizes; those of 16-bit heads multiply probabilities of 11 bits, which
    with float16 costs up to as much as the rounding of the result.

    A training step may be captured into a graph (``torch.cuda.graph``).  As with any operator, let go of eager losses of the
    same leaves first (torch ties a leaf's gradient to the stream of its oldest living graph), or capture
    ``torch.autograd.grad`` instead of ``backward()``."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
    if input.dim() < 1 or weight.dim() != 2 or input.shape[-1] != weight.shape[1]:
        raise ValueError(f"linear_cross_entropy: input {tuple(input.shape)} does not fit weight {tuple(weight.shape)}")
    if tuple(target.shape) != tuple(input.shape[:-1]):
        raise ValueError(f"linear_cross_entropy: target {tuple(target.shape)} does not fit input {tuple(input.shape)}")
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise ValueError(f"linear_cross_entropy: bias {tuple(bias.shape)} does not fit {weight.shape[0]} classes")
    if weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("linear_cross_entropy needs at least one class and one feature")
    if input.is_complex():
        raise TypeError("linear_cross_entropy needs real features (take backend.real of expectation values)")
    linalg._train_code(input)
    for name, x in (("weight", weight), ("bias", bias)):
        if x is not None and x.dtype != input.dtype:
            raise TypeError(f"linear_cross_entropy: {name} is {x.dtype}, input is {input.dtype}")
    if target.dtype != torch.int64:
        raise TypeError(f"linear_cross_entropy: target must be int64, got {target.dtype}")
    linalg._need_gpu("linear_cross_entropy", input, weight, target, bias)
    input, w = input.resolve_neg(), weight.resolve_neg()
    h = input if input.dim() == 2 else input.reshape(-1, input.shape[-1])
    # features contiguous, rows apart (a broadcast or transposed operand is copied; autograd takes its gradient back)
    h = h if h.stride(1) == 1 and h.stride(0) >= h.shape[1] else h.contiguous()
    w = w if w.stride(1) == 1 and w.stride(0) >= w.shape[1] else w.contiguous()
    b = None if bias is None else bias.resolve_neg().contiguous()
    y = (target if target.dim() == 1 else target.reshape(-1)).contiguous()
    args = (h, w, y, b, int(ignore_index), reduction)
    if not linalg._tracked(h, w, b, y):
        loss = _lce_raw(*args, False)[0]
    elif torch._C._are_functorch_transforms_active():
        loss = _LinearCrossEntropy.apply(*args)[0]
    else:
        loss = _LinearCrossEntropyEager.apply(*args)
    return loss.reshape(target.shape) if reduction == "none" else loss


class LinearCrossEntropy(torch.nn.Module):
    """A linear head over ``classes`` outcomes together with its loss, e.g. over the ``2 ** n`` bitstrings a circuit answers
    with: ``forward(features, target)`` is :func:`linear_cross_entropy` of its own weight and bias."""

    def __init__(self, features: int, classes: int, bias: bool = True, ignore_index: int = -100, reduction: str = "mean",
                 device: Any = None, dtype: Any = torch.float32):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction must be one of {_REDUCTIONS}, got {reduction!r}")
        self.ignore_index, self.reduction = ignore_index, reduction
        self.weight = torch.nn.Parameter(torch.empty(classes, features, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.empty(classes, device=device, dtype=dtype)) if bias else None
        bound = 1.0 / math.sqrt(features)
        with torch.no_grad():
            for p in self.parameters():
                p.uniform_(-bound, bound)

    def forward(self, features: Tensor, target: Tensor) -> Tensor:
        return linear_cross_entropy(features, self.weight, target, self.bias, self.ignore_index, self.reduction)


# ----------------------------------------------------------------------------- optimiser
_ADJUST = ("original", "match_rms_adamw")


def _matrix_view(t, what):
    try:
        return t.view((-1,) + tuple(t.shape[-2:]))
    except RuntimeError:
        raise ValueError(f"muon_step: the leading axes of {what} cannot be read as one batch axis") from None


def muon_step(param: Tensor, grad: Tensor, momentum_buffer: Tensor, lr: float = 1e-3, weight_decay: float = 0.1,
              momentum: float = 0.95, nesterov: bool = True, ns_coefficients: Any = linalg.NS_COEFFICIENTS, eps: float = 1e-7,
              ns_steps: int = 5, adjust_lr_fn: Optional[str] = None) -> None:
    """One step of momentum with an orthogonalised update, in place on ``param`` and ``momentum_buffer`` (float32):

        buf <- momentum buf + (1 - momentum) grad;   u = nesterov ? (1 - momentum) grad + momentum buf : buf
        param <- (1 - lr weight_decay) param - lr r newton_schulz(u)

    with ``r = sqrt(max(1, rows / cols))`` (``adjust_lr_fn`` None or "original") or ``0.2 sqrt(max(rows, cols))``
    ("match_rms_adamw").  Parameters with more than two axes are batches of matrices in their last two; float32,
    bfloat16, float16.  The momentum update, the norm, the products and the weight update are one sequence of kernels:
    no update matrix reaches memory in float32 but the carried iterate."""
    if adjust_lr_fn not in (None,) + _ADJUST:
        raise ValueError(f"adjust_lr_fn must be None or one of {_ADJUST}, got {adjust_lr_fn!r}")
    if param.dim() < 2:
        raise ValueError(f"muon_step: a parameter needs at least two axes, got {tuple(param.shape)}")
    if grad.shape != param.shape or momentum_buffer.shape != param.shape:
        raise ValueError(f"muon_step: param {tuple(param.shape)}, grad {tuple(grad.shape)} and momentum_buffer "
                         f"{tuple(momentum_buffer.shape)} must have one shape")
    if param.is_complex():
        raise TypeError("muon_step takes real parameters")
    code = linalg._train_code(param)
    if grad.dtype != param.dtype:
        raise TypeError(f"muon_step: grad is {grad.dtype}, param is {param.dtype}")
    if grad.is_sparse or momentum_buffer.dtype != torch.float32:
        raise TypeError("muon_step: needs a dense grad and a float32 momentum_buffer")
    if not (0.0 <= momentum < 1.0) or not math.isfinite(lr) or not math.isfinite(weight_decay):
        raise ValueError(f"muon_step: momentum must lie in [0, 1), lr and weight_decay be finite (got {momentum}, {lr}, {weight_decay})")
    steps, flat = linalg._ns_coefficients(ns_steps, ns_coefficients, eps)
    for name, x in (("param", param), ("momentum_buffer", momentum_buffer)):
        if x.is_neg():
            raise ValueError(f"muon_step: {name} is a view that negates its memory")
        if torch._debug_has_internal_overlap(x) == 1:
            raise ValueError(f"muon_step: {name} has elements that share memory")
    if momentum_buffer.numel() and momentum_buffer.data_ptr() in (param.data_ptr(), grad.data_ptr()):
        raise ValueError("muon_step: momentum_buffer must not share memory with param or grad")
    linalg._no_tangent(param, grad, momentum_buffer)
    linalg._need_gpu("muon_step", param, grad, momentum_buffer)
    if param.numel() == 0:
        return
    with torch.no_grad():
        p, v = _matrix_view(param.detach(), "param"), _matrix_view(momentum_buffer.detach(), "momentum_buffer")
        g = linalg._as_batch(grad.detach())
        b, m, n = p.shape
        full = int(param.dtype != torch.bfloat16)
        L, coef = _lib.lib(), linalg._host_doubles(flat)
        nbytes = L.tcmi_ns_work_bytes_coef(m, n, b, steps, coef, full, code, _lib.NS_WORK)
        if nbytes < 0:
            raise ValueError(f"muon_step: {b} matrices of {m} x {n} are out of range ({steps} steps)")
        work = torch.empty(nbytes, dtype=torch.uint8, device=p.device)
        r = 0.2 * math.sqrt(max(m, n)) if adjust_lr_fn == "match_rms_adamw" else math.sqrt(max(1.0, m / n))
        with linalg._on(p.device):
            _lib.check(L.tcmi_muon_step(
                p.data_ptr(), p.stride(1), p.stride(2), p.stride(0), g.data_ptr(), g.stride(1), g.stride(2), g.stride(0),
                v.data_ptr(), v.stride(1), v.stride(2), v.stride(0), m, n, b, float(momentum), int(bool(nesterov)),
                1.0 - float(lr) * float(weight_decay), -float(lr) * r, steps, coef, float(eps), full,
                work.data_ptr(), nbytes, code, linalg._raw_stream(p.device)), "tcmi_muon_step")
        torch.autograd.graph.increment_version(param)
        torch.autograd.graph.increment_version(momentum_buffer)


class Muon(torch.optim.Optimizer):
    """Optimiser of matrix-shaped parameters (:func:`muon_step` for each): ``QuantumNet``'s ``[layers, qubits]`` angles, the
    weight of a classical head.  Vectors (biases) belong to another optimiser and are refused.  ``step`` may be captured into a
    graph once every parameter has its momentum (after one eager step); the options of the captured step are fixed in it."""

    def __init__(self, params: Any, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95, nesterov: bool = True,
                 ns_coefficients: Any = linalg.NS_COEFFICIENTS, eps: float = 1e-7, ns_steps: int = 5,
                 adjust_lr_fn: Optional[str] = None):
        if not lr >= 0 or not weight_decay >= 0 or not 0 <= momentum < 1:
            raise ValueError(f"lr and weight_decay must not be negative, momentum must lie in [0, 1): got {lr}, {weight_decay}, {momentum}")
        linalg._ns_coefficients(ns_steps, ns_coefficients, eps)
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                                      ns_coefficients=ns_coefficients, eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn))

    def add_param_group(self, param_group: Any) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2 or p.is_complex():
                self.param_groups.pop()
                raise ValueError(f"Muon takes real parameters with at least two axes, got {tuple(p.shape)} {p.dtype}")

    def load_state_dict(self, state_dict: Any) -> None:
        super().load_state_dict(state_dict)
        # torch casts floating-point state to the parameter's dtype: the momentum stays float32
        params = [p for group in self.param_groups for p in group["params"]]
        keys = [k for group in state_dict["param_groups"] for k in group["params"]]
        for k, p in zip(keys, params):
            buf = state_dict["state"].get(k, {}).get("momentum_buffer")
            if buf is not None:
                self.state[p]["momentum_buffer"] = buf.detach().to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure: Optional[Callable[[], Any]] = None) -> Any:
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("Muon: take one step before the capture (a captured first step would clear the "
                                           "momentum on every replay)")
                    state["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
                muon_step(p, p.grad, state["momentum_buffer"], **{k: group[k] for k in self.defaults})   # not a scheduler's keys
        return loss
