"""The HIP entry points as ``torch.library`` custom operators.

``torch.compile`` cannot trace a ctypes call; it can trace an opaque custom
operator that comes with a shape/dtype rule ("fake" implementation).  The
autograd nodes in ``warp``, ``scalar`` and ``complex`` therefore switch to
these operators while a graph is being captured and call the C ABI directly
otherwise (less Python overhead per call).  The reference advertises
``torch.compile`` for its torch scan only (README.md:36 of the reference).

The three forward operators carry autograd formulas of their own
(``torch.library.register_autograd``, at the end of this file), so
``torch.ops.accelerated_scan.scan_forward(gates, tokens, False)`` is
differentiable without any ``autograd.Function`` around it, in eager mode and
under ``torch.compile``.  Every operator validates its arguments itself: they
are public as ``torch.ops.accelerated_scan.*``.
"""

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _abi


def _check_dense(first: torch.Tensor, others, token_like=None, states=()) -> None:
    """All tensors of a call: device tensors on one device, contiguous, of one
    shape; ``others`` share the dtype of ``first``; ``token_like`` may be
    float32 beside complex64; ``states`` hold one element per row."""
    def fail(what):
        raise RuntimeError(f"accelerated_scan: expected {what}")

    if not first.is_cuda:
        fail("device tensors")
    if first.dim() < 1:
        fail("tensors with a sequence axis")
    for t in tuple(others) + ((token_like,) if token_like is not None else ()):
        if not t.is_cuda or t.device != first.device:
            fail("all tensors on one GPU")
        if t.shape != first.shape:
            fail(f"tensors of one shape, got {tuple(first.shape)} and {tuple(t.shape)}")
        if not t.is_contiguous():
            fail("contiguous tensors")
    if not first.is_contiguous():
        fail("contiguous tensors")
    for t in others:
        if t.dtype != first.dtype:
            fail(f"tensors of one dtype, got {first.dtype} and {t.dtype}")
    if token_like is not None:
        _abi.dtype_code(first.dtype, token_like.dtype)  # raises for unsupported combinations
    for t in states:
        if (not t.is_cuda or t.device != first.device or t.dtype != first.dtype
                or t.shape != first.shape[:-1] or not t.is_contiguous()):
            fail(f"a contiguous {first.dtype} state of shape {tuple(first.shape[:-1])} on {first.device}")


@torch.library.custom_op("accelerated_scan::scan_forward", mutates_args=())
def scan_forward(gates: torch.Tensor, tokens: torch.Tensor, reverse: bool) -> torch.Tensor:
    _check_dense(gates, (), token_like=tokens)
    out = torch.empty_like(gates)  # complex gates with real tokens give complex states
    _abi.forward(gates, tokens, out, reverse)
    return out


@scan_forward.register_fake
def _(gates, tokens, reverse):
    return torch.empty_like(gates)


@torch.library.custom_op("accelerated_scan::scan_backward", mutates_args=())
def scan_backward(
    gates: torch.Tensor, states: torch.Tensor, grad_out: torch.Tensor, real_tokens: bool
) -> Tuple[torch.Tensor, torch.Tensor]:
    _check_dense(gates, (states, grad_out))
    d_gates = torch.empty_like(gates)
    d_tokens = _empty_token_grad(gates, real_tokens)
    _abi.backward(gates, states, grad_out, d_gates, d_tokens)
    return d_gates, d_tokens


@scan_backward.register_fake
def _(gates, states, grad_out, real_tokens):
    return torch.empty_like(gates), _empty_token_grad(gates, real_tokens)


@torch.library.custom_op("accelerated_scan::scan_forward_from", mutates_args=())
def scan_forward_from(gates: torch.Tensor, tokens: torch.Tensor, initial: torch.Tensor, reverse: bool) -> torch.Tensor:
    _check_dense(gates, (), token_like=tokens, states=(initial,))
    out = torch.empty_like(gates)
    _abi.forward(gates, tokens, out, reverse, initial=initial)
    return out


@scan_forward_from.register_fake
def _(gates, tokens, initial, reverse):
    return torch.empty_like(gates)


@torch.library.custom_op("accelerated_scan::scan_backward_from", mutates_args=())
def scan_backward_from(
    gates: torch.Tensor, states: torch.Tensor, initial: torch.Tensor, grad_out: torch.Tensor, real_tokens: bool
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_dense(gates, (states, grad_out), states=(initial,))
    d_gates = torch.empty_like(gates)
    d_tokens = _empty_token_grad(gates, real_tokens)
    d_initial = torch.zeros_like(initial)  # stays zero for an empty sequence
    _abi.backward(gates, states, grad_out, d_gates, d_tokens, initial=initial, d_initial=d_initial)
    return d_gates, d_tokens, d_initial


@scan_backward_from.register_fake
def _(gates, states, initial, grad_out, real_tokens):
    return torch.empty_like(gates), _empty_token_grad(gates, real_tokens), torch.empty_like(initial)


@torch.library.custom_op("accelerated_scan::scan_backward_reverse", mutates_args=())
def scan_backward_reverse(
    gates: torch.Tensor, states: torch.Tensor, initial: torch.Tensor, grad_out: torch.Tensor, real_tokens: bool
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Backward pass of a reverse scan (``scan_forward`` / ``scan_forward_from`` with ``reverse=True``)."""
    _check_dense(gates, (states, grad_out), states=(initial,))
    d_gates = torch.empty_like(gates)
    d_tokens = _empty_token_grad(gates, real_tokens)
    d_initial = torch.zeros_like(initial)  # stays zero for an empty sequence
    _abi.backward(gates, states, grad_out, d_gates, d_tokens, initial=initial, d_initial=d_initial, reverse=True)
    return d_gates, d_tokens, d_initial


@scan_backward_reverse.register_fake
def _(gates, states, initial, grad_out, real_tokens):
    return torch.empty_like(gates), _empty_token_grad(gates, real_tokens), torch.empty_like(initial)


@torch.library.custom_op("accelerated_scan::scan_forward_gated", mutates_args=())
def scan_forward_gated(gate_inputs: torch.Tensor, tokens: torch.Tensor, initial: torch.Tensor, gate: int) -> torch.Tensor:
    _check_dense(gate_inputs, (tokens,), states=(initial,))
    out = torch.empty_like(gate_inputs)
    _abi.forward_gated(gate_inputs, tokens, out, gate, initial=initial)
    return out


@scan_forward_gated.register_fake
def _(gate_inputs, tokens, initial, gate):
    return torch.empty_like(gate_inputs)


@torch.library.custom_op("accelerated_scan::scan_backward_gated", mutates_args=())
def scan_backward_gated(
    gate_inputs: torch.Tensor, states: torch.Tensor, initial: torch.Tensor, grad_out: torch.Tensor, gate: int
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_dense(gate_inputs, (states, grad_out), states=(initial,))
    d_gate_inputs = torch.empty_like(gate_inputs)
    d_tokens = torch.empty_like(gate_inputs)
    d_initial = torch.zeros_like(initial)  # stays zero for an empty sequence
    _abi.backward_gated(gate_inputs, states, grad_out, d_gate_inputs, d_tokens, gate, initial=initial,
                        d_initial=d_initial)
    return d_gate_inputs, d_tokens, d_initial


@scan_backward_gated.register_fake
def _(gate_inputs, states, initial, grad_out, gate):
    return torch.empty_like(gate_inputs), torch.empty_like(gate_inputs), torch.empty_like(initial)


@torch.library.custom_op("accelerated_scan::scan_backward_lerp", mutates_args=())
def scan_backward_lerp(
    gate_inputs: torch.Tensor, values: torch.Tensor, states: torch.Tensor, initial: torch.Tensor, grad_out: torch.Tensor
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_dense(gate_inputs, (values, states, grad_out), states=(initial,))
    d_gate_inputs = torch.empty_like(gate_inputs)
    d_values = torch.empty_like(gate_inputs)
    d_initial = torch.zeros_like(initial)  # stays zero for an empty sequence
    _abi.backward_lerp(gate_inputs, values, states, grad_out, d_gate_inputs, d_values, initial=initial,
                       d_initial=d_initial)
    return d_gate_inputs, d_values, d_initial


@scan_backward_lerp.register_fake
def _(gate_inputs, values, states, initial, grad_out):
    return torch.empty_like(gate_inputs), torch.empty_like(gate_inputs), torch.empty_like(initial)


@torch.library.custom_op("accelerated_scan::scan_backward_gated_values", mutates_args=())
def scan_backward_gated_values(
    gate_inputs: torch.Tensor, values: torch.Tensor, states: torch.Tensor, initial: torch.Tensor,
    grad_out: torch.Tensor, gate: int
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    _check_dense(gate_inputs, (values, states, grad_out), states=(initial,))
    d_gate_inputs = torch.empty_like(gate_inputs)
    d_values = torch.empty_like(gate_inputs)
    d_initial = torch.zeros_like(initial)  # stays zero for an empty sequence
    _abi.backward_gated_values(gate_inputs, values, states, grad_out, d_gate_inputs, d_values, gate, initial=initial,
                               d_initial=d_initial)
    return d_gate_inputs, d_values, d_initial


@scan_backward_gated_values.register_fake
def _(gate_inputs, values, states, initial, grad_out, gate):
    return torch.empty_like(gate_inputs), torch.empty_like(gate_inputs), torch.empty_like(initial)


def _empty_token_grad(gates: torch.Tensor, real_tokens: bool) -> torch.Tensor:
    """Token gradient buffer: real when complex gates were scanned over real tokens."""
    if real_tokens and gates.is_complex():
        return torch.empty(gates.shape, dtype=gates.real.dtype, device=gates.device)
    return torch.empty_like(gates)


def capturing() -> bool:
    """True while torch.compile is tracing the caller."""
    return torch.compiler.is_compiling()


# ---------------------------------------------------------------------------
# Autograd formulas of the forward operators.  The gradient of a scan is the
# fused backward operator (accelerated_scan/warp.py:50-65 of the reference:
# g[t] = grad[t] + gates[t+1] * g[t+1], d_tokens = g, d_gates[t] = g[t] * x[t-1]).
# A reverse scan has a fused backward operator of its own, the mirror image in time.
# ---------------------------------------------------------------------------
def _real_tokens(gates: torch.Tensor, tokens: torch.Tensor) -> bool:
    return gates.is_complex() and not tokens.is_complex()


def _setup_scan_forward(ctx, inputs, output):
    gates, tokens, reverse = inputs
    ctx.save_for_backward(gates, output)
    ctx.reverse = reverse
    ctx.real_tokens = _real_tokens(gates, tokens)


def _backward_scan_forward(ctx, grad):
    gates, states = ctx.saved_tensors
    grad = grad.contiguous()
    if ctx.reverse:
        zero = torch.zeros(gates.shape[:-1], dtype=gates.dtype, device=gates.device)
        d_gates, d_tokens, _ = scan_backward_reverse(gates, states, zero, grad, ctx.real_tokens)
        return d_gates, d_tokens, None
    d_gates, d_tokens = scan_backward(gates, states, grad, ctx.real_tokens)
    return d_gates, d_tokens, None


torch.library.register_autograd(
    "accelerated_scan::scan_forward", _backward_scan_forward, setup_context=_setup_scan_forward)


def _setup_scan_forward_from(ctx, inputs, output):
    gates, tokens, initial, reverse = inputs
    ctx.save_for_backward(gates, output, initial)
    ctx.reverse = reverse
    ctx.real_tokens = _real_tokens(gates, tokens)


def _backward_scan_forward_from(ctx, grad):
    gates, states, initial = ctx.saved_tensors
    grad = grad.contiguous()
    if ctx.reverse:
        d_gates, d_tokens, d_initial = scan_backward_reverse(gates, states, initial, grad, ctx.real_tokens)
        return d_gates, d_tokens, d_initial, None
    d_gates, d_tokens, d_initial = scan_backward_from(gates, states, initial, grad, ctx.real_tokens)
    return d_gates, d_tokens, d_initial, None


torch.library.register_autograd(
    "accelerated_scan::scan_forward_from", _backward_scan_forward_from, setup_context=_setup_scan_forward_from)


def _setup_scan_forward_gated(ctx, inputs, output):
    gate_inputs, tokens, initial, gate = inputs
    if gate in _abi.GATES_WITH_VALUES:  # the second input holds values, and the backward pass reads them
        ctx.save_for_backward(gate_inputs, output, initial, tokens)
    else:
        ctx.save_for_backward(gate_inputs, output, initial)
    ctx.gate = gate


def _backward_scan_forward_gated(ctx, grad):
    if ctx.gate in _abi.GATES_WITH_VALUES:
        gate_inputs, states, initial, values = ctx.saved_tensors
        d_gate_inputs, d_values, d_initial = scan_backward_gated_values(gate_inputs, values, states, initial,
                                                                        grad.contiguous(), ctx.gate)
        return d_gate_inputs, d_values, d_initial, None
    gate_inputs, states, initial = ctx.saved_tensors
    d_gate_inputs, d_tokens, d_initial = scan_backward_gated(gate_inputs, states, initial, grad.contiguous(), ctx.gate)
    return d_gate_inputs, d_tokens, d_initial, None


torch.library.register_autograd(
    "accelerated_scan::scan_forward_gated", _backward_scan_forward_gated, setup_context=_setup_scan_forward_gated)


# ---------------------------------------------------------------------------
# Gated delta rule and gated norm (modules ``delta`` and ``norm``).  The ``*_run`` functions choose between the
# custom operator, while a graph is being captured, and the direct call.
# ---------------------------------------------------------------------------
def no_tangents(*tensors) -> None:
    """Refuse tensors that carry a forward-mode tangent: these operators have none to hand on, and results without one
    read as a derivative of zero.  (Outside a dual level, where no tensor has one, this is one comparison.)"""
    if forward_ad._current_level < 0:
        return
    # (the body of an operator that changes an argument runs behind the dispatch key that takes a dual tensor apart)
    hidden = torch._C._dispatch_tls_local_exclude_set().remove(torch._C.DispatchKey.ADInplaceOrView)
    with torch._C._ForceDispatchKeyGuard(torch._C._dispatch_tls_local_include_set(), hidden):
        duals = any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    if duals:
        raise NotImplementedError("accelerated_scan: the gated delta rule and the gated norm have no forward-mode derivatives")


def _delta_outputs(queries, values, initial, offsets, keep):
    """Empty (out, final, states, updates) of a delta rule call."""
    batch, tokens, _, key_dim = queries.shape
    heads, value_dim = values.shape[2:]
    sequences = batch if offsets is None else offsets.shape[0] - 1
    blocks = -(-tokens // 64) * batch if offsets is None else batch * tokens // 64 + sequences
    new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=queries.device)  # noqa: E731
    final = new(sequences, heads, key_dim, value_dim)
    if not keep:
        return torch.empty_like(values), final, new(0), new(0)
    return torch.empty_like(values), final, new(blocks, heads, key_dim, value_dim), new(batch, tokens, heads, value_dim)


def _delta_forward(queries, keys, values, log_gates, beta, initial, offsets, scale, keep):
    out, final, states, updates = _delta_outputs(queries, values, initial, offsets, keep)
    if final.shape[0] == 0:
        out.zero_()  # no sequence: rows outside all of them
    else:
        _abi.delta_forward(queries, keys, values, log_gates, beta, initial, offsets, scale, out, final,
                           states if keep else None, updates if keep else None)
    return out, final, states, updates


def delta_outputs(queries, keys, values, log_gates, beta, initial, offsets, scale):
    """(out, final) alone, by the direct call."""
    sequences = queries.shape[0] if offsets is None else offsets.shape[0] - 1
    out = torch.empty_like(values)
    final = torch.empty((sequences, values.shape[2], queries.shape[3], values.shape[3]), dtype=torch.float32,
                        device=values.device)
    if sequences == 0:
        out.zero_()  # rows outside all sequences
    else:
        _abi.delta_forward(queries, keys, values, log_gates, beta, initial, offsets, scale, out, final)
    return out, final


@torch.library.custom_op("accelerated_scan::delta_forward", mutates_args=())
def delta_forward(
    queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, log_gates: torch.Tensor, beta: torch.Tensor,
    initial: Optional[torch.Tensor], offsets: Optional[torch.Tensor], scale: float, keep: bool
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``keep``: also return what ``delta_backward`` needs (else empty tensors)."""
    from . import delta

    delta._check_scan(queries, keys, values, log_gates, beta, initial, offsets)
    return _delta_forward(queries, keys, values, log_gates, beta, initial, offsets, scale, keep)


@delta_forward.register_fake
def _(queries, keys, values, log_gates, beta, initial, offsets, scale, keep):
    return _delta_outputs(queries, values, initial, offsets, keep)


def _delta_gradients(queries, keys, values, log_gates, beta, states, started, offsets):
    """Empty gradients of the inputs; that of the initial states has no elements where there are none."""
    sequences = queries.shape[0] if offsets is None else offsets.shape[0] - 1
    shape = (sequences, values.shape[2], queries.shape[3], values.shape[3]) if started else (0,)
    d_initial = torch.empty(shape, dtype=torch.float32, device=queries.device)
    return (*(torch.empty_like(t) for t in (queries, keys, values, log_gates, beta)), d_initial)


def _on_16_bytes(t):
    """A gradient can be a piece of a larger tensor, from where the kernels do not read."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _delta_backward(queries, keys, values, log_gates, beta, states, updates, offsets, scale, d_out, d_final, started):
    no_tangents(states, updates, d_out, d_final)
    grads = _delta_gradients(queries, keys, values, log_gates, beta, states, started, offsets)
    if offsets is not None and offsets.shape[0] == 1:
        for g in grads:
            g.zero_()
    else:
        _abi.delta_backward(queries, keys, values, log_gates, beta, states, updates, offsets, scale,
                            _on_16_bytes(d_out), _on_16_bytes(d_final), *grads[:5], grads[5] if started else None)
    return grads


@torch.library.custom_op("accelerated_scan::delta_backward", mutates_args=())
def delta_backward(
    queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, log_gates: torch.Tensor, beta: torch.Tensor,
    states: torch.Tensor, updates: torch.Tensor, offsets: Optional[torch.Tensor], scale: float,
    d_out: Optional[torch.Tensor], d_final: Optional[torch.Tensor], started: bool
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``started``: the forward pass had initial states, whose gradient is the last result."""
    from . import delta

    sequences = delta._check_scan(queries, keys, values, log_gates, beta, None, offsets)
    state = (values.shape[2], queries.shape[3], values.shape[3])
    blocks = _abi.delta_blocks(queries.shape[0] * queries.shape[1], sequences, offsets is not None)
    for t, shape, dtype in ((states, (blocks, *state), torch.float32), (updates, values.shape, torch.float32),
                            (d_out, values.shape, values.dtype), (d_final, (sequences, *state), torch.float32)):
        if t is not None and (t.shape != shape or t.dtype != dtype or t.device != queries.device or not t.is_contiguous()):
            raise RuntimeError(f"accelerated_scan: expected a contiguous {dtype} tensor of shape {tuple(shape)} on "
                               f"{queries.device}, got {t.dtype}, {tuple(t.shape)}")
    return _delta_backward(queries, keys, values, log_gates, beta, states, updates, offsets, scale, d_out, d_final, started)


@delta_backward.register_fake
def _(queries, keys, values, log_gates, beta, states, updates, offsets, scale, d_out, d_final, started):
    return _delta_gradients(queries, keys, values, log_gates, beta, states, started, offsets)


def delta_forward_run(*args):
    return delta_forward(*args) if capturing() else _delta_forward(*args)


def delta_backward_run(*args):
    return delta_backward(*args) if capturing() else _delta_backward(*args)


def _setup_delta_forward(ctx, inputs, output):
    queries, keys, values, log_gates, beta, initial, offsets, scale, keep = inputs
    if not keep:
        raise RuntimeError("accelerated_scan: delta_forward is differentiable with keep=True only")
    _, _, states, updates = output
    ctx.save_for_backward(queries, keys, values, log_gates, beta, states, updates, offsets)
    ctx.scale = scale
    ctx.started = initial is not None
    ctx.set_materialize_grads(False)


def _backward_delta_forward(ctx, d_out, d_final, d_states, d_updates):
    *inputs, states, updates, offsets = ctx.saved_tensors
    if d_out is None and d_final is None:
        return (None,) * 9
    grads = delta_backward(*inputs, states, updates, offsets, ctx.scale,
                           d_out.contiguous() if d_out is not None else None,
                           d_final.contiguous() if d_final is not None else None, ctx.started)
    return (*grads[:5], grads[5] if ctx.started else None, None, None, None)


torch.library.register_autograd(
    "accelerated_scan::delta_forward", _backward_delta_forward, setup_context=_setup_delta_forward)


@torch.library.custom_op("accelerated_scan::delta_step", mutates_args=("states",))
def delta_step(
    queries: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, log_gates: torch.Tensor, beta: torch.Tensor,
    states: torch.Tensor, slots: Optional[torch.Tensor], scale: float
) -> torch.Tensor:
    from . import delta

    delta._check_step(queries, keys, values, log_gates, beta, states, slots)
    out = torch.empty_like(values)
    _abi.delta_step(queries, keys, values, log_gates, beta, states, slots, scale, out)
    return out


@delta_step.register_fake
def _(queries, keys, values, log_gates, beta, states, slots, scale):
    return torch.empty_like(values)


@torch.library.custom_op("accelerated_scan::gated_norm", mutates_args=())
def gated_norm(x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    from . import norm

    norm._check(x, gate, weight)
    out = torch.empty_like(x)
    if x.numel():
        _abi.gated_norm(x, gate, weight, eps, out)
    return out


@gated_norm.register_fake
def _(x, gate, weight, eps):
    return torch.empty_like(x)


def _gated_norm_backward(x, gate, weight, d_out, eps):
    no_tangents(d_out)
    d_x, d_gate = torch.empty_like(x), torch.empty_like(gate)
    if x.numel() == 0:
        return d_x, d_gate, torch.zeros_like(weight)
    d_weight = torch.empty_like(weight)
    _abi.gated_norm_backward(x, gate, weight, eps, d_out, d_x, d_gate, d_weight)
    return d_x, d_gate, d_weight


@torch.library.custom_op("accelerated_scan::gated_norm_backward", mutates_args=())
def gated_norm_backward(
    x: torch.Tensor, gate: torch.Tensor, weight: torch.Tensor, d_out: torch.Tensor, eps: float
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    from . import norm

    norm._check(x, gate, weight)
    if d_out.shape != x.shape or d_out.dtype != x.dtype or d_out.device != x.device or not d_out.is_contiguous():
        raise RuntimeError("accelerated_scan: expected d_out to be contiguous, with the shape and dtype of x")
    return _gated_norm_backward(x, gate, weight, d_out, eps)


@gated_norm_backward.register_fake
def _(x, gate, weight, d_out, eps):
    return torch.empty_like(x), torch.empty_like(gate), torch.empty_like(weight)


def gated_norm_backward_run(*args):
    return gated_norm_backward(*args) if capturing() else _gated_norm_backward(*args)


torch.library.register_autograd(
    "accelerated_scan::gated_norm",
    lambda ctx, grad: (*gated_norm_backward(*ctx.saved_tensors, grad.contiguous(), ctx.eps), None),
    setup_context=lambda ctx, inputs, output: (ctx.save_for_backward(*inputs[:3]), setattr(ctx, "eps", inputs[3]))[0])
