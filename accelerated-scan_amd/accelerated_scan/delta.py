"""Gated delta rule: the linear recurrence whose state is a matrix per head.

Where the scans of this package multiply a state by a gate per channel, the delta rule keeps a
(key_dim, value_dim) matrix per head that maps keys to values, forgets by a gate per head and token, and
corrects what it holds for the current key towards the current value:

    S[t]   = a[t] S[t-1] + beta[t] k[t] (v[t] - (a[t] S[t-1])^T k[t])^T,    a = exp(log_gates)
    out[t] = scale S[t]^T q[t]

``gated_delta_scan`` runs it over whole sequences (batched, or packed behind each other), differentiable in all
inputs; ``gated_delta_step`` advances the states of many conversations by one token, in place.  As in
``gated.exp_scan`` the gates come as logarithms.  Features are innermost here, since the kernels multiply
matrices of (token, feature) rows: (B, T, heads, dim) tensors, contiguous, as projections of a layer give them.
Heads may share their keys and queries: value head h uses key head ``h // (heads // key_heads)``.

States are float32 whatever the tensors' type.  The reference has no operator of this kind; its scans are
diagonal (accelerated_scan/warp.cuh:49-223).
"""

import torch
from torch.autograd.function import once_differentiable

from . import _abi, _ops

_REAL_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _fail(what):
    raise RuntimeError(f"accelerated_scan: {what}")


def _check_tensors(like, named):
    """All device tensors on one device, contiguous."""
    device = like.device
    for name, t in named:
        if t is None or (t.is_cuda and t.device == device and t.is_contiguous()):
            continue
        if not t.is_cuda:
            _fail(f"expected {name} to be a device tensor")
        if t.device != like.device:
            _fail(f"expected {name} to be on the device of queries")
        if not t.is_contiguous():
            _fail(f"expected {name} to be contiguous")


def _check_types(queries, keys, values, log_gates, beta):
    dtype = queries.dtype
    if dtype not in _REAL_DTYPES or keys.dtype != dtype or values.dtype != dtype:
        _fail(f"unsupported tensor dtypes {queries.dtype}, {keys.dtype}, {values.dtype}: expecting queries, keys and "
              "values all bfloat16, float16 or float32")
    if log_gates.dtype not in (dtype, torch.float32) or beta.dtype != log_gates.dtype:
        _fail(f"unsupported tensor dtypes {log_gates.dtype}, {beta.dtype}: expecting log_gates and beta both "
              f"{dtype} or float32")


def _check_heads(queries, keys, values, log_gates, beta):
    lead, (key_heads, key_dim) = queries.shape[:-2], queries.shape[-2:]
    heads, value_dim = values.shape[-2:]
    if keys.shape != queries.shape or values.shape[:-2] != lead:
        _fail(f"expected keys of the shape of queries and values of the same tokens, got {tuple(queries.shape)}, "
              f"{tuple(keys.shape)} and {tuple(values.shape)}")
    if log_gates.shape != values.shape[:-1] or beta.shape != values.shape[:-1]:
        _fail(f"expected log_gates and beta of shape {tuple(values.shape[:-1])}, got {tuple(log_gates.shape)} and "
              f"{tuple(beta.shape)}")
    if key_heads == 0 or heads == 0 or heads % key_heads:
        _fail(f"expected key heads that divide the heads, got {key_heads} and {heads}")
    if not (0 < key_dim <= 128 and key_dim % 8 == 0 and 0 < value_dim <= 4096 and value_dim % 8 == 0):
        _fail(f"expected a key size up to 128 and a value size up to 4096, both multiples of 8, got {key_dim} and "
              f"{value_dim}")


def _plainly_right(queries, keys, values, log_gates, beta):
    """Whether a call passes the checks of what both operators have in common (no message is built)."""
    lead_heads, dtype, device = values.shape[:-1], queries.dtype, queries.device
    *lead, key_heads, key_dim = queries.shape
    heads, value_dim = lead_heads[-1], values.shape[-1]
    return (dtype in _REAL_DTYPES and keys.dtype == dtype and values.dtype == dtype and beta.dtype == log_gates.dtype
            and (log_gates.dtype == dtype or log_gates.dtype == torch.float32) and keys.shape == queries.shape
            and log_gates.shape == lead_heads and beta.shape == lead_heads and (*lead, heads) == lead_heads
            and key_heads and heads and heads % key_heads == 0 and 0 < key_dim <= 128 and key_dim % 8 == 0
            and 0 < value_dim <= 4096 and value_dim % 8 == 0
            and queries.is_cuda and keys.device == device and values.device == device and log_gates.device == device
            and beta.device == device and queries.is_contiguous() and keys.is_contiguous() and values.is_contiguous()
            and log_gates.is_contiguous() and beta.is_contiguous())


def _check_scan(queries, keys, values, log_gates, beta, initial, offsets):
    _ops.no_tangents(queries, keys, values, log_gates, beta, initial)
    if (initial is None and offsets is None and queries.dim() == 4 and values.dim() == 4
            and _plainly_right(queries, keys, values, log_gates, beta)):
        return queries.shape[0]
    if queries.dim() != 4 or values.dim() != 4:
        _fail("expected queries, keys and values of shape (B, T, heads, dim)")
    _check_types(queries, keys, values, log_gates, beta)
    _check_heads(queries, keys, values, log_gates, beta)
    sequences = queries.shape[0]
    if offsets is not None:
        if offsets.dim() != 1 or offsets.shape[0] < 1 or offsets.dtype not in (torch.int32, torch.int64):
            _fail("expected offsets of shape (sequences + 1,), int32 or int64")
        if queries.shape[0] != 1:
            _fail(f"expected packed sequences in a batch of one, got a batch of {queries.shape[0]}")
        sequences = offsets.shape[0] - 1
    if initial is not None:
        shape = (sequences, values.shape[2], queries.shape[3], values.shape[3])
        if initial.shape != shape or initial.dtype != torch.float32:
            _fail(f"expected initial of shape {shape} and dtype torch.float32, got {tuple(initial.shape)} and "
                  f"{initial.dtype}")
    _check_tensors(queries, (("queries", queries), ("keys", keys), ("values", values), ("log_gates", log_gates),
                             ("beta", beta), ("initial", initial), ("offsets", offsets)))
    return sequences


class GatedDeltaScan(torch.autograd.Function):
    """Autograd node: saves the inputs, the state in front of every block of 64 tokens and the rows that the
    tokens added to it."""

    @staticmethod
    def forward(ctx, queries, keys, values, log_gates, beta, initial, offsets, scale):
        keep = any(ctx.needs_input_grad)
        out, final, states, updates = _ops.delta_forward_run(queries, keys, values, log_gates, beta, initial, offsets,
                                                             scale, keep)
        if keep:
            ctx.save_for_backward(queries, keys, values, log_gates, beta, states, updates, offsets)
        ctx.scale = scale
        ctx.started = initial is not None
        ctx.set_materialize_grads(False)
        return out, final

    @staticmethod
    def backward(ctx, d_out, d_final):
        if torch.is_grad_enabled() and not _ops.capturing():  # create_graph: no second derivatives
            return once_differentiable(_scan_gradients)(ctx, d_out, d_final)
        return _scan_gradients(ctx, d_out, d_final)


def _scan_gradients(ctx, d_out, d_final):
    if d_out is None and d_final is None:
        return (None,) * 8
    *inputs, states, updates, offsets = ctx.saved_tensors
    grads = _ops.delta_backward_run(*inputs, states, updates, offsets, ctx.scale,
                                    d_out.contiguous() if d_out is not None else None,
                                    d_final.contiguous() if d_final is not None else None, ctx.started)
    return (*grads[:5], grads[5] if ctx.started else None, None, None)


def gated_delta_scan(queries, keys, values, log_gates, beta, initial=None, scale=None, offsets=None):
    """Run the gated delta rule over whole sequences.

    Arguments:
        queries, keys (torch.Tensor): shape (B, T, key_heads, key_dim), contiguous; fp32, bf16 or fp16.
            Keys of unit length keep the state bounded for ``beta`` between 0 and 2.
        values (torch.Tensor): shape (B, T, heads, value_dim), contiguous, same dtype; ``heads`` a multiple of
            ``key_heads``.
        log_gates, beta (torch.Tensor): shape (B, T, heads), contiguous, the same dtype or fp32.  A log gate of
            ``-inf`` starts the state anew; where they are positive, 64 of them sum to less than 88.
        initial (torch.Tensor, optional): shape (B, heads, key_dim, value_dim), fp32: the states to start from
            (zero if absent); with ``offsets`` one per sequence.
        scale (float, optional): factor of the outputs, ``key_dim ** -0.5`` if absent.
        offsets (torch.Tensor, optional): int32 or int64 on the device, shape (sequences + 1,): the tensors hold
            sequences of different lengths behind each other in a batch of one, sequence n in rows
            ``offsets[n]`` to ``offsets[n + 1] - 1``; empty ones are allowed.  Rows outside all of them are not
            read, and their outputs and gradients are zero.

    Returns:
        (torch.Tensor, torch.Tensor): the outputs, shape (B, T, heads, value_dim), and the states behind the last
        tokens, fp32, as ``initial`` has them: hand them to the next chunk or to ``gated_delta_step``.
        Differentiable once, in reverse mode, in all tensors but ``offsets``.  A token that is not finite leaves the
        outputs of the tokens before it as they are.
    """
    _check_scan(queries, keys, values, log_gates, beta, initial, offsets)
    scale = float(scale) if scale is not None else queries.shape[-1] ** -0.5
    if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad or values.requires_grad
                                    or log_gates.requires_grad or beta.requires_grad
                                    or (initial is not None and initial.requires_grad)):
        return GatedDeltaScan.apply(queries, keys, values, log_gates, beta, initial, offsets, scale)
    if _ops.capturing():
        return _ops.delta_forward(queries, keys, values, log_gates, beta, initial, offsets, scale, False)[:2]
    return _ops.delta_outputs(queries, keys, values, log_gates, beta, initial, offsets, scale)


def _check_step(queries, keys, values, log_gates, beta, states, slots):
    _ops.no_tangents(queries, keys, values, log_gates, beta, states)
    if (queries.dim() == 3 and values.dim() == 3 and states.dtype == torch.float32 and states.dim() == 4
            and states.shape[1:] == (values.shape[1], queries.shape[2], values.shape[2]) and states.device == queries.device
            and states.is_contiguous()
            and (states.shape[0] == queries.shape[0] if slots is None else
                 slots.shape == queries.shape[:1] and slots.dtype in (torch.int32, torch.int64)
                 and slots.device == queries.device and slots.is_contiguous())
            and _plainly_right(queries, keys, values, log_gates, beta)):
        return
    if queries.dim() != 3 or values.dim() != 3:
        _fail("expected queries, keys and values of shape (B, heads, dim)")
    _check_types(queries, keys, values, log_gates, beta)
    _check_heads(queries, keys, values, log_gates, beta)
    shape = (values.shape[1], queries.shape[2], values.shape[2])
    if states.dim() != 4 or states.shape[1:] != shape or states.dtype != torch.float32:
        _fail(f"expected states of shape (slots, {', '.join(map(str, shape))}) and dtype torch.float32, got "
              f"{tuple(states.shape)} and {states.dtype}")
    if slots is None:
        if states.shape[0] != queries.shape[0]:
            _fail(f"expected a state to each of {queries.shape[0]} rows, got {states.shape[0]}")
    else:
        if slots.shape != queries.shape[:1] or slots.dtype not in (torch.int32, torch.int64):
            _fail(f"expected slots of shape ({queries.shape[0]},), int32 or int64")
    _check_tensors(queries, (("queries", queries), ("keys", keys), ("values", values), ("log_gates", log_gates),
                             ("beta", beta), ("states", states), ("slots", slots)))


def gated_delta_step(queries, keys, values, log_gates, beta, states, slots=None, scale=None):
    """Advance states by one token each, in place (no autograd, in either mode: for generation).

    Arguments:
        queries, keys (torch.Tensor): shape (B, key_heads, key_dim), contiguous; fp32, bf16 or fp16.
        values (torch.Tensor): shape (B, heads, value_dim), contiguous, same dtype.
        log_gates, beta (torch.Tensor): shape (B, heads), contiguous, the same dtype or fp32.
        states (torch.Tensor): shape (S, heads, key_dim, value_dim), contiguous, fp32: updated in place.
        slots (torch.Tensor, optional): shape (B,), int32 or int64 on the device: row b uses ``states[slots[b]]``
            (row b uses ``states[b]`` if absent).  Rows that name the same slot are consecutive tokens of it, in
            their order.  A slot outside ``0 .. S - 1`` marks a row without a state: its output is zero.
        scale (float, optional): factor of the outputs, ``key_dim ** -0.5`` if absent.

    Returns:
        (torch.Tensor): the outputs, shape (B, heads, value_dim).
    """
    _check_step(queries, keys, values, log_gates, beta, states, slots)
    if torch.is_grad_enabled() and (queries.requires_grad or keys.requires_grad or values.requires_grad
                                    or log_gates.requires_grad or beta.requires_grad or states.requires_grad):
        _fail("gated_delta_step is not differentiable: use gated_delta_scan, or torch.no_grad()")
    scale = float(scale) if scale is not None else queries.shape[-1] ** -0.5
    if _ops.capturing():
        return _ops.delta_step(queries, keys, values, log_gates, beta, states, slots, scale)
    out = torch.empty_like(values)
    _abi.delta_step(queries, keys, values, log_gates, beta, states, slots, scale, out)
    if not states.is_inference():
        torch.autograd.graph.increment_version(states)
    return out
