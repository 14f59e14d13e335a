"""The gated delta rule and the gated norm from their definitions, token by token in float64 on the CPU
(differentiable by autograd), and the error bounds the GPU tests hold the kernels to.

Bounds, for an output type with rounding step u = finfo.eps / 2 (bf16 2^-8, fp16 2^-11, fp32 2^-24):

* One rounding to the output's type moves a value by at most u times itself.
* Inside, 16-bit inputs are exact and everything else is held to e = 2^-16 or better (a value as two bfloat16
  parts), for fp32 inputs to e = 2^-22 (three parts, and sums of up to 128 products in fp32).  A product of two
  such values is off by at most 3 e of its size: what each operand lacks, and the product of the low parts.
* An output lies behind at most 6 such products in the forward pass (K S, T R twice, P U, Q S, K^T U), a gradient
  behind at most 12.  In the root mean square the errors of a sum's terms grow like the sum itself, so a
  stage adds at most 3 e to the relative error of a tensor, times the condition of I + L, which random keys of
  unit length keep below 4: 6 * 3 * 4 = 72 e forward, 144 e backward (``close``'s first bound).
* A single value may come out of cancellation: its terms' magnitudes sum to at most sqrt(128) < 12 times the
  largest output where signs are random.  The second bound is u |value| + 12 * 72 e (144 e) of the largest.
"""

import torch


def delta_scan(q, k, v, log_gates, beta, initial=None, scale=None):
    """(B, T, heads, dim) float64 tensors -> (out, final)."""
    share = v.shape[2] // q.shape[2]
    q, k = q.repeat_interleave(share, 2), k.repeat_interleave(share, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    S = q.new_zeros(q.shape[0], v.shape[2], q.shape[3], v.shape[3]) if initial is None else initial
    out = []
    for t in range(q.shape[1]):
        S = S * log_gates[:, t].exp()[..., None, None]
        held = torch.einsum("bhk,bhkv->bhv", k[:, t], S)
        S = S + k[:, t].unsqueeze(-1) * (beta[:, t].unsqueeze(-1) * (v[:, t] - held)).unsqueeze(-2)
        out.append(scale * torch.einsum("bhk,bhkv->bhv", q[:, t], S))
    return (torch.stack(out, 1) if out else v.clone()), S


def gated_norm(x, gate, weight, eps=1e-6):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight * gate * torch.sigmoid(gate)


def inputs(B, T, key_heads, heads, dk, dv, dtype, seed=0, gates=None, sequences=None, decay=1.0):
    """Seeded inputs on the CPU: unit keys and queries, gates of a layer.  Values are those of ``dtype``."""
    gen = torch.Generator().manual_seed(seed)
    gates = gates or dtype
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)  # noqa: E731
    q = unit(torch.randn(B, T, key_heads, dk, generator=gen)).to(dtype)
    k = unit(torch.randn(B, T, key_heads, dk, generator=gen)).to(dtype)
    v = torch.randn(B, T, heads, dv, generator=gen).to(dtype)
    log_gates = (-decay * torch.rand(B, T, heads, generator=gen) ** 3).to(gates)
    beta = torch.rand(B, T, heads, generator=gen).to(gates)
    initial = 0.3 * torch.randn(B if sequences is None else sequences, heads, dk, dv, generator=gen)
    return q, k, v, log_gates, beta, initial


def close(got, want, like, backward=False, what="", grow=1.0):
    """``got`` (any device) against ``want`` (float64), computed from inputs of type ``like``."""
    got = got.detach().cpu()
    u = torch.finfo(got.dtype).eps / 2
    e = 2.0 ** (-22 if like == torch.float32 else -16) * grow
    stages = 144 if backward else 72
    got, want = got.double(), want.detach()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if not want.numel():
        return
    assert torch.isfinite(got).all(), what
    off, size = (got - want), want.norm().item()
    if size == 0:
        assert off.abs().max().item() == 0, what
        return
    rel = off.norm().item() / size
    assert rel <= u + stages * e, f"{what}: relative error {rel:.3g} over {u + stages * e:.3g}"
    most = want.abs().max().item()
    over = (off.abs() - (u * want.abs() + 12 * stages * e * most)).max().item()
    assert over <= 0, f"{what}: a value is {over:.3g} beyond its bound"


def close_in_32_bits(got, want, backward=False, what=""):
    """A float32 result against float64, whatever the inputs' type, in the root mean square.

    An operand lacks at most 2^-25 of itself (three bfloat16 parts hold a float32 value), the pairs of parts that are left
    out come to 3 * 2^-25, and a sum of up to 128 products is made in at most 24 steps, each rounded to 2^-24 of a partial
    sum.  Roundings are independent, so they add in squares: a product is off by at most sqrt((24 + 6) / 3) < 3.2 times
    2^-24 of its size.  The six of the forward pass come to sqrt(6) 3.2 < 8, the twelve of a gradient to 11, and the condition
    of I + L, below 4 for the largest error, takes a random one to twice its size at most: 16 and, with
    the states' own error that the gradients are formed with, 32 times 2^-24."""
    assert got.dtype == torch.float32
    got, want = got.detach().cpu().double(), want.detach()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    rel, most = (got - want).norm().item() / want.norm().item(), (32 if backward else 16) * 2.0 ** -24
    assert rel <= most, f"{what}: relative error {rel:.3g} over {most:.3g}"
