"""The delta-rule operators and the gated norm, as a program calls them, with a plain form of each.

``listed()`` names fixed workloads, ``draw(rng)`` makes more of the same ranges, ``prepare(case, seed)`` builds a
workload's inputs on the GPU, ``run(state)`` makes one pass -- in elementary torch operations, or through
``accelerated_scan`` where ``own`` is true -- ``work(case)`` counts what a pass cannot do without and
``exact(case, seed)`` computes its outputs from the definition in 64 bits, token by token.

The operators (h a value head, j the key head it shares, S a (key_dim, value_dim) state, a = exp(log_gate)):

    S[t] = a[t] S[t-1] + beta[t] k[t] (v[t] - (a[t] S[t-1])^T k[t])^T,     out[t] = scale S[t]^T q[t]
    y    = weight * x / sqrt(mean(x^2) + eps) * silu(gate)
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 64     # tokens the plain form takes at a time
EPS = 1e-6


def _scan(name, kind, dtype, gates, batch, tokens, key_heads, heads, key_dim, value_dim, lengths="", start=False):
    return {"name": name, "kind": kind, "dtype": dtype, "gates": gates, "batch": batch, "tokens": tokens,
            "key_heads": key_heads, "heads": heads, "key_dim": key_dim, "value_dim": value_dim, "lengths": lengths,
            "start": start}


def _step(name, dtype, gates, batch, slots, key_heads, heads, key_dim, value_dim):
    return {"name": name, "kind": "step", "dtype": dtype, "gates": gates, "batch": batch, "slots": slots,
            "key_heads": key_heads, "heads": heads, "key_dim": key_dim, "value_dim": value_dim}


def _norm(name, kind, dtype, rows, heads, width):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "heads": heads, "width": width}


def listed():
    return [
        # a short prompt: less than one block of tokens, latency is all
        _scan("prompt_short", "prompt", "bfloat16", "float32", 1, 50, 8, 8, 64, 64),
        # one long prompt, two value heads to a key head, logarithms of the gates kept in 32 bits
        _scan("prompt_long", "prompt", "bfloat16", "float32", 1, 16384, 16, 32, 128, 128),
        # the next pieces of several conversations packed behind each other, one of them empty, one a single token
        _scan("prompt_packed", "prompt", "float16", "float16", 1, 12291, 16, 16, 128, 128,
              "1,0,4097,63,64,65,2500,777,129,1024,300,1500,31,640,260,840", True),
        # a batch in 32 bits with head sizes that are no powers of two
        _scan("prompt_f32", "prompt", "float32", "float32", 4, 1537, 2, 6, 96, 80, "", True),
        # a training step of a middle-sized layer
        _scan("train", "train", "bfloat16", "bfloat16", 2, 4096, 16, 16, 128, 128),
        # a training step on packed documents of different lengths, shared key heads
        _scan("train_packed", "train", "float16", "float16", 1, 5000, 4, 8, 64, 128,
              "700,1,1300,0,129,1870,64,936", True),
        # a small training step in 32 bits, ragged length
        _scan("train_f32", "train", "float32", "float32", 3, 333, 4, 4, 64, 64, "", True),
        # one new token of one conversation
        _step("step_one", "bfloat16", "float32", 1, 4, 16, 32, 128, 128),
        # one new token of many conversations, their states in slots of a pool
        _step("step_many", "bfloat16", "float32", 256, 300, 16, 32, 128, 128),
        # the norm behind the scan for a batch of new tokens
        _norm("norm_tokens", "norm", "bfloat16", 64, 32, 128),
        # the same norm in a training step
        _norm("norm_train", "norm_train", "bfloat16", 16384, 32, 128),
        # and over whole rows of an odd width in 32 bits
        _norm("norm_train_f32", "norm_train", "float32", 5001, 1, 1000),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "train", "train", "train", "step", "step", "norm", "norm_train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind in ("norm", "norm_train"):
        heads = rng.choice([1, 1, 4, 16, 32])
        width = rng.choice([64, 96, 128, 256]) if heads > 1 else _spread(rng, 8, 8192)
        rows = _spread(rng, 1, max(2, 16384 * 4096 // (heads * width) // 4))
        case = _norm("", kind, dtype, rows, heads, width)
    else:
        key_heads = rng.choice([1, 2, 4, 8, 16])
        heads = key_heads * rng.choice([1, 1, 2, 3])
        key_dim, value_dim = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (96, 80), (40, 72), (128, 256)])
        gates = rng.choice([dtype, "float32"]) if kind != "train" else dtype
        if kind == "step":
            batch = _spread(rng, 1, 256 * 32 // heads // 2)
            case = _step("", dtype, gates, batch, batch + rng.randrange(9), key_heads, heads, key_dim, value_dim)
        else:
            most = 16384 * 32 if kind == "prompt" else 8192 * 16
            tokens = _spread(rng, 1, max(2, most // heads // (1 if dtype != "float32" else 4)))
            tokens = min(tokens, 20000)
            if rng.random() < 0.5:
                cuts = sorted(rng.randrange(tokens + 1) for _ in range(rng.randrange(7)))
                ends = cuts + [tokens]
                lengths = ",".join(str(b - a) for a, b in zip([0] + cuts, ends))
                case = _scan("", kind, dtype, gates, 1, tokens, key_heads, heads, key_dim, value_dim, lengths, True)
            else:
                batch = rng.choice([1, 2, 3, 4])
                case = _scan("", kind, dtype, gates, batch, max(1, tokens // batch), key_heads, heads, key_dim,
                             value_dim, "", rng.random() < 0.5)
    del case["name"]
    return case


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    state = {"case": case}
    if case["kind"] in ("norm", "norm_train"):
        shape = (case["rows"], case["heads"], case["width"])
        state["x"] = normal(*shape).to(dtype)
        state["gate"] = normal(*shape).to(dtype)
        state["weight"] = (1 + 0.1 * normal(case["width"])).to(dtype)
        if case["kind"] == "norm_train":
            state["d_out"] = normal(*shape).to(dtype)
        return state

    lead = (case["batch"],) if case["kind"] == "step" else (case["batch"], case["tokens"])
    heads, key_dim, value_dim = case["heads"], case["key_dim"], case["value_dim"]
    # keys and queries of unit length, as a layer hands them over; gates and beta as its projections give them
    for name in ("q", "k"):
        rows = normal(*lead, case["key_heads"], key_dim)
        state[name] = (rows / rows.square().sum(-1, keepdim=True).sqrt()).to(dtype)
    state["v"] = normal(*lead, heads, value_dim).to(dtype)
    rate = torch.exp(2.5 * torch.rand(heads, generator=gen, device="cuda") - 4)
    state["log_gates"] = (-rate * torch.log1p(torch.exp(normal(*lead, heads)))).to(DTYPES[case["gates"]])
    state["beta"] = torch.sigmoid(normal(*lead, heads)).to(DTYPES[case["gates"]])
    if case["kind"] == "step":
        # states as earlier tokens left them, and the slots of this batch's conversations in no order
        state["states"] = normal(case["slots"], heads, key_dim, value_dim) * 0.3
        state["slots"] = torch.randperm(case["slots"], generator=gen, device="cuda")[: case["batch"]].to(torch.int32)
        return state
    sequences = case["batch"]
    state["offsets"] = None
    if case["lengths"]:
        lengths = [int(n) for n in case["lengths"].split(",")]
        ends = [sum(lengths[:n]) for n in range(len(lengths) + 1)]
        state["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        sequences = len(lengths)
    state["initial"] = normal(sequences, heads, key_dim, value_dim) * 0.3 if case["start"] else None
    if case["kind"] == "train":
        state["d_out"] = normal(*lead, heads, value_dim).to(dtype)
        state["d_final"] = normal(sequences, heads, key_dim, value_dim) * 0.3
    return state


# ---------------------------------------------------------------------------------------------------------------
# Plain forms: 32 bits, rounded once at the end
# ---------------------------------------------------------------------------------------------------------------
def _inverse(lower):
    """(I + lower)^-1 of strictly lower triangular blocks (..., BLOCK, BLOCK): inverses of the diagonal's blocks
    joined to blocks of twice the size, [[A, 0], [C, D]]^-1 = [[A', 0], [-D' C A', D']], from 1 to BLOCK."""
    inverse = torch.ones(*lower.shape[:-2], BLOCK, 1, 1, device=lower.device)
    size = 1
    while size < BLOCK:
        pairs = BLOCK // (2 * size)
        cells = lower.reshape(*lower.shape[:-2], pairs, 2, size, pairs, 2, size)
        corner = torch.stack([cells[..., n, 1, :, n, 0, :] for n in range(pairs)], dim=-3)
        first, second = inverse[..., 0::2, :, :], inverse[..., 1::2, :, :]
        joined = -(second @ corner @ first)
        upper = torch.cat([first, torch.zeros_like(first)], dim=-1)
        inverse = torch.cat([upper, torch.cat([joined, second], dim=-1)], dim=-2)
        size *= 2
    return inverse[..., 0, :, :]


def _plain_scan(q, k, v, log_gates, beta, initial, scale):
    """Batches (N, T, heads, dim) of whole sequences, a block of BLOCK tokens at a time: inside a block all tokens at
    once, from block to block through the state (that loop is the recurrence itself)."""
    batch, tokens, heads, value_dim = v.shape
    shared = heads // q.shape[2]
    blocks = -(-tokens // BLOCK)

    def cut(t):
        t = torch.nn.functional.pad(t, (0, 0) * (t.dim() - 2) + (0, blocks * BLOCK - tokens))
        return t.reshape(batch, blocks, BLOCK, *t.shape[2:]).transpose(2, 3)  # (N, blocks, heads, BLOCK, ...)

    q = cut(q.float()).repeat_interleave(shared, dim=2) * scale
    k = cut(k.float()).repeat_interleave(shared, dim=2)
    v, beta = cut(v.float()), cut(beta.float())
    decay = cut(log_gates.double()).cumsum(-1)  # sums whose differences count: 64 bits
    i = torch.arange(BLOCK, device=v.device)
    between = (decay[..., :, None] - decay[..., None, :]).float()
    between = torch.exp(between.masked_fill(i[:, None] < i, -math.inf))
    since, until, whole = (torch.exp(x.float()) for x in (decay, decay[..., -1:] - decay, decay[..., -1]))
    inverse = _inverse((beta[..., None] * between * (k @ k.transpose(-1, -2))).masked_fill(i[:, None] <= i, 0))
    scores = between * (q @ k.transpose(-1, -2))
    own_part = inverse @ (beta[..., None] * v)
    state_part = inverse @ ((beta * since)[..., None] * k)
    keys_until = (k * until[..., None]).transpose(-1, -2)
    queries_since = q * since[..., None]
    state = initial if initial is not None else v.new_zeros(batch, heads, k.shape[-1], value_dim)
    out = []
    for n in range(blocks):
        update = own_part[:, n] - state_part[:, n] @ state
        out.append(queries_since[:, n] @ state + scores[:, n] @ update)
        state = whole[:, n, :, None, None] * state + keys_until[:, n] @ update
    out = torch.stack(out, dim=1).transpose(2, 3).reshape(batch, blocks * BLOCK, heads, value_dim)
    return out[:, :tokens], state


def _plain_sequences(q, k, v, log_gates, beta, initial, scale, offsets, longest):
    """Packed sequences: gathered into a padded batch, scanned, and put back."""
    if offsets is None:
        return _plain_scan(q, k, v, log_gates, beta, initial, scale)
    at = offsets[:-1, None] + torch.arange(longest, device=v.device)
    there = at < offsets[1:, None]
    at = at.clamp(max=v.shape[1] - 1)
    padded = [torch.where(there.reshape(*there.shape, *[1] * (t.dim() - 2)), t[0][at], 0)
              for t in (q, k, v, log_gates, beta)]
    out, final = _plain_scan(*padded, initial, scale)
    return out[there][None], final


def _plain_norm(x, gate, weight):
    x, gate = x.float(), gate.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float() * (gate * torch.sigmoid(gate))


def _longest(case):
    return max(int(n) for n in case["lengths"].split(",")) if case["lengths"] else case["tokens"]


def _package():
    """This repository's package, which lies in a folder of its own beside this one."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "accelerated-scan_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from accelerated_scan import delta, norm

    return delta, norm


def run(state):
    case = state["case"]
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        if own:
            _, norm = _package()
            return norm.gated_norm(state["x"], state["gate"], state["weight"], eps=EPS)
        return _plain_norm(state["x"], state["gate"], state["weight"]).to(dtype)
    if case["kind"] == "norm_train":
        leaves = [state[name].detach().requires_grad_() for name in ("x", "gate", "weight")]
        if own:
            _, norm = _package()
            out = norm.gated_norm(*leaves, eps=EPS)
        else:
            out = _plain_norm(*leaves).to(dtype)
        return {"out": out.detach(), "grads": list(torch.autograd.grad(out, leaves, state["d_out"]))}

    scale = case["key_dim"] ** -0.5
    if case["kind"] == "step":
        inputs = [state[name] for name in ("q", "k", "v", "log_gates", "beta")]
        if own:
            delta, _ = _package()
            out = delta.gated_delta_step(*inputs, state["states"], slots=state["slots"], scale=scale)
            return {"out": out, "states": state["states"]}
        shared = case["heads"] // case["key_heads"]
        q, k, v, log_gates, beta = (t.float() for t in inputs)
        q, k = q.repeat_interleave(shared, dim=1) * scale, k.repeat_interleave(shared, dim=1)
        slots = state["slots"].long()
        new = state["states"][slots] * torch.exp(log_gates)[..., None, None]
        update = beta[..., None] * (v - (k[..., None, :] @ new)[..., 0, :])
        new = new + k[..., :, None] * update[..., None, :]
        state["states"][slots] = new
        return {"out": (q[..., None, :] @ new)[..., 0, :].to(dtype), "states": state["states"]}

    names = ["q", "k", "v", "log_gates", "beta"] + (["initial"] if state["initial"] is not None else [])
    train = case["kind"] == "train"
    leaves = [state[name].detach().requires_grad_(train) for name in names]
    initial = leaves[5] if len(leaves) > 5 else None
    if own:
        delta, _ = _package()
        out, final = delta.gated_delta_scan(*leaves[:5], initial=initial, scale=scale, offsets=state["offsets"])
    else:
        out, final = _plain_sequences(*leaves[:5], initial, scale, state["offsets"], _longest(case))
        out = out.to(dtype)
    if not train:
        return {"out": out, "final": final}
    grads = torch.autograd.grad([out, final], leaves, [state["d_out"], state["d_final"]])
    return {"out": out.detach(), "final": final.detach(), "grads": list(grads)}


def work(case):
    """Inputs read once and outputs written once; operations of the token-by-token formulas, a multiplication and an
    addition counted as two, without the elementwise ones."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] in ("norm", "norm_train"):
        n = case["rows"] * case["heads"] * case["width"]
        train = case["kind"] == "norm_train"
        return {"bytes": n * size * (6 if train else 3), "flops": n * (20 if train else 7)}
    gate_size = 4 if case["gates"] == "float32" else 2
    tokens = case["batch"] * case.get("tokens", 1)
    heads, cells = case["heads"], case["key_dim"] * case["value_dim"]
    qk, v = 2 * case["key_heads"] * case["key_dim"] * size, heads * case["value_dim"] * size
    gates = 2 * heads * gate_size
    sequences = len(case["lengths"].split(",")) if case.get("lengths") else case["batch"]
    state = sequences * heads * cells * 4
    if case["kind"] == "step":
        return {"bytes": tokens * (qk + 2 * v + gates) + 2 * state, "flops": tokens * heads * cells * 6}
    started = 1 if case["start"] else 0
    if case["kind"] == "prompt":
        return {"bytes": tokens * (qk + 2 * v + gates) + state * (1 + started), "flops": tokens * heads * cells * 6}
    # forward, then inputs and the two incoming gradients in, gradients of all inputs out
    moved = tokens * ((qk + 2 * v + gates) + (qk + 2 * v + gates) + (qk + v + gates)) + state * (2 + 2 * started)
    return {"bytes": moved, "flops": tokens * heads * cells * (6 + 12)}


# ---------------------------------------------------------------------------------------------------------------
# The definition, token by token, in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _exact_span(S, q, k, v, log_gates, beta, scale):
    """States after the tokens of a span and their outputs; tensors (N, T, heads, ...), heads already shared out."""
    out = []
    for t in range(q.shape[1]):
        S = S * log_gates[:, t, :, None, None].exp()
        kept = (S * k[:, t, :, :, None]).sum(-2)
        S = S + k[:, t, :, :, None] * (beta[:, t, :, None] * (v[:, t] - kept))[:, :, None, :]
        out.append(scale * (S * q[:, t, :, :, None]).sum(-2))
    return S, torch.stack(out, 1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("norm", "norm_train"):
        x, z, w = (state[name].double() for name in ("x", "gate", "weight"))
        inv = 1 / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
        s = 1 / (1 + (-z).exp())
        out = x * inv * w * z * s
        if case["kind"] == "norm":
            return out
        d = state["d_out"].double()
        du = d * w * z * s
        dx = inv * (du - x * inv.pow(2) * (du * x).mean(-1, keepdim=True))
        dz = d * w * x * inv * (s + z * s * (1 - s))
        return {"out": out, "grads": [dx, dz, (d * x * inv * z * s).sum((0, 1))]}

    scale, shared = case["key_dim"] ** -0.5, case["heads"] // case["key_heads"]
    inputs = [state[name].double() for name in ("q", "k", "v", "log_gates", "beta")]
    if case["kind"] == "step":
        slots = state["slots"].long()
        share = [inputs[0].repeat_interleave(shared, 1), inputs[1].repeat_interleave(shared, 1), *inputs[2:]]
        S, out = _exact_span(state["states"][slots].double(), *(t[:, None] for t in share), scale)
        states = state["states"].double()
        states[slots] = S
        return {"out": out[:, 0], "states": states}

    if case["lengths"]:  # one sequence after the other into a batch padded with tokens that change nothing
        lengths = [int(n) for n in case["lengths"].split(",")]
        apart = []
        for t in inputs:
            wide = t.new_zeros(len(lengths), max(lengths), *t.shape[2:])
            for n, piece in enumerate(t[0].split(lengths)):
                wide[n, : lengths[n]] = piece
            apart.append(wide)
    else:
        lengths, apart = [case["tokens"]] * case["batch"], inputs
    longest = max(lengths)
    start = state["initial"].double() if state["initial"] is not None else None
    S = start if start is not None else apart[2].new_zeros(len(lengths), case["heads"], case["key_dim"], case["value_dim"])

    def together(t):
        return torch.cat([t[n, : lengths[n]] for n in range(len(lengths))])[None] if case["lengths"] else t

    def span_inputs(first, last):
        return [t[:, first:last].detach() for t in apart]

    def span(S, q, k, *rest):
        return _exact_span(S, q.repeat_interleave(shared, 2), k.repeat_interleave(shared, 2), *rest, scale)

    edges, states, out = list(range(0, longest, BLOCK)), [], []
    with torch.no_grad():
        for first in edges:
            states.append(S)
            S, o = span(S, *span_inputs(first, first + BLOCK))
            out.append(o)
    result = {"out": together(torch.cat(out, 1)), "final": S}
    if case["kind"] != "train":
        return result
    d_out = state["d_out"].double()
    if case["lengths"]:
        wide = d_out.new_zeros(len(lengths), longest, *d_out.shape[2:])
        for n, piece in enumerate(d_out[0].split(lengths)):
            wide[n, : lengths[n]] = piece
        d_out = wide
    d_S, grads = state["d_final"].double(), [[] for _ in apart]
    for first, S0 in zip(reversed(edges), reversed(states)):  # span by span from the end, each differentiated by itself
        leaves = [t.requires_grad_() for t in [S0.detach(), *span_inputs(first, first + BLOCK)]]
        S1, o = span(*leaves)
        d_S, *found = torch.autograd.grad([S1, o], leaves, [d_S, d_out[:, first: first + BLOCK]])
        for to, g in zip(grads, found):
            to.insert(0, g)
    result["grads"] = [together(torch.cat(g, 1)) for g in grads] + ([d_S] if start is not None else [])
    return result
