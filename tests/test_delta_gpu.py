"""Gated delta rule on the GPU against the token-by-token recurrence in float64 (tests/delta_reference.py, where
the error bounds are derived)."""

import pytest
import torch

import delta_reference as ref

pytestmark = pytest.mark.gpu

DEVICE = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("queries", "keys", "values", "log_gates", "beta", "initial")


def on_gpu(tensors, grad=False):
    return [t.to(DEVICE).requires_grad_(grad) for t in tensors]


def as_exact(tensors, grad=False):
    return [t.double().requires_grad_(grad) for t in tensors]


SHAPES = [
    # B, T, key heads, heads, dk, dv
    (1, 1, 1, 1, 64, 64),
    (2, 2, 1, 2, 8, 8),
    (1, 63, 2, 2, 32, 48),
    (1, 64, 1, 3, 64, 64),
    (2, 65, 2, 4, 128, 128),
    (1, 129, 1, 1, 96, 80),
    (1, 200, 1, 2, 40, 200),
    (1, 191, 2, 2, 128, 256),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(shape, dtype):
    from accelerated_scan import delta

    data = ref.inputs(*shape, dtype, seed=1)
    want, final = ref.delta_scan(*as_exact(data))
    got, state = delta.gated_delta_scan(*on_gpu(data))
    assert got.dtype == dtype and state.dtype == torch.float32
    ref.close(got, want, dtype, what="out")
    ref.close(state, final, dtype, what="final")
    want, final = ref.delta_scan(*as_exact(data[:5]), scale=0.7)  # no initial state, a scale of one's own
    got, state = delta.gated_delta_scan(*on_gpu(data[:5]), scale=0.7)
    ref.close(got, want, dtype, what="out")
    ref.close(state, final, dtype, what="final")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients(shape, dtype):
    from accelerated_scan import delta

    data = ref.inputs(*shape, dtype, seed=2)
    exact = as_exact(data, grad=True)
    out, final = ref.delta_scan(*exact)
    gen = torch.Generator().manual_seed(5)
    d_out = torch.randn(out.shape, generator=gen).to(dtype)
    d_final = 0.3 * torch.randn(final.shape, generator=gen)
    want = torch.autograd.grad([out, final], exact, [d_out.double(), d_final.double()])
    leaves = on_gpu(data, grad=True)
    got = torch.autograd.grad(delta.gated_delta_scan(*leaves), leaves, on_gpu([d_out, d_final]))
    for name, a, b, leaf in zip(NAMES, got, want, leaves):
        assert a.dtype == leaf.dtype
        ref.close(a, b, dtype, backward=True, what=name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_gates_in_32_bits_beside_16_bit_tensors(dtype):
    from accelerated_scan import delta

    data = ref.inputs(2, 150, 2, 4, 64, 72, dtype, seed=3, gates=torch.float32)
    exact = as_exact(data, grad=True)
    out, final = ref.delta_scan(*exact)
    d_out = torch.randn(out.shape, generator=torch.Generator().manual_seed(6)).to(dtype)
    want = torch.autograd.grad(out, exact, d_out.double())
    leaves = on_gpu(data, grad=True)
    got_out, got_final = delta.gated_delta_scan(*leaves)
    ref.close(got_out, out, dtype)
    ref.close(got_final, final, dtype)
    for name, a, b in zip(NAMES, torch.autograd.grad(got_out, leaves, d_out.to(DEVICE)), want):
        ref.close(a, b, dtype, backward=True, what=name)


@pytest.mark.parametrize("wide", [False, True], ids=["int32", "int64"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_packed_sequences(dtype, wide):
    """Sequences of many lengths, empty ones among them, behind rows that belong to none: those are not read."""
    from accelerated_scan import delta

    lengths, front, back = [3, 0, 64, 1, 130, 0, 65, 63], 5, 70
    T = front + sum(lengths) + back
    data = ref.inputs(1, T, 2, 4, 48, 56, dtype, seed=4, sequences=len(lengths))
    for t in data[:5]:
        t[:, :front] = float("nan")
        t[:, T - back:] = float("inf")
    ends = [front + sum(lengths[:n]) for n in range(len(lengths) + 1)]
    offsets = torch.tensor(ends, dtype=torch.int64 if wide else torch.int32, device=DEVICE)
    gen = torch.Generator().manual_seed(7)
    d_out = torch.randn(1, T, 4, 56, generator=gen).to(dtype)
    d_final = torch.randn(len(lengths), 4, 48, 56, generator=gen)
    leaves = on_gpu(data, grad=True)
    got, final = delta.gated_delta_scan(*leaves, offsets=offsets)
    grads = torch.autograd.grad([got, final], leaves, on_gpu([d_out, d_final]))
    for rows in (slice(0, front), slice(T - back, T)):
        assert not got[:, rows].any()
        for g in grads[:5]:
            assert not g[:, rows].any()
    want_out, want_final, want = [], [], []
    for n in range(len(lengths)):
        rows = slice(ends[n], ends[n + 1])
        one = [t[:, rows].double().requires_grad_() for t in data[:5]] + [data[5][n:n + 1].double().requires_grad_()]
        o, f = ref.delta_scan(*one)
        want_out.append(o)
        want_final.append(f)
        want.append(torch.autograd.grad([o, f], one, [d_out[:, rows].double(), d_final[n:n + 1].double()],
                                        allow_unused=True, materialize_grads=True))
    inside = slice(front, T - back)
    ref.close(got[:, inside], torch.cat(want_out, 1), dtype)
    ref.close(final, torch.cat(want_final), dtype)
    for i, name in enumerate(NAMES):
        w = torch.cat([g[i] for g in want], 1 if i < 5 else 0)
        ref.close(grads[i][:, inside] if i < 5 else grads[i], w, dtype, backward=True, what=name)


def test_many_packed_sequences():
    """More sequences than a wave has lanes: the tables' search."""
    from accelerated_scan import delta

    gen = torch.Generator().manual_seed(8)
    lengths = torch.randint(0, 9, (300,), generator=gen).tolist()
    lengths[170] = 200
    T = sum(lengths)
    data = ref.inputs(1, T, 1, 1, 16, 16, torch.float32, seed=9, sequences=len(lengths))
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).to(DEVICE)
    got, final = delta.gated_delta_scan(*on_gpu(data), offsets=offsets)
    at = 0
    for n, length in enumerate(lengths):
        o, f = ref.delta_scan(*[t[:, at:at + length].double() for t in data[:5]], data[5][n:n + 1].double())
        ref.close(final[n:n + 1], f, torch.float32)
        ref.close(got[:, at:at + length], o, torch.float32)
        at += length


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_closed_and_strong_gates(dtype):
    """Log gates of -inf, of the type's lowest value and far below what an exponential holds start the state anew,
    and tokens behind them are as exact as any."""
    from accelerated_scan import delta

    data = ref.inputs(1, 150, 1, 2, 32, 32, dtype, seed=10)
    g = data[3]
    g[0, 0, 0] = g[0, 70, 0] = g[0, 71, 1] = float("-inf")
    g[0, 100, 1] = torch.finfo(dtype).min
    g[0, 30:60, 1] = -90.0
    g[0, 149, 0] = -1e4
    exact = as_exact(data, grad=True)
    out, final = ref.delta_scan(*exact)
    d_out = torch.randn(out.shape, generator=torch.Generator().manual_seed(11)).to(dtype)
    # the loop's own gradient at exp(-inf) is 0 * S, finite: states are
    want = torch.autograd.grad(out, exact, d_out.double())
    leaves = on_gpu(data, grad=True)
    got, state = delta.gated_delta_scan(*leaves)
    ref.close(got, out, dtype)
    ref.close(state, final, dtype)
    for name, a, b in zip(NAMES, torch.autograd.grad(got, leaves, d_out.to(DEVICE)), want):
        ref.close(a, b, dtype, backward=True, what=name)


def test_open_gates_and_equal_keys():
    """The matrix to invert at its worst: one key again and again, beta 1, gates 1, and beta up to 2."""
    from accelerated_scan import delta

    for top in (1.0, 2.0):
        data = ref.inputs(1, 200, 1, 1, 64, 64, torch.float32, seed=12)
        data[1][:] = data[1][:, :1]
        data[3].zero_()
        data[4].fill_(top)
        want, final = ref.delta_scan(*as_exact(data))
        got, state = delta.gated_delta_scan(*on_gpu(data))
        # |1 - beta| = 1 for beta = 2: errors of 200 tokens add up instead of fading, sqrt(200) < 16 times the bound
        ref.close(got, want, torch.float32, grow=16.0)
        ref.close(state, final, torch.float32, grow=16.0)


@pytest.mark.parametrize("which", ["out", "final"])
def test_one_of_the_two_results_differentiated(which):
    from accelerated_scan import delta

    data = ref.inputs(2, 100, 1, 2, 32, 32, torch.float32, seed=13)
    exact, leaves = as_exact(data, grad=True), on_gpu(data, grad=True)
    n = 0 if which == "out" else 1
    want_of, got_of = ref.delta_scan(*exact)[n], delta.gated_delta_scan(*leaves)[n]
    d = torch.randn(want_of.shape, generator=torch.Generator().manual_seed(14))
    used = range(6) if which == "out" else range(1, 6)  # the final state does not depend on the queries
    want = torch.autograd.grad(want_of, [exact[i] for i in used], d.double())
    got = torch.autograd.grad(got_of, leaves, d.to(DEVICE))
    if which == "final":
        assert not got[0].any()
    for i, b in zip(used, want):
        ref.close(got[i], b, torch.float32, backward=True, what=NAMES[i])


def test_gradient_against_differences():
    """Central differences of the operator itself along random directions, in fp32: with a step of 2^-5 the
    truncation is of the order of 2^-10 of the third derivative and the operator's own error of 2^-20 of the sum's
    size is divided by 2^-4, so the two agree to 2^-8 of the largest directional derivative."""
    from accelerated_scan import delta

    data = on_gpu(ref.inputs(1, 90, 1, 2, 32, 32, torch.float32, seed=15), grad=True)
    gen = torch.Generator(device=DEVICE).manual_seed(16)
    out, final = delta.gated_delta_scan(*data)
    d_out = torch.randn(out.shape, generator=gen, device=DEVICE)
    d_final = torch.randn(final.shape, generator=gen, device=DEVICE)

    def value(tensors):
        with torch.no_grad():
            o, f = delta.gated_delta_scan(*tensors)
            return ((o.double() * d_out).sum() + (f.double() * d_final).sum()).item()

    grads = torch.autograd.grad([out, final], data, [d_out, d_final])
    slopes, wants = [], []
    for i, (t, g) in enumerate(zip(data, grads)):
        direction = torch.randn(t.shape, generator=gen, device=DEVICE)
        direction *= 1 / direction.norm()
        h = 2.0 ** -5
        moved = [[x.detach() + (s * h * direction if j == i else 0) for j, x in enumerate(data)] for s in (1, -1)]
        slopes.append((value(moved[0]) - value(moved[1])) / (2 * h))
        wants.append((g.double() * direction).sum().item())
    most = max(map(abs, wants))
    for name, a, b in zip(NAMES, slopes, wants):
        assert abs(a - b) <= 2.0 ** -8 * most, (name, a, b)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1, 1, 64, 64), (3, 2, 4, 128, 128), (5, 1, 2, 40, 72), (2, 2, 2, 8, 520)], ids=str)
def test_step(shape, dtype):
    from accelerated_scan import delta

    B, key_heads, heads, dk, dv = shape
    data = ref.inputs(B, 1, key_heads, heads, dk, dv, dtype, seed=17)
    want, final = ref.delta_scan(*as_exact(data))
    *inputs, state = on_gpu(data)
    got = delta.gated_delta_step(*[t[:, 0].contiguous() for t in inputs], state)
    assert got.dtype == dtype
    ref.close(got, want[:, 0], dtype)
    ref.close(state, final, torch.float32)


@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=str)
def test_step_slots(index):
    """States in a pool: rows without one, rows that share one (tokens of it in their order), the rest untouched."""
    from accelerated_scan import delta

    slots = torch.tensor([7, 2, -1, 2, 0, 9, 2, 100, 7])
    data = ref.inputs(len(slots), 1, 1, 2, 32, 40, torch.float32, seed=18, sequences=10)
    q, k, v, g, b, pool = as_exact(data)
    want, want_pool = torch.zeros_like(v[:, 0]), pool.clone()
    for row, slot in enumerate(slots.tolist()):
        if 0 <= slot < 10:
            one = [t[row:row + 1] for t in (q, k, v, g, b)]
            o, want_pool[slot:slot + 1] = ref.delta_scan(*one, want_pool[slot:slot + 1].clone())
            want[row] = o[0, 0]
    *inputs, states = on_gpu(data)
    before = states.clone()
    got = delta.gated_delta_step(*[t[:, 0].contiguous() for t in inputs], states, slots=slots.to(index).to(DEVICE))
    ref.close(got, want, torch.float32)
    ref.close(states, want_pool, torch.float32)
    for slot in (1, 3, 4, 5, 6, 8):
        assert torch.equal(states[slot], before[slot])
    for row in (2, 7):
        assert not got[row].any()


def test_step_with_many_rows_of_one_slot():
    """More rows than a workgroup has threads, all tokens of one state."""
    from accelerated_scan import delta

    data = ref.inputs(1, 600, 1, 1, 16, 16, torch.float32, seed=19)
    want, final = ref.delta_scan(*as_exact(data))
    *inputs, state = on_gpu(data)
    got = delta.gated_delta_step(*[t[0].contiguous() for t in inputs], state,
                                 slots=torch.zeros(600, dtype=torch.int32, device=DEVICE))
    ref.close(got, want[0], torch.float32)
    ref.close(state, final, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_prompt_then_tokens_then_norm(dtype):
    """As a program runs them: a prompt in two pieces, new tokens one by one, each output through the gated norm --
    against one run over all tokens."""
    from accelerated_scan import delta, norm

    B, T, heads, dk, dv = 2, 140, 4, 64, 64
    data = ref.inputs(B, T, 2, heads, dk, dv, dtype, seed=20)
    gen = torch.Generator().manual_seed(21)
    gate, weight = torch.randn(B, T, heads, dv, generator=gen).to(dtype), torch.randn(dv, generator=gen).to(dtype)
    want, final = ref.delta_scan(*as_exact(data))
    *inputs, state = on_gpu(data)
    parts, cuts = [], [0, 70, 130]
    for a, b in zip(cuts, cuts[1:]):
        out, state = delta.gated_delta_scan(*[t[:, a:b].contiguous() for t in inputs], state)
        parts.append(out)
    for t in range(cuts[-1], T):
        parts.append(delta.gated_delta_step(*[x[:, t].contiguous() for x in inputs], state)[:, None])
    out = torch.cat(parts, 1)
    ref.close(out, want, dtype)
    ref.close(state, final, dtype)
    # the norm of what the kernels gave: held to its own rounding (a dozen fp32 operations, 12 * 2^-24 < 2^-20)
    got = norm.gated_norm(out, gate.to(DEVICE), weight.to(DEVICE))
    exact = ref.gated_norm(out.cpu().double(), gate.double(), weight.double())
    u = torch.finfo(dtype).eps / 2 + 2.0 ** -20
    # below the type's normal numbers the step no longer shrinks with the value (fp16: half a step of 2^-25)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 + 2.0 ** -40
    assert ((got.cpu().double() - exact).abs() <= u * exact.abs() + tiny).all()


def test_layer_gradients():
    """Projections, scan, gated norm and projection: parameter gradients against the same layer in float64."""
    from accelerated_scan import delta, norm

    B, T, dim, heads, hd = 2, 100, 24, 2, 16
    gen = torch.Generator().manual_seed(22)
    u = torch.randn(B, T, dim, generator=gen)
    sizes = {"q": heads * hd, "k": heads * hd, "v": heads * hd, "z": heads * hd, "g": heads, "b": heads}
    params = {n: torch.randn(s, dim, generator=gen) / dim ** 0.5 for n, s in sizes.items()}
    params["o"] = torch.randn(dim, heads * hd, generator=gen) / (heads * hd) ** 0.5
    params["w"] = 1 + 0.1 * torch.randn(hd, generator=gen)
    target = torch.randn(B, T, dim, generator=gen)

    def layer(p, u, scan, gated):
        cut = lambda t: t.reshape(B, T, heads, hd)  # noqa: E731
        q, k, v, z = (cut(u @ p[n].T) for n in "qkvz")
        q, k = (torch.nn.functional.normalize(t, dim=-1) for t in (q, k))
        o, _ = scan(q, k, v, -torch.nn.functional.softplus(u @ p["g"].T), torch.sigmoid(u @ p["b"].T))
        return gated(o, z, p["w"]).reshape(B, T, heads * hd) @ p["o"].T

    def grads(device, dtype, scan, gated):
        p = {n: t.to(device=device, dtype=dtype).requires_grad_() for n, t in params.items()}
        loss = (layer(p, u.to(device=device, dtype=dtype), scan, gated) - target.to(device=device, dtype=dtype)).square().mean()
        return dict(zip(p, torch.autograd.grad(loss, list(p.values()))))

    got = grads(DEVICE, torch.float32, delta.gated_delta_scan, norm.gated_norm)
    want = grads("cpu", torch.float64, ref.delta_scan, ref.gated_norm)
    for n in params:
        # the operators' 144 * 2^-22 and the projections' and the norm's sums of up to 200 products in fp32 on the way
        ref.close(got[n], want[n], torch.float32, backward=True, what=n, grow=4.0)


def test_results_repeat_bit_for_bit():
    from accelerated_scan import delta

    data = on_gpu(ref.inputs(2, 300, 2, 4, 64, 64, torch.bfloat16, seed=23), grad=True)
    runs = []
    for _ in range(3):
        out, final = delta.gated_delta_scan(*data)
        runs.append([out, final, *torch.autograd.grad([out, final], data, [torch.ones_like(out), torch.ones_like(final)])])
    for run in runs[1:]:
        for a, b in zip(runs[0], run):
            assert torch.equal(a, b)


def test_captured_graphs_and_other_streams():
    """Two captured graphs and eager work in turn: each call owns its workspace."""
    from accelerated_scan import delta

    first = on_gpu(ref.inputs(1, 200, 1, 2, 64, 64, torch.bfloat16, seed=24))
    second = on_gpu(ref.inputs(1, 333, 1, 2, 64, 64, torch.bfloat16, seed=25))
    eager = [delta.gated_delta_scan(*x) for x in (first, second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = delta.gated_delta_scan(*first)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager[0], again))
    graphs, results = [], []
    for x in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            results.append(delta.gated_delta_scan(*x))
        graphs.append(g)
    for turn in range(4):
        for r in results:
            for t in r:
                t.zero_()
        for g in graphs:
            g.replay()
        delta.gated_delta_scan(*first)
        torch.cuda.synchronize()
        for want, got in zip(eager, results):
            assert all(torch.equal(a, b) for a, b in zip(want, got)), turn
    # a captured step moves its states on at every replay
    q, k, v, g_, b, _ = second
    token = [t[:, 0].contiguous() for t in (q, k, v, g_, b)]
    states, mirror = torch.zeros(1, 2, 64, 64, device=DEVICE), torch.zeros(1, 2, 64, 64, device=DEVICE)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = delta.gated_delta_step(*token, states)
    states.zero_()
    for _ in range(3):
        graph.replay()
        want = delta.gated_delta_step(*token, mirror)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(states, mirror)


def test_compiled():
    from accelerated_scan import delta, norm

    data = on_gpu(ref.inputs(1, 100, 1, 2, 32, 32, torch.float32, seed=26), grad=True)
    weight = torch.ones(32, device=DEVICE, requires_grad=True)

    def loss(*x):
        out, final = delta.gated_delta_scan(*x)
        return norm.gated_norm(out, x[2], weight).square().sum() + final.sum()

    want = torch.autograd.grad(loss(*data), [*data, weight])
    got = torch.autograd.grad(torch.compile(loss, backend="aot_eager", fullgraph=True)(*data), [*data, weight])
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=2e-6, atol=2e-6 * b.abs().max().item())  # the same kernels; the sums around differ
    with torch.no_grad():
        token = [t.detach()[:, 0].contiguous() for t in data[:5]]
        state, mirror = data[5].detach().clone(), data[5].detach().clone()
        out = torch.compile(lambda *x: delta.gated_delta_step(*x), backend="aot_eager", fullgraph=True)(*token, state)
        assert torch.equal(out, delta.gated_delta_step(*token, mirror)) and torch.equal(state, mirror)


def test_operators_by_themselves():
    from accelerated_scan import _ops

    data = on_gpu(ref.inputs(1, 70, 1, 2, 16, 16, torch.float32, seed=27), grad=True)
    torch.library.opcheck(_ops.delta_forward, (*data, None, 0.25, True))
    plain = [t.detach() for t in data]
    out, final, states, updates = _ops.delta_forward(*plain, None, 0.25, True)
    torch.library.opcheck(_ops.delta_backward, (*plain[:5], states, updates, None, 0.25, out, final, True))
    token = [t[:, 0].contiguous() for t in plain[:5]]
    torch.library.opcheck(_ops.delta_step, (*token, plain[5].clone(), None, 0.25))
    x, w = plain[2], torch.ones(16, device=DEVICE)
    torch.library.opcheck(_ops.gated_norm, (x, x + 1, w, 1e-6))
    torch.library.opcheck(_ops.gated_norm_backward, (x, x + 1, w, x, 1e-6))


def test_empty_inputs():
    from accelerated_scan import delta

    new = lambda *s: torch.zeros(*s, device=DEVICE)  # noqa: E731
    start = torch.randn(2, 2, 16, 16, device=DEVICE, requires_grad=True)
    out, final = delta.gated_delta_scan(new(2, 0, 1, 16), new(2, 0, 1, 16), new(2, 0, 2, 16), new(2, 0, 2), new(2, 0, 2), start)
    assert out.shape == (2, 0, 2, 16) and torch.equal(final, start)
    (d,) = torch.autograd.grad(final, start, torch.ones_like(final))
    assert torch.equal(d, torch.ones_like(d))
    out, final = delta.gated_delta_scan(new(0, 5, 1, 16), new(0, 5, 1, 16), new(0, 5, 2, 16), new(0, 5, 2), new(0, 5, 2))
    assert out.shape == (0, 5, 2, 16) and final.shape == (0, 2, 16, 16)
    nothing = torch.zeros(1, dtype=torch.int32, device=DEVICE)
    out, final = delta.gated_delta_scan(new(1, 5, 1, 16) + 1, new(1, 5, 1, 16), new(1, 5, 2, 16) + 1, new(1, 5, 2), new(1, 5, 2),
                                        offsets=nothing)
    assert not out.any() and final.shape == (0, 2, 16, 16)
    step = delta.gated_delta_step(new(0, 1, 16), new(0, 1, 16), new(0, 2, 16), new(0, 2), new(0, 2), new(0, 2, 16, 16))
    assert step.shape == (0, 2, 16)


@pytest.mark.parametrize("t", [0, 37, 64, 149])
@pytest.mark.parametrize("what", ["queries", "keys", "values", "log_gates", "beta"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_tokens_that_are_not_finite_leave_earlier_ones_alone(dtype, what, t):
    """As in a padded batch whose padding holds anything."""
    from accelerated_scan import delta

    for dk, bad in ((64, float("nan")), (128, float("inf"))):
        data = ref.inputs(1, 150, 2, 2, dk, 40, dtype, seed=31)
        want, state = ref.delta_scan(*as_exact(data))
        broken = [x.clone() for x in data]
        x = broken[NAMES.index(what)]
        if x.dim() == 4:
            x[0, t, 1, 5] = bad
        else:
            x[0, t, 1] = bad
        got, final = delta.gated_delta_scan(*on_gpu(broken))
        got, final = got.cpu(), final.cpu()
        ref.close(got[:, :, :1], want[:, :, :1], dtype, what="the other head")
        ref.close(final[:, :1], state[:, :1], dtype, what="the other head's state")
        if t:
            ref.close(got[:, :t], want[:, :t], dtype, what="earlier tokens")
        if what == "queries":
            assert not torch.isfinite(got[0, t, 1]).any()
            if t < 149:
                ref.close(got[:, t + 1:], want[:, t + 1:], dtype, what="later tokens")
            ref.close(final, state, dtype, what="final")
            continue
        if what == "values":
            others = [c for c in range(40) if c != 5]
            ref.close(got[..., others], want[..., others], dtype, what="other columns")
            ref.close(final[..., others], state[..., others], dtype, what="other columns of the state")
            got, final = got[..., 5:6], final[..., 5:6]
        assert not torch.isfinite(got[0, t:, 1]).any()
        assert not torch.isfinite(final[0, 1]).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_gradients_beside_padding_that_is_not_finite(dtype):
    """Values that are NaN behind the end of each sequence of a batch, where no gradient comes from."""
    from accelerated_scan import delta

    T, ends = 150, (81, 130)
    data = ref.inputs(2, T, 1, 2, 64, 40, dtype, seed=32)
    d_out = torch.randn(2, T, 2, 40, generator=torch.Generator().manual_seed(33)).to(dtype)
    for b, end in enumerate(ends):
        d_out[b, end:] = 0
    exact = as_exact(data, grad=True)
    want = torch.autograd.grad(ref.delta_scan(*exact)[0], exact, d_out.double())
    for b, end in enumerate(ends):
        data[2][b, end:] = float("nan")
    leaves = on_gpu(data, grad=True)
    got = torch.autograd.grad(delta.gated_delta_scan(*leaves)[0], leaves, d_out.to(DEVICE))
    for name, a, b in zip(NAMES, got, want):
        for n, end in enumerate(ends):
            rows = slice(None) if name == "initial" else slice(0, end)
            ref.close(a[n][rows], b[n][rows], dtype, backward=True, what=name)


@pytest.mark.parametrize("packed", [False, True], ids=["one", "packed"])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_many_blocks(dtype, packed):
    """Long enough that every block of a chain is asked for ahead by another one; four heads to a key head."""
    from accelerated_scan import delta

    T, ends = 64 * 11 + 17, [0, 64 * 9 + 1, 64 * 11 + 17]
    data = ref.inputs(1, T, 1, 4, 128, 32, dtype, seed=34, sequences=2 if packed else None)
    exact = as_exact(data, grad=True)
    d_out = torch.randn(1, T, 4, 32, generator=torch.Generator().manual_seed(35)).to(dtype)
    if packed:
        parts = [ref.delta_scan(*(x[:, a:b] for x in exact[:5]), exact[5][n:n + 1]) for n, (a, b) in enumerate(zip(ends, ends[1:]))]
        out, final = (torch.cat(x, d) for x, d in zip(zip(*parts), (1, 0)))
    else:
        out, final = ref.delta_scan(*exact)
    d_final = torch.randn(final.shape, generator=torch.Generator().manual_seed(36))
    want = torch.autograd.grad([out, final], exact, [d_out.double(), d_final.double()])
    leaves = on_gpu(data, grad=True)
    offsets = torch.tensor(ends, dtype=torch.int32, device=DEVICE) if packed else None
    results = delta.gated_delta_scan(*leaves, offsets=offsets)
    ref.close(results[0], out, dtype, what="out")
    ref.close(results[1], final, dtype, what="final")
    for name, a, b in zip(NAMES, torch.autograd.grad(results, leaves, on_gpu([d_out, d_final])), want):
        ref.close(a, b, dtype, backward=True, what=name)


def test_gradients_that_are_pieces_of_larger_tensors():
    from accelerated_scan import delta, norm

    data = on_gpu(ref.inputs(1, 70, 1, 2, 16, 16, torch.bfloat16, seed=37), grad=True)
    weight = torch.ones(16, device=DEVICE, dtype=torch.bfloat16, requires_grad=True)
    out, final = delta.gated_delta_scan(*data)
    gated = norm.gated_norm(out, data[2], weight)
    gen = torch.Generator(DEVICE).manual_seed(38)
    pieces = [torch.randn(t.numel() + 1, generator=gen, device=DEVICE).to(t.dtype) for t in (out, final, gated)]
    odd = [p[1:].view(t.shape) for p, t in zip(pieces, (out, final, gated))]
    assert all(t.data_ptr() % 16 for t in odd)
    inputs = [*data, weight]
    got = torch.autograd.grad([out, final, gated], inputs, odd, retain_graph=True)
    want = torch.autograd.grad([out, final, gated], inputs, [t.clone() for t in odd])
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    from accelerated_scan import delta, norm

    data = on_gpu(ref.inputs(1, 70, 1, 2, 16, 16, torch.float32, seed=39), grad=True)
    weight = torch.ones(16, device=DEVICE, requires_grad=True)
    out, _ = delta.gated_delta_scan(*data)
    for result, leaf in ((out, data[0]), (norm.gated_norm(data[2], data[2], weight), weight)):
        (first,) = torch.autograd.grad(result.square().sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            first.sum().backward()


def test_step_marks_its_states_as_changed():
    from accelerated_scan import delta

    q, k, v, g, b, states = on_gpu(ref.inputs(2, 1, 1, 2, 16, 16, torch.float32, seed=40))
    factor = torch.ones((), device=DEVICE, requires_grad=True)
    kept = factor * states  # keeps the states for its gradient
    with torch.no_grad():
        delta.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], b[:, 0], states)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.sum().backward()
    with torch.inference_mode():
        held = states.clone()
        out = delta.gated_delta_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], b[:, 0], held)
        assert torch.isfinite(out).all()


def test_offsets_that_do_not_ascend():
    """Unspecified values, and no access outside: what follows is right."""
    from accelerated_scan import delta

    data = on_gpu(ref.inputs(1, 300, 1, 2, 32, 32, torch.bfloat16, seed=41, sequences=5), grad=True)
    good = torch.tensor([0, 40, 40, 150, 299, 300], device=DEVICE)
    want = delta.gated_delta_scan(*data, offsets=good)
    for table in ([130, 10, 200, 70, 300, 0], [-5, 600, -1, 64, 128, 1 << 40], [300, 200, 100, 50, 20, 0]):
        out, final = delta.gated_delta_scan(*data, offsets=torch.tensor(table, device=DEVICE))
        torch.autograd.grad([out, final], data, [torch.ones_like(out), torch.ones_like(final)])
    got = delta.gated_delta_scan(*data, offsets=good)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tensors_beyond_two_to_the_31():
    """The last tokens of a sequence whose values have more elements than 32 bits count, and a slot behind as many
    state elements."""
    from accelerated_scan import delta

    heads, dv, T, cut = 32, 128, (1 << 19) + 200, (1 << 19) - 64 * 3
    gen = torch.Generator(DEVICE).manual_seed(42)
    new = lambda *s: torch.randn(s, generator=gen, device=DEVICE, dtype=torch.bfloat16)  # noqa: E731
    q, k = (torch.nn.functional.normalize(new(1, T, 1, 8), dim=-1) for _ in range(2))
    v = new(1, T, heads, dv)
    g, b = -new(1, T, heads).abs(), new(1, T, heads).sigmoid()
    out, final = delta.gated_delta_scan(q, k, v, g, b)
    head, state = delta.gated_delta_scan(*(t[:, :cut].contiguous() for t in (q, k, v, g, b)))
    tail, last = delta.gated_delta_scan(*(t[:, cut:].contiguous() for t in (q, k, v, g, b)), state)
    assert torch.equal(out[:, :cut], head) and torch.equal(out[:, cut:], tail) and torch.equal(final, last)
    del head, tail, out
    part = [t[:, cut:].contiguous().requires_grad_() for t in (q, k, v, g, b)]
    out, _ = delta.gated_delta_scan(*part, state)
    want = torch.autograd.grad(out, part, torch.ones_like(out))
    whole = [t.requires_grad_() for t in (q, k, v, g, b)]
    out, _ = delta.gated_delta_scan(*whole)
    got = torch.autograd.grad(out, whole, torch.ones_like(out))
    for a, w in zip(got, want):
        assert torch.equal(a[:, cut:], w)
    del got, out, whole, v
    states = torch.zeros(4100, 32, 128, 128, device=DEVICE)
    token = [new(2, 1, 128), new(2, 1, 128), new(2, 32, 128), -new(2, 32).abs(), new(2, 32).sigmoid()]
    small = states[:2].clone()
    out = delta.gated_delta_step(*token, states, slots=torch.tensor([4099, 0], device=DEVICE))
    assert torch.equal(out, delta.gated_delta_step(*token, small))
    assert torch.equal(states[4099], small[0]) and torch.equal(states[0], small[1]) and not states[1:4099].any()


def test_captured_training_step():
    from accelerated_scan import delta, norm

    data = on_gpu(ref.inputs(2, 150, 1, 2, 64, 64, torch.bfloat16, seed=43), grad=True)
    weight = torch.ones(64, device=DEVICE, dtype=torch.bfloat16, requires_grad=True)
    d_out = torch.randn(2, 150, 2, 64, generator=torch.Generator().manual_seed(44)).to(DEVICE, torch.bfloat16)
    inputs = [*data, weight]

    def gradients():
        out, _ = delta.gated_delta_scan(*data)
        return torch.autograd.grad(norm.gated_norm(out, data[2], weight), inputs, d_out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = gradients()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gradients()
    for turn in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        gradients()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tokens", [1, 2, 3, 70])
def test_gate_gradients_without_a_state(tokens, dtype):
    """A first token's gate scales nothing, and closed gates leave little: no rest of terms that cancel."""
    from accelerated_scan import delta

    data = ref.inputs(2, tokens, 1, 2, 64, 48, dtype, seed=50 + tokens, gates=torch.float32, decay=30.0 if tokens < 70 else 6.0)[:5]
    exact = as_exact(data, grad=True)
    out, final = ref.delta_scan(*exact)
    gen = torch.Generator().manual_seed(51)
    d_out, d_final = torch.randn(out.shape, generator=gen).to(dtype), torch.randn(final.shape, generator=gen)
    want = torch.autograd.grad([out, final], exact, [d_out.double(), d_final.double()])
    leaves = on_gpu(data, grad=True)
    got = torch.autograd.grad(delta.gated_delta_scan(*leaves), leaves, on_gpu([d_out, d_final]))
    assert not got[3][:, 0].any()
    for name, a, b in zip(NAMES, got, want):
        ref.close(a, b, dtype, backward=True, what=name)


def test_forward_mode_is_refused_and_leaves_the_rest_alone():
    """Tangents of inputs and of incoming gradients; calls without one inside a dual level go on as they do outside."""
    from torch.autograd import forward_ad

    from accelerated_scan import delta, norm

    data = on_gpu(ref.inputs(1, 70, 1, 2, 16, 16, torch.float32, seed=41))
    weight = torch.ones(16, device=DEVICE)
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    want = delta.gated_delta_scan(*data)
    with forward_ad.dual_level():
        assert all(torch.equal(a, b) for a, b in zip(delta.gated_delta_scan(*data), want))
        for i in range(6):
            some = [dual(t) if i == j else t for j, t in enumerate(data)]
            with pytest.raises(NotImplementedError):
                delta.gated_delta_scan(*some)
        with pytest.raises(NotImplementedError):
            norm.gated_norm(dual(data[2]), data[2], weight)
        leaves = [t.clone().requires_grad_() for t in data]
        out, final = delta.gated_delta_scan(*leaves)
        for d in ((dual(want[0]), want[1]), (want[0], dual(want[1]))):
            with pytest.raises(NotImplementedError):
                torch.autograd.grad([out, final], leaves, d, retain_graph=True)
        normed = norm.gated_norm(leaves[2], data[2], weight)
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(normed, leaves[2], dual(data[2]), retain_graph=True)
        torch.autograd.grad([out, final], leaves, want)
        token, states = [t[:, 0].contiguous() for t in data[:5]], data[5].clone()
        for step in (delta.gated_delta_step, lambda *a: torch.ops.accelerated_scan.delta_step(*a, None, 0.25)):
            with pytest.raises(NotImplementedError):
                step(*token[:4], dual(token[4]), states)
            assert torch.equal(states, data[5])
        first = delta.gated_delta_step(*token, states)
        assert torch.equal(first, torch.ops.accelerated_scan.delta_step(*token, data[5], None, 0.25)) and torch.equal(states, data[5])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(4, 50, 2, 2, 64, 64), (1, 700, 2, 2, 64, 64), (1, 500, 1, 2, 128, 128), (2, 90, 1, 3, 40, 72)], ids=str)
def test_results_in_32_bits(shape, dtype):
    """States and their gradients, and the gradients of gates in 32 bits, are as exact from 16-bit tensors as from others."""
    from accelerated_scan import delta

    data = ref.inputs(*shape, dtype, seed=42, gates=torch.float32, decay=0.2)
    exact, leaves = as_exact(data, grad=True), on_gpu(data, grad=True)
    results, got = ref.delta_scan(*exact), delta.gated_delta_scan(*leaves)
    ref.close_in_32_bits(got[1], results[1], what="final")
    gen = torch.Generator().manual_seed(43)
    d_out, d_final = torch.randn(got[0].shape, generator=gen).to(dtype), torch.randn(got[1].shape, generator=gen)
    want = torch.autograd.grad(results, exact[3:], [d_out.double(), d_final.double()])
    for name, a, b in zip(NAMES[3:], torch.autograd.grad(got, leaves[3:], on_gpu([d_out, d_final])), want):
        ref.close_in_32_bits(a, b, backward=True, what=name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_states_after_many_tokens(dtype):
    from accelerated_scan import delta

    data = ref.inputs(1, 4000, 1, 1, 128, 32, dtype, seed=44, gates=torch.float32, decay=0.02)
    with torch.no_grad():
        _, want = ref.delta_scan(*as_exact(data))
        _, got = delta.gated_delta_scan(*on_gpu(data))
    ref.close_in_32_bits(got, want, what="final")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("tokens, key_dim", [(64, 64), (640, 128)])
def test_equal_keys_of_16_bits(tokens, key_dim, dtype):
    """The matrix to invert at its worst: what a token adds to the state is a small difference of large terms, so that
    fewer bits in them would show at once.  The state is held to the bound of 32-bit calls."""
    from accelerated_scan import delta

    data = ref.inputs(1, tokens, 1, 2, key_dim, 64, dtype, seed=45, gates=torch.float32)
    data[1][:] = data[1][:, :1]
    data[3].zero_()
    data[4].fill_(0.99)
    want, final = ref.delta_scan(*as_exact(data))
    got, state = delta.gated_delta_scan(*on_gpu(data))
    ref.close(got, want, dtype)
    ref.close(state, final, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_packed_rows_without_a_sequence(dtype):
    """The C entry points by themselves: all rows are outside of the sequences, outputs and gradients are zero."""
    from accelerated_scan import _abi

    for rows in (1, 70, 5000):
        q, k, v, g, b, _ = on_gpu(ref.inputs(1, rows, 1, 3, 40, 24, dtype, seed=46))
        offsets = torch.zeros(1, dtype=torch.int32, device=DEVICE)
        new = lambda t: torch.full_like(t, float("nan"))  # noqa: E731
        nothing = torch.empty(0, device=DEVICE)
        out, final = new(v), torch.empty(0, 3, 40, 24, device=DEVICE)
        _abi.delta_forward(q, k, v, g, b, None, offsets, 1.0, out, final)
        grads = [new(t) for t in (q, k, v, g, b)]
        _abi.delta_backward(q, k, v, g, b, nothing, nothing, offsets, 1.0, v, None, *grads, None)
        for t in (out, *grads):
            assert torch.equal(t, torch.zeros_like(t))


MANY = [(64, 4, 8, 128, 128), (40, 8, 16, 96, 200), (90, 2, 6, 40, 256), (128, 2, 4, 64, 128), (35, 2, 8, 128, 136)]  # as in test_step


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", MANY, ids=str)
def test_step_of_many_conversations(shape, dtype):
    """512 workgroups of 128 columns and more: the wide variants, with states that leave a part of the rows or columns over."""
    from accelerated_scan import delta

    B, key_heads, heads, dk, dv = shape
    assert B * heads * -(-dv // 128) >= 512
    data = ref.inputs(B, 1, key_heads, heads, dk, dv, dtype, seed=47)
    want, final = ref.delta_scan(*as_exact(data))
    *inputs, state = on_gpu(data)
    token = [t[:, 0].contiguous() for t in inputs]
    got = delta.gated_delta_step(*token, state)
    ref.close(got, want[:, 0], dtype)
    ref.close(state, final, torch.float32)
    # in the slots of a pool, in another order: the same states
    gen = torch.Generator().manual_seed(48)
    slots = torch.randperm(B + 5, generator=gen)[:B].to(DEVICE)
    pool = torch.full((B + 5, heads, dk, dv), 7.0, device=DEVICE)
    pool[slots] = data[5].to(DEVICE)
    assert torch.equal(delta.gated_delta_step(*token, pool, slots=slots), got) and torch.equal(pool[slots], state)
    rest = torch.ones(B + 5, dtype=torch.bool, device=DEVICE)
    rest[slots] = False
    assert (pool[rest] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", MANY[:3], ids=str)
def test_slots_of_many_conversations(shape, dtype):
    """Rows that share a slot, and rows without a state, among many."""
    from accelerated_scan import delta

    B, key_heads, heads, dk, dv = shape
    count = B // 3
    slots = torch.randint(-2, count + 2, (B,), generator=torch.Generator().manual_seed(49))
    data = ref.inputs(B, 1, key_heads, heads, dk, dv, dtype, seed=50, sequences=count)
    q, k, v, g, b, pool = as_exact(data)
    want, want_pool = torch.zeros_like(v[:, 0]), pool.clone()
    for row, slot in enumerate(slots.tolist()):
        if 0 <= slot < count:
            o, want_pool[slot:slot + 1] = ref.delta_scan(*(t[row:row + 1] for t in (q, k, v, g, b)), want_pool[slot:slot + 1].clone())
            want[row] = o[0, 0]
    *inputs, states = on_gpu(data)
    got = delta.gated_delta_step(*[t[:, 0].contiguous() for t in inputs], states, slots=slots.to(torch.int32).to(DEVICE))
    ref.close(got, want, dtype)
    ref.close(states, want_pool, torch.float32)
    for row, slot in enumerate(slots.tolist()):
        if not 0 <= slot < count:
            assert not got[row].any()
