"""CPU tests of the gated delta rule and the gated norm: what the C entry points refuse by return code before
they touch the GPU, what the Python operators refuse, and the definition that the GPU tests use against a plain
double loop.  No kernel is launched here."""

import ctypes

import pytest
import torch

import delta_reference as ref
from accelerated_scan import _abi, delta, norm

OK, NULL, SHAPE, DTYPE, MISALIGNED, OVERLAP, HEADS, WORKSPACE = 0, 1, 2, 3, 4, 7, 9, 10


@pytest.fixture(scope="module")
def room():
    buf = ctypes.create_string_buffer(1 << 20)
    base = ctypes.addressof(buf)
    yield base + (-base % 64)
    del buf


def forward(p, **change):
    """Arguments of a valid call on 2 x 70 tokens with buffers 64 KiB apart, with some of them changed."""
    a = dict(q=p, k=p + 0x10000, v=p + 0x20000, log_gates=p + 0x30000, beta=p + 0x31000, initial=None, offsets=None,
             out=p + 0x40000, final=None, states=None, updates=None, rows=140, sequences=2, heads=2, key_heads=1, dk=16,
             dv=16, scale=1.0, dtype=0, flags=0, workspace=p + 0x80000, bytes=1 << 19, stream=None)
    a.update(change)
    return _abi.load().ascan_delta_forward(*a.values())


def backward(p, **change):
    a = dict(q=p, k=p + 0x4000, v=p + 0x8000, log_gates=p + 0x10000, beta=p + 0x11000, states=p + 0x14000,
             updates=p + 0x20000, offsets=None, d_out=p + 0x28000, d_final=None, d_q=p + 0x30000, d_k=p + 0x34000,
             d_v=p + 0x38000, d_log_gates=p + 0x40000, d_beta=p + 0x41000, d_initial=None, rows=140, sequences=2, heads=2,
             key_heads=1, dk=16, dv=16, scale=1.0, dtype=0, flags=0, workspace=p + 0x60000, bytes=0xa0000, stream=None)
    a.update(change)
    return _abi.load().ascan_delta_backward(*a.values())


def step(p, **change):
    a = dict(q=p, k=p + 0x1000, v=p + 0x2000, log_gates=p + 0x3000, beta=p + 0x3800, states=p + 0x10000, slots=None,
             out=p + 0x4000, batch=3, count=3, heads=2, key_heads=1, dk=16, dv=16, scale=1.0, dtype=0, flags=0, stream=None)
    a.update(change)
    return _abi.load().ascan_delta_step(*a.values())


@pytest.mark.parametrize("call", [forward, backward, step])
def test_sizes_and_types_are_refused(room, call):
    assert call(room, dtype=3) == DTYPE and call(room, dtype=-1) == DTYPE
    for bad in (dict(heads=0), dict(key_heads=0), dict(heads=3, key_heads=2), dict(dk=0), dict(dk=12), dict(dk=136),
                dict(dv=4), dict(dv=4104), dict(dv=-8), dict(heads=-2)):
        assert call(room, **bad) == HEADS, bad


@pytest.mark.parametrize("call", [forward, backward])
def test_scan_arguments_are_refused(room, call):
    for bad in (dict(rows=-1), dict(sequences=-1), dict(rows=141), dict(sequences=0), dict(rows=1 << 41, sequences=1 << 10)):
        assert call(room, **bad) == SHAPE, bad
    for name in ("q", "k", "v", "log_gates", "beta", "workspace"):
        assert call(room, **{name: None}) == NULL, name
    for name in ("q", "k", "v", "workspace"):
        assert call(room, **{name: room + 0x90008}) == MISALIGNED, name
    assert call(room, log_gates=room + 0x30002) == MISALIGNED
    assert call(room, offsets=room + 0x90002) == MISALIGNED
    assert call(room, offsets=room + 0x90004, flags=2) == MISALIGNED
    assert call(room, bytes=100) == WORKSPACE
    # nothing to do
    assert call(room, rows=0, sequences=0, q=None, k=None, v=None) == OK
    assert call(room, rows=0, sequences=3, q=None, k=None, v=None) == OK


def test_scan_buffers_that_overlap_are_refused(room):
    assert forward(room, out=room) == OVERLAP
    assert forward(room, final=room + 0x20000) == OVERLAP
    assert forward(room, states=room + 0x40000) == OVERLAP
    assert forward(room, workspace=room + 0x30000) == OVERLAP
    assert forward(room, initial=room + 0x90000, final=room + 0x90000) == OVERLAP
    assert forward(room, out=None) == NULL
    assert forward(room, final=room + 0x90004) == MISALIGNED
    assert backward(room, d_q=room) == OVERLAP
    assert backward(room, d_k=room + 0x30000) == OVERLAP
    assert backward(room, d_beta=room + 0x40000) == OVERLAP
    assert backward(room, d_log_gates=None) == NULL
    assert backward(room, states=None) == NULL
    assert backward(room, d_out=room + 0x28004) == MISALIGNED


def test_step_arguments_are_refused(room):
    for bad in (dict(batch=-1), dict(count=-1), dict(batch=4), dict(batch=1 << 31, count=1 << 31)):
        assert step(room, **bad) == SHAPE, bad
    for name in ("q", "k", "v", "log_gates", "beta", "states", "out"):
        assert step(room, **{name: None}) == NULL, name
    for name in ("q", "k", "v", "states", "out"):
        assert step(room, **{name: room + 0x20008}) == MISALIGNED, name
    assert step(room, slots=room + 0x20002) == MISALIGNED
    assert step(room, out=room) == OVERLAP
    assert step(room, states=room + 0x3000) == OVERLAP
    assert step(room, batch=0, q=None) == OK


def test_norm_arguments_are_refused(room):
    f, b = _abi.load().ascan_gated_norm, _abi.load().ascan_gated_norm_backward
    p = [room + i * 0x10000 for i in range(8)]
    assert f(*p[:4], 4, 8, 1e-6, 3, None) == DTYPE
    assert f(*p[:4], -4, 8, 1e-6, 0, None) == SHAPE
    assert f(*p[:4], 1 << 50, 1 << 20, 1e-6, 0, None) == SHAPE
    assert f(None, *p[1:4], 4, 8, 1e-6, 0, None) == NULL
    assert f(p[0] + 2, *p[1:4], 4, 8, 1e-6, 0, None) == MISALIGNED
    assert f(p[0], p[1], p[2], p[0] + 64, 4, 8, 1e-6, 0, None) == OVERLAP
    assert f(*p[:4], 0, 8, 1e-6, 0, None) == OK and f(*p[:4], 8, 0, 1e-6, 0, None) == OK
    need = _abi.load().ascan_gated_norm_workspace_bytes(4, 8)
    assert need > 0 and _abi.load().ascan_gated_norm_workspace_bytes(0, 8) == 0
    assert b(*p[:7], 4, 8, 1e-6, 0, p[7], need - 1, None) == WORKSPACE
    assert b(*p[:7], 4, 8, 1e-6, 0, None, need, None) == NULL
    assert b(*p[:4], p[0], p[5], p[6], 4, 8, 1e-6, 0, p[7], need, None) == OVERLAP
    assert b(*p[:4], p[4], p[4] + 64, p[6], 4, 8, 1e-6, 0, p[7], need, None) == OVERLAP
    assert b(*p[:6], p[6] + 2, 4, 8, 1e-6, 0, p[7], need, None) == MISALIGNED


def test_status_texts():
    lib = _abi.load()
    texts = {lib.ascan_status_string(i).decode() for i in range(11)}
    assert len(texts) == 11 and "unknown status" not in texts


def test_table_sizes():
    blocks = _abi.load().ascan_delta_blocks
    assert blocks(140, 2, 0) == 4 and blocks(128, 2, 0) == 2 and blocks(0, 0, 0) == 0
    assert blocks(140, 2, 1) == 4 and blocks(64, 5, 1) == 6
    assert blocks(141, 2, 0) == -1 and blocks(-1, 2, 0) == -1
    # packed sequences: every one has room for its last, partial block, and no two share an entry
    gen = torch.Generator().manual_seed(1)
    for _ in range(50):
        lengths = torch.randint(0, 200, (7,), generator=gen).tolist()
        start, taken = 0, set()
        for n, length in enumerate(lengths):
            mine = {start // 64 + n + c for c in range(-(-length // 64))}
            assert not mine & taken and all(m < blocks(sum(lengths), 7, 1) for m in mine)
            taken |= mine
            start += length


def tensors(B=1, T=4, key_heads=1, heads=2, dk=16, dv=8, dtype=torch.float32):
    return list(ref.inputs(B, T, key_heads, heads, dk, dv, dtype))


@pytest.mark.parametrize("change, message", [
    (lambda t: t.__setitem__(0, t[0].double()), "unsupported tensor dtypes"),
    (lambda t: t.__setitem__(2, t[2].half()), "unsupported tensor dtypes"),
    (lambda t: t.__setitem__(3, t[3].half()), "unsupported tensor dtypes"),
    (lambda t: t.__setitem__(4, t[4].double()), "unsupported tensor dtypes"),
    (lambda t: t.__setitem__(0, t[0][0]), "shape"),
    (lambda t: t.__setitem__(1, t[1][:, :3]), "shape of queries"),
    (lambda t: t.__setitem__(3, t[3][:, :3]), "log_gates and beta of shape"),
    (lambda t: t.__setitem__(5, t[5][:, :1]), "expected initial of shape"),
    (lambda t: t.__setitem__(5, t[5].double()), "expected initial of shape"),
    (lambda t: None, "device tensor"),
])
def test_scan_refusals(change, message):
    t = tensors()
    change(t)
    with pytest.raises(RuntimeError, match=message):
        delta.gated_delta_scan(*t)


@pytest.mark.parametrize("sizes, message", [
    (dict(dk=12), "multiples of 8"), (dict(dk=136), "up to 128"), (dict(dv=4), "multiples of 8"),
    (dict(key_heads=2, heads=3), "key heads that divide"),
])
def test_sizes_the_kernels_do_not_take(sizes, message):
    with pytest.raises(RuntimeError, match=message):
        delta.gated_delta_scan(*tensors(**sizes))
    *t, states = tensors(B=2, T=1, **sizes)
    with pytest.raises(RuntimeError, match=message):
        delta.gated_delta_step(*[x[:, 0] for x in t], states)


def test_offsets_refusals():
    t = tensors()
    for bad in (torch.tensor([0.0, 4.0]), torch.tensor([[0, 4]]), torch.zeros(0, dtype=torch.int32)):
        with pytest.raises(RuntimeError, match="expected offsets"):
            delta.gated_delta_scan(*t[:5], offsets=bad)
    with pytest.raises(RuntimeError, match="batch of one"):
        delta.gated_delta_scan(*tensors(B=2)[:5], offsets=torch.tensor([0, 4]))
    with pytest.raises(RuntimeError, match="expected initial of shape"):
        delta.gated_delta_scan(*t, offsets=torch.tensor([0, 2, 4]))


def test_step_refusals():
    *t, states = tensors(B=3, T=1)
    t = [x[:, 0] for x in t]
    with pytest.raises(RuntimeError, match="device tensor"):
        delta.gated_delta_step(*t, states)
    with pytest.raises(RuntimeError, match="a state to each"):
        delta.gated_delta_step(*t, states[:2])
    with pytest.raises(RuntimeError, match="expected states of shape"):
        delta.gated_delta_step(*t, states.half())
    with pytest.raises(RuntimeError, match="expected slots"):
        delta.gated_delta_step(*t, states, slots=torch.tensor([0, 1]))
    with pytest.raises(RuntimeError, match="expected slots"):
        delta.gated_delta_step(*t, states, slots=torch.tensor([0.0, 1.0, 2.0]))
    with pytest.raises(RuntimeError, match="shape"):
        delta.gated_delta_step(t[0][0], *t[1:], states)


def test_norm_refusals():
    x, w = torch.randn(3, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="device tensor"):
        norm.gated_norm(x, x, w)
    with pytest.raises(RuntimeError, match="one shape"):
        norm.gated_norm(x, x[:2], w)
    with pytest.raises(RuntimeError, match="last axis"):
        norm.gated_norm(x, x, torch.ones(4))
    with pytest.raises(RuntimeError, match="unsupported tensor dtypes"):
        norm.gated_norm(x, x.half(), w)


def test_the_definition_itself():
    """One head, plain Python numbers, against the tests' reference."""
    q, k, v, g, b, s = (t.double() for t in tensors(T=5, heads=1, dk=8, dv=8))
    want, final = ref.delta_scan(q, k, v, g, b, s, scale=0.5)
    S = [[s[0, 0, i, j].item() for j in range(8)] for i in range(8)]
    for t in range(5):
        a, beta = g[0, t, 0].exp().item(), b[0, t, 0].item()
        S = [[a * x for x in row] for row in S]
        for j in range(8):
            held = sum(S[i][j] * k[0, t, 0, i].item() for i in range(8))
            for i in range(8):
                S[i][j] += beta * k[0, t, 0, i].item() * (v[0, t, 0, j].item() - held)
        for j in range(8):
            o = 0.5 * sum(S[i][j] * q[0, t, 0, i].item() for i in range(8))
            assert abs(o - want[0, t, 0, j].item()) < 1e-12
    assert all(abs(S[i][j] - final[0, 0, i, j].item()) < 1e-12 for i in range(8) for j in range(8))


def test_launches_beyond_the_hardware_are_refused(room):
    wide = dict(rows=0, sequences=65535, heads=64, key_heads=64, dk=128, dv=128)  # 33 million workgroups of 768 threads
    assert forward(room, **wide, final=room) == SHAPE and backward(room, **wide, d_initial=room) == SHAPE
    assert _abi.load().ascan_delta_workspace_bytes(0, 65535, 64, 64, 128, 128, 0, 0, 0) == 0
    many = dict(heads=1, key_heads=1, dk=8, dv=8)
    assert forward(room, rows=1 << 30, sequences=1, **many) == SHAPE  # 2^24 blocks
    assert step(room, batch=1 << 24, count=1 << 24, **many) == SHAPE
    assert step(room, count=1 << 62) == SHAPE


def test_forward_mode_tangents_are_refused():
    """A tangent would get lost, and a result without one reads as a derivative of zero."""
    from torch.autograd import forward_ad

    *t, states = tensors(B=3, T=1)
    token = [x[:, 0] for x in t]
    rows = [torch.randn(3, 8), torch.randn(3, 8), torch.ones(8)]
    ops = torch.ops.accelerated_scan
    calls = [(lambda *a: delta.gated_delta_scan(*a), [*t, states]),
             (lambda *a: ops.delta_forward(*a, None, 1.0, False), [*t, states]),
             (lambda *a: delta.gated_delta_step(*a), [*token, states]),
             (lambda *a: ops.delta_step(*a, None, 1.0), [*token, states]),
             (lambda *a: norm.gated_norm(*a), rows),
             (lambda *a: ops.gated_norm(*a, 1e-6), rows)]
    for call, args in calls:
        for i in range(len(args)):
            with forward_ad.dual_level():
                some = list(args)
                some[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                for grad in (True, False):
                    with pytest.raises(NotImplementedError, match="forward-mode"), torch.set_grad_enabled(grad):
                        call(*some)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="device tensor"):
            call(*args)  # no tangent: the next check's turn


def test_states_and_updates_come_together(room):
    """What a backward pass needs is both or none: the kernel that keeps one writes the other too."""
    kept = dict(states=room + 0x50000, updates=room + 0x58000)
    for name in kept:
        assert forward(room, **{name: kept[name]}) == NULL, name
    assert forward(room, **kept, out=room) == OVERLAP  # a pair gets past that check
    assert forward(room, states=room + 0x50000, rows=0, sequences=0) == OK


@pytest.mark.parametrize("call, outputs", [(forward, ["out"]), (backward, ["d_q", "d_k", "d_v", "d_log_gates", "d_beta"])])
def test_outputs_of_packed_rows_without_a_sequence_are_wanted(room, call, outputs):
    for name in outputs:
        assert call(room, sequences=0, offsets=room + 0xf0000, **{name: None}) == NULL, name
        assert call(room, sequences=0, offsets=room + 0xf0000, **{name: room + 0x40001}) == MISALIGNED, name


@pytest.mark.parametrize("call, outputs", [(forward, ["out"]), (backward, ["d_q", "d_v", "d_beta"])])
def test_overlaps_of_packed_rows_without_a_sequence(room, call, outputs):
    for name in outputs:
        assert call(room, sequences=0, offsets=room + 0xf0000, **{name: room}) == OVERLAP, name
