"""Gated norm on the GPU against float64.

A value goes through at most a dozen fp32 operations, each off by 2^-24 of its result, an exponential of 2 steps
among them, and the sums over a row of non-negative squares (error below 2^-24 times the depth of the tree and the 32
elements a lane adds: 2^-18 at 8192): together below 2^-17, and one rounding u to the output's type.  Gradients
subtract a row's mean: their error is relative to the row's largest term, and a row's product sum e.h can cancel, so
it counts against the size of its terms, which a row's largest element bounds up to the 8 of random signs."""

import pytest
import torch

import delta_reference as ref

pytestmark = pytest.mark.gpu

DEVICE = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (3, 8), (70, 64), (33, 96), (5, 128), (17, 130), (9, 257), (4, 512), (3, 1000), (2, 2048), (2, 2049),
          (3, 5001), (2, 8192), (2, 8200), (1, 20000), (2, 9, 4, 128), (5000, 64)]


def make(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x, z, d = (torch.randn(*shape, generator=gen).to(dtype) for _ in range(3))
    return x, z, (1 + 0.2 * torch.randn(shape[-1], generator=gen)).to(dtype), d


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_and_gradients(shape, dtype):
    from accelerated_scan import norm

    x, z, w, d = make(shape, dtype, 1)
    exact = [t.double().requires_grad_() for t in (x, z, w)]
    want = ref.gated_norm(*exact)
    leaves = [t.to(DEVICE).requires_grad_() for t in (x, z, w)]
    got = norm.gated_norm(*leaves)
    assert got.dtype == dtype and got.shape == want.shape
    u = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * u * 2 + 2.0 ** -40  # below the type's normal numbers
    off = (got.detach().cpu().double() - want.detach()).abs()
    assert (off <= (u + 2.0 ** -17) * want.detach().abs() + tiny).all(), off.max()
    want_grads = torch.autograd.grad(want, exact, d.double())
    got_grads = torch.autograd.grad(got, leaves, d.to(DEVICE))
    for name, a, b in zip(("x", "gate"), got_grads, want_grads):
        a = a.cpu().double()
        most = b.abs().amax(-1, keepdim=True) if name == "x" else 0
        off = (a - b).abs() - (u + 2.0 ** -17) * b.abs() - 8 * 2.0 ** -17 * most
        if name == "gate":
            # s (1 + z (1 - s)) cancels near z = -1.28: its two terms are as large as s (1 + |z|), and so their
            # rounding errors count against dy w h s (1 + |z|), h = x / r
            h = x.double() / (x.double().square().mean(-1, keepdim=True) + 1e-6).sqrt()
            off = off - 2.0 ** -17 * (d.double() * w.double() * h * torch.sigmoid(z.double()) * (1 + z.double().abs())).abs()
        if name == "x" and shape[-1] == 1:  # a row of one: the two terms cancel but for eps
            off = (a - b).abs() - 2.0 ** -17 * (d.double() * w.double() * z.double() / x.double()).abs()
        assert (off <= tiny).all(), (name, off.max())
    # the weight's gradient: a sum over rows, in fp32 with at most rows / 16 terms in one chain
    terms = (d.double() * want.detach() / w.double()).abs().reshape(-1, shape[-1]).sum(0)
    off = (got_grads[2].cpu().double() - want_grads[2]).abs()
    assert (off <= u * want_grads[2].abs() + 2.0 ** -15 * terms + tiny).all(), off.max()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_that_start_anywhere(dtype):
    """Tensors whose storage does not start on 16 bytes take the element-wise variant: same values."""
    from accelerated_scan import norm

    x, z, w, d = make((6, 128), dtype, 2)
    shifted = []
    for t in (x, z, w, d):
        room = torch.empty(t.numel() + 1, dtype=dtype, device=DEVICE)
        view = room[1:].view(t.shape)
        view.copy_(t)
        shifted.append(view)
    want = ref.gated_norm(x.double(), z.double(), w.double())
    u = torch.finfo(dtype).eps / 2 + 2.0 ** -17
    sx, sz, sw = (t.requires_grad_() for t in shifted[:3])
    got = norm.gated_norm(sx, sz, sw)
    assert ((got.detach().cpu().double() - want).abs() <= u * want.abs() + 2.0 ** -24).all()
    plain = [t.to(DEVICE).requires_grad_() for t in (x, z, w)]
    a = torch.autograd.grad(got, (sx, sz, sw), shifted[3])
    b = torch.autograd.grad(norm.gated_norm(*plain), plain, d.to(DEVICE))
    for g, h in zip(a, b):  # sums in another order
        torch.testing.assert_close(g, h, rtol=4 * torch.finfo(dtype).eps, atol=2.0 ** -14)


def test_special_rows_and_gates():
    """Rows of zeros, gates far out, a NaN that stays in its row."""
    from accelerated_scan import norm

    x, z, w, _ = make((5, 64), torch.float32, 3)
    x[0] = 0
    z[1, :4] = torch.tensor([-200.0, 200.0, -88.0, 0.0])
    x[2, 5] = float("nan")
    x[3] *= 1e-18  # the squares vanish beside eps
    got = norm.gated_norm(*(t.to(DEVICE) for t in (x, z, w))).cpu().double()
    want = ref.gated_norm(x.double(), z.double(), w.double())
    assert torch.equal(got.isnan(), want.isnan()) and got.isnan().all(-1).tolist() == [False, False, True, False, False]
    keep = [0, 1, 3, 4]
    assert ((got - want)[keep].abs() <= 2.0 ** -17 * want[keep].abs() + 2.0 ** -100).all()


def test_gradient_against_differences():
    """Central differences along a direction: a step of 2^-6 leaves 2^-12 of the third derivative and 2^-17 / 2^-5 of the
    operator's own error, 2^-9 of the slope's scale in all."""
    from accelerated_scan import norm

    x, z, w, d = (t.to(DEVICE) for t in make((7, 200), torch.float32, 4))
    leaves = [t.requires_grad_() for t in (x, z, w)]
    grads = torch.autograd.grad(norm.gated_norm(*leaves), leaves, d)
    gen = torch.Generator(device=DEVICE).manual_seed(5)
    for i, g in enumerate(grads):
        v = torch.randn(leaves[i].shape, generator=gen, device=DEVICE)
        v *= 1 / v.norm()
        h, ends = 2.0 ** -6, []
        for s in (1, -1):
            moved = [t.detach() + (s * h * v if j == i else 0) for j, t in enumerate(leaves)]
            ends.append((norm.gated_norm(*moved).double() * d).sum().item())
        assert abs((ends[0] - ends[1]) / (2 * h) - (g.double() * v).sum().item()) <= 2.0 ** -9 * g.norm().item()


def test_captured_backward_and_empty_rows():
    from accelerated_scan import norm

    x, z, w, d = (t.to(DEVICE) for t in make((500, 96), torch.bfloat16, 6))
    eager = None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [t.clone().requires_grad_() for t in (x, z, w)]
        eager = [t.clone() for t in torch.autograd.grad(norm.gated_norm(*leaves), leaves, d)]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    leaves = [t.clone().requires_grad_() for t in (x, z, w)]
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(norm.gated_norm(*leaves), leaves, d)
    for _ in range(3):
        for g in grads:
            g.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, eager))
    empty = torch.zeros(0, 8, device=DEVICE, requires_grad=True)
    weight = torch.ones(8, device=DEVICE, requires_grad=True)
    out = norm.gated_norm(empty, empty, weight)
    assert out.shape == (0, 8)
    assert not torch.autograd.grad(out.sum(), weight)[0].any()


def test_rows_wider_than_a_launch_has_threads_for():
    """The weight's gradient of 2^26 columns and more.  Elements of +-1 make the row's sum of squares exact; the mean over the
    row that dx subtracts is a sum of 2^18 terms to a lane, each rounded to 2^-24 of it: 2^-6 of the terms' mean size."""
    from accelerated_scan import norm

    width = 2 ** 26 + 24
    gen = torch.Generator(device=DEVICE).manual_seed(7)
    x = torch.randn(1, width, generator=gen, device=DEVICE).sign().add(0.5).sign().to(torch.bfloat16)
    z, d = (torch.randn(1, width, generator=gen, device=DEVICE).to(torch.bfloat16) for _ in range(2))
    w = torch.ones(width, device=DEVICE, dtype=torch.bfloat16)
    leaves = [t.requires_grad_() for t in (x, z, w)]
    dx, _, dw = torch.autograd.grad(norm.gated_norm(*leaves), leaves, d)
    with torch.no_grad():
        inverse = (1 + 1e-6) ** -0.5
        e = d.double() * z.double() * torch.sigmoid(z.double())
        want = (e * x.double()).squeeze(0) * inverse
        u = 2.0 ** -8
        assert ((dw.double() - want).abs() <= (u + 2.0 ** -17) * want.abs() + 2.0 ** -40).all()
        mean = want.mean()
        off = (dx.double() - (e - x.double() * inverse * mean) * inverse).abs()
        assert (off <= (u + 2.0 ** -17) * e.abs() + 2 * 2.0 ** -6 * want.abs().mean()).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(33000, 96), (40001, 64), (8300, 257), (8203, 512), (2100, 1000), (2500, 1025), (2049, 2052),
                                   (2100, 8200), (2050, 5001)], ids=str)
def test_more_rows_than_workgroups(shape, dtype):
    """The backward kernel's workgroups, 2048 at most, take several rows (of 16, 64 or 256 lanes) after one another, in every
    variant: the bounds are those of test_norm_and_gradients."""
    from accelerated_scan import norm

    x, z, w, d = (t.to(DEVICE) for t in make(shape, dtype, 8))
    leaves = [t.clone().requires_grad_() for t in (x, z, w)]
    got = norm.gated_norm(*leaves)
    dx, dz, dw = torch.autograd.grad(got, leaves, d)
    u, e17 = torch.finfo(dtype).eps / 2, 2.0 ** -17
    tiny = torch.finfo(dtype).smallest_normal * u * 2 + 2.0 ** -40
    x, z, w, d = (t.double() for t in (x, z, w, d))
    inverse = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    s, h = torch.sigmoid(z), x * inverse
    want = h * w * z * s
    assert ((got.double() - want).abs() <= (u + e17) * want.abs() + tiny).all()
    e = d * w * z * s
    want_x = (e - h * (e * h).mean(-1, keepdim=True)) * inverse
    assert ((dx.double() - want_x).abs() <= (u + e17) * want_x.abs() + 8 * e17 * want_x.abs().amax(-1, keepdim=True) + tiny).all()
    want_z = d * w * h * s * (1 + z * (1 - s))
    assert ((dz.double() - want_z).abs() <= (u + e17) * want_z.abs() + e17 * (d * w * h * s * (1 + z.abs())).abs() + tiny).all()
    terms = d * h * z * s
    # in fp32: rows / 2048 at most in a workgroup's chain, 32 shares in a thread's, then a tree
    assert ((dw.double() - terms.sum(0)).abs() <= u * terms.sum(0).abs() + 2.0 ** -15 * terms.abs().sum(0) + tiny).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_more_rows_than_workgroups_start_anywhere(dtype):
    """The same rows in tensors that do not start on 16 bytes, which take the element-wise variant."""
    from accelerated_scan import norm

    for shape in ((33000, 96), (2100, 1000), (2050, 5000)):
        plain = [t.to(DEVICE) for t in make(shape, dtype, 9)]
        odd = []
        for t in plain:
            odd.append(torch.empty(t.numel() + 1, dtype=dtype, device=DEVICE)[1:].view(t.shape).copy_(t))
        assert odd[0].data_ptr() % 16
        results = []
        for x, z, w, d in (plain, odd):
            leaves = [t.detach().requires_grad_() for t in (x, z, w)]
            out = norm.gated_norm(*leaves)
            results.append([out.detach(), *torch.autograd.grad(out, leaves, d)])
        for a, b in zip(*results):  # sums in another order: 2^-15 of a sum's terms, whose size is at most its largest times 8
            most = b.float().abs().max().item()
            torch.testing.assert_close(a, b, rtol=2 * torch.finfo(dtype).eps, atol=8 * 2.0 ** -15 * most)


@pytest.mark.parametrize("rows, width", [(2 ** 24 + 17, 8), (2 ** 22 + 3, 130), (2 ** 20 + 5, 520)])
def test_more_rows_than_forward_workgroups(rows, width):
    """The forward kernel's workgroups, 2^20 at most, take several rows after one another."""
    from accelerated_scan import norm

    gen = torch.Generator(device=DEVICE).manual_seed(10)
    x, z = (torch.randn(rows, width, generator=gen, device=DEVICE, dtype=torch.bfloat16) for _ in range(2))
    w = torch.randn(width, generator=gen, device=DEVICE, dtype=torch.bfloat16)
    got = norm.gated_norm(x, z, w)
    first = 2 ** 20 * (16 if width <= 128 else 4 if width <= 512 else 1)  # the second turn's first row
    for some in (slice(0, 50), slice(first - 20, rows)):
        want = ref.gated_norm(x[some].double(), z[some].double(), w.double())
        assert ((got[some].double() - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * want.abs() + 2.0 ** -40).all()
