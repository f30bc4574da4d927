"""The norms before and after a block against their definitions in 64 bits: types, widths from one channel to the widest, strides, scales,
gates far out, rows of zeros, gradients by the formula and by differences."""
import pytest
import torch

from block_reference import gated_norm, residual_norm, within
from cute_triadic_gdn_b200 import _lib, gated_norm_call, residual_norm_call

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
PAIRS = [(BF16, BF16), (BF16, F32), (F16, F16), (F16, F32), (F32, F32)]
EPS = 1e-6


def randn(*shape, dtype=F32, seed=0):
    gen = torch.Generator().manual_seed(seed + sum(shape))
    return torch.randn(*shape, generator=gen).to(dtype).cuda()


def leaf(t):
    return t.detach().requires_grad_(True) if torch.is_tensor(t) else t


def check_residual(x, residual, weight, scale, dy, ds, eps=EPS):
    args = [leaf(t) for t in (x, residual, weight, scale)]
    y, stream = residual_norm_call(*args, eps=eps)
    assert y.dtype == x.dtype and stream.dtype == residual.dtype and y.is_contiguous() and stream.is_contiguous()
    names = [n for n, t in zip(("dx", "dresidual", "dweight", "dscale"), args) if torch.is_tensor(t)]
    outs, grads = [(o, d) for o, d in ((y, dy), (stream, ds)) if d is not None], None
    grads = torch.autograd.grad([o for o, _ in outs], [t for t in args if torch.is_tensor(t)], [d for _, d in outs], allow_unused=dy is None)
    ref = residual_norm(x, residual, weight, scale, eps, dy, ds)
    within(y, *ref["y"], "y")
    within(stream, *ref["stream"], "stream")
    for name, got in zip(names, grads):
        within(got, *ref[name], name)
    return y, stream, grads


def check_gated(x, gate, weight, residual, scale, activation, dout, eps=EPS):
    args = [leaf(t) for t in (x, gate, weight, residual, scale)]
    out = gated_norm_call(*args, activation=activation, eps=eps)
    assert out.dtype == (x if residual is None else residual).dtype and out.is_contiguous()
    names = [n for n, t in zip(("dx", "dgate", "dweight", "dresidual", "dscale"), args) if torch.is_tensor(t)]
    grads = torch.autograd.grad(out, [t for t in args if torch.is_tensor(t)], dout)
    ref = gated_norm(x, gate, weight, residual, scale, activation, eps, dout)
    within(out, *ref["out"], "out")
    for name, got in zip(names, grads):
        if name == "dresidual":
            assert torch.equal(got, dout)
        else:
            within(got, *ref[name], name)
    return out, grads


@pytest.mark.parametrize("x_type,r_type", PAIRS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 33), (1, 64), (300, 128), (7, 200), (5, 257), (2, 1024), (3, 1032), (2, 2001), (2, 8192), (1, 8200),
                                   (2, 16384), (1, 16383)])
def test_residual_norm_against_the_definition(shape, x_type, r_type):
    N = shape[-1]
    x, residual = randn(*shape, dtype=x_type), randn(*shape, dtype=r_type, seed=1)
    dy, ds = randn(*shape, dtype=x_type, seed=2), randn(*shape, dtype=r_type, seed=3)
    w, c = 1 + 0.2 * randn(N, seed=4), 0.5 + 0.2 * randn(N, seed=5)
    check_residual(x, residual, w.to(x_type), c.to(x_type), dy, ds)
    check_residual(x, residual, None, 0.25, dy, ds)
    check_residual(x, residual, w, None, dy, None)


@pytest.mark.parametrize("x_type,r_type", PAIRS)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 33), (2, 3, 4, 128), (300, 64), (7, 200), (5, 257), (2, 1024), (3, 1032), (2, 2001), (2, 8192),
                                   (1, 8200), (2, 16384), (1, 16383)])
def test_gated_norm_against_the_definition(shape, x_type, r_type):
    N = shape[-1]
    x, z, residual = randn(*shape, dtype=x_type), 3 * randn(*shape, seed=1), randn(*shape, dtype=r_type, seed=2)
    z, dout = z.to(x_type), randn(*shape, dtype=r_type, seed=3)
    w, c = 1 + 0.2 * randn(N, seed=4), 0.5 + 0.2 * randn(N, seed=5)
    check_gated(x, z, w.to(x_type), None, None, "silu", dout.to(x_type))
    check_gated(x, z, w, residual, c.to(x_type), "sigmoid", dout)
    check_gated(x, None, None, residual, 0.25, "silu", dout)
    check_gated(x, z, None, None, c, "silu", dout.to(x_type))


def test_many_rows_and_sums_over_them():
    """More rows than the grid holds at once, in heads and whole."""
    for shape in ((40000, 16), (9001, 128), (5000, 264), (3001, 1100)):
        x, z, dy = randn(*shape, dtype=BF16), randn(*shape, dtype=BF16, seed=1), randn(*shape, dtype=BF16, seed=2)
        w = randn(shape[-1], dtype=BF16, seed=3)
        check_gated(x, z, w, None, w, "silu", dy)
        check_residual(x, z, w, w, dy, dy)


def test_rows_of_zeros_and_gates_far_out():
    x, w = randn(6, 96), randn(96, seed=1)
    x[2] = 0
    x[3] = 1e-30
    x[4] *= 1e15
    z = randn(6, 96, seed=2)
    z[0, :8] = torch.tensor([-1e4, -200.0, -100.0, -88.0, 88.0, 200.0, 1e4, 0.0])
    for act in ("silu", "sigmoid"):
        out, grads = check_gated(x, z, w, None, None, act, randn(6, 96, seed=3))
        assert all(torch.isfinite(t).all() for t in (out, *grads))
    check_residual(x, -x, w, None, randn(6, 96, seed=4), randn(6, 96, seed=5))     # every row of the stream is zero
    z[1, 3] = -float("inf")
    assert gated_norm_call(x, z, w, activation="sigmoid")[1, 3] == 0


def test_nan_stays_in_its_row():
    x, r, w = randn(9, 40), randn(9, 40, seed=1), randn(40, seed=2)
    y, s = residual_norm_call(x, r, w)
    x[4, 7] = float("nan")
    y2, s2 = residual_norm_call(x, r, w)
    keep = [i for i in range(9) if i != 4]
    assert torch.equal(y[keep], y2[keep]) and torch.equal(s[keep], s2[keep]) and torch.isnan(y2[4]).all() and torch.isnan(s2[4]).sum() == 1


def test_strides_are_read_in_place_and_change_nothing():
    B, T, H, N = 2, 9, 4, 128
    x, z, dout = (randn(B, T, H, N, dtype=BF16, seed=s) for s in range(3))
    w = randn(N, dtype=BF16, seed=4)

    def step(x, z, dout):
        x, z, wl = x.detach().requires_grad_(True), z.detach().requires_grad_(True), w.clone().requires_grad_(True)
        out = gated_norm_call(x, z, wl)
        return (out.detach(), *torch.autograd.grad(out, (x, z, wl), dout))

    ref = step(x, z, dout)
    slices = lambda t: torch.cat([t.flatten(2), t.flatten(2)], -1)[..., H * N:].view(B, T, H, N)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    channels_apart = lambda t: t.transpose(2, 3).contiguous().transpose(2, 3)
    for view in (slices, heads_first, channels_apart):
        for a, b in zip(step(view(x), view(z), view(dout)), ref):
            assert torch.equal(a, b)
    for a, b in zip(step(shifted(x), shifted(z), shifted(dout)), ref):          # by single channels: other sums, the same to rounding
        assert torch.allclose(a.float(), b.float(), rtol=2 ** -6, atol=2e-2)
    out = gated_norm_call(x, z, w)                                              # the gradient of a sum: an expanded number
    y, s = residual_norm_call(x.requires_grad_(True), z, w)
    (y.float().sum() + s.float().sum()).backward()
    ones = torch.ones_like(y)
    within(x.grad, *residual_norm(x, z, w, None, EPS, ones, ones)["dx"], "dx")
    assert out.shape == x.shape
    # one residual for every batch row, and one row for every token
    r = randn(1, T, H, N, dtype=BF16, seed=7)
    y1, s1 = residual_norm_call(x, r.expand(B, T, H, N), w)
    y2, s2 = residual_norm_call(x, r.repeat(B, 1, 1, 1), w)
    assert torch.equal(y1, y2) and torch.equal(s1, s2)


def test_one_token_and_vectors_of_any_type():
    x, r = randn(1, 1, 512, dtype=BF16), randn(1, 1, 512, dtype=BF16, seed=1)
    for w_type in (F32, BF16, F16):
        w, c = randn(512, dtype=w_type, seed=2), randn(512, dtype=w_type, seed=3)
        check_residual(x, r, w, c, x, r)
        check_gated(x, r, w, r, c, "silu", x)
    y, s = residual_norm_call(x[0, 0], r[0, 0], scale=2)
    assert y.shape == (512,) and torch.equal(s, (r[0, 0].float() + 2 * x[0, 0].float()).to(BF16))


def test_gradients_against_differences():
    """Central differences of the f32 forward along random directions, steps of 2^-6: the truncation is of the order of the step squared
    times the loss's third derivative (terms of order one), the roundings are those of 12 * 48 terms over the step."""
    x, r, z, w, c = randn(12, 48), randn(12, 48, seed=1), randn(12, 48, seed=2), 1 + 0.1 * randn(48, seed=3), 1 + 0.1 * randn(48, seed=4)
    d1, d2 = randn(12, 48, seed=5).double(), randn(12, 48, seed=6).double()

    def before(x, r, w, c):
        y, s = residual_norm_call(x, r, w, c)
        return (y.double() * d1).sum() + (s.double() * d2).sum()

    def after(act):
        return lambda x, z, w, r, c: (gated_norm_call(x, z, w, r, c, activation=act).double() * d1).sum()

    step = 2.0 ** -6
    for loss, args in ((before, (x, r, w, c)), (after("silu"), (x, z, w, r, c)), (after("sigmoid"), (x, z, w, r, c))):
        leaves = [leaf(t) for t in args]
        grads = torch.autograd.grad(loss(*leaves), leaves)
        for i, got in enumerate(grads):
            way = randn(*args[i].shape, seed=30 + i)
            with torch.no_grad():
                slope = (loss(*[t + step * way if j == i else t for j, t in enumerate(args)]) -
                         loss(*[t - step * way if j == i else t for j, t in enumerate(args)])) / (2 * step)
            want, size = (got.double() * way.double()).sum(), (got.double() * way.double()).abs().sum()
            assert abs(slope - want) < 64 * 2.0 ** -24 * (12 * 48) ** 0.5 * 3 / step + 4 * step ** 2 * size, (i, slope.item(), want.item())


def test_captured_in_a_graph_and_on_another_stream():
    x, r, z = (randn(500, 320, dtype=BF16, seed=s) for s in range(3))
    w, c, dy = randn(320, dtype=BF16, seed=3), randn(320, dtype=BF16, seed=4), randn(500, 320, dtype=BF16, seed=5)
    leaves = [leaf(t) for t in (x, r, z, w, c)]

    def step():
        x, r, z, w, c = leaves
        y, s = residual_norm_call(x, r, w, c)
        out = gated_norm_call(y, z, w, s, c)
        return (out, *torch.autograd.grad(out, leaves, dy))

    ref = [t.detach().clone() for t in step()]               # (no eager graph of the leaves outlives its step: torch cannot capture beside one)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        for i, t in enumerate(leaves):
            t.copy_(randn(*t.shape, dtype=BF16, seed=60 + i))
    graph.replay()
    again = [t.clone() for t in out]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(again, out))
    assert all(torch.equal(a, b) for a, b in zip(again, step()))


def test_no_gradients_where_none_are_wanted():
    x, r, z, w = randn(4, 64), randn(4, 64, seed=1), randn(4, 64, seed=2), randn(64, seed=3)
    y, s = residual_norm_call(x, r, w)
    assert not y.requires_grad and not s.requires_grad and not gated_norm_call(x, z, w).requires_grad
    xl = leaf(x)
    y, s = residual_norm_call(xl, r, w, 0.5)
    dx, = torch.autograd.grad((y, s), (xl,), (r, z))
    within(dx, *residual_norm(x, r, w, 0.5, EPS, r, z)["dx"], "dx")
    wl = leaf(w)
    dw, = torch.autograd.grad(gated_norm_call(x, z, wl), (wl,), r)
    within(dw, *gated_norm(x, z, w, None, None, "silu", EPS, r)["dweight"], "dweight")
    with torch.no_grad():
        assert not residual_norm_call(xl, r, wl)[0].requires_grad


def test_refusals():
    x, r, w = randn(4, 64), randn(4, 64, seed=1), randn(64, seed=2)
    for bad in (lambda: residual_norm_call(x, r[:2], w), lambda: residual_norm_call(x, r.half(), w), lambda: residual_norm_call(x.double(), r, w),
                lambda: residual_norm_call(x, r, w[:32]), lambda: residual_norm_call(x, r, w.double()), lambda: residual_norm_call(x, r.cpu(), w),
                lambda: residual_norm_call(x, r, w.cpu()), lambda: residual_norm_call(x, r, w, scale=torch.tensor(1.0, device="cuda")),
                lambda: residual_norm_call(x, r, w, scale=x), lambda: gated_norm_call(x, r[:2], w), lambda: gated_norm_call(x, r.half(), w),
                lambda: gated_norm_call(x, r, w, residual=r.half()), lambda: gated_norm_call(x, r, w, activation="relu"),
                lambda: gated_norm_call(x, r, w[None]), lambda: gated_norm_call(x[0, 0], r[0, 0]),
                lambda: gated_norm_call(torch.empty(1, 16385, device="cuda"))):
        with pytest.raises(ValueError):
            bad()
    for shape in ((0, 8), (3, 0)):
        e = torch.empty(shape, device="cuda")
        with pytest.raises(_lib.TgdnError):
            residual_norm_call(e, e)
        with pytest.raises(_lib.TgdnError):
            gated_norm_call(e, e)
