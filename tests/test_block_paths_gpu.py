"""The inner loops and layouts of the operators around the core that small calls do not reach: many tiles of few slices (stages asked for again,
the walk over the states in several lots), wide rows in several rounds, rows off a vector's border, padded rows of odd length, odd heads in
wider rows, many short odd rows."""
import pytest
import torch

from cute_triadic_gdn_b200 import _lib, gated_scan_call
from test_block_norm_gpu import check_gated, check_residual, randn

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("lo,D,g_type", [(64, 512, F32), (0, 512, BF16), (1, 450, F32)])
@pytest.mark.parametrize("packed", (False, True))
def test_many_tiles_of_few_slices_give_the_bits_of_the_whole_way(packed, lo, D, g_type):
    """313 tiles: five lots of the walk over the states, five tiles and more a block.  The channels are those of a call wide enough to be walked
    whole; the second narrow call runs beside the first on another stream."""
    T, W = 40000, 6144
    assert _lib.lib.tgdn_scan_scratch_floats(1, T, W) == 0 < _lib.lib.tgdn_scan_scratch_floats(1, T, D)
    gen = torch.Generator(device="cuda").manual_seed(D)
    randn_ = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    cu = torch.tensor([0, 1, 5000, 5120, 20000, 20001, 39999, T], dtype=torch.int32, device="cuda") if packed else None
    n = 7 if packed else 1
    rate = 10.0 ** (-4.0 * torch.rand(W, generator=gen, device="cuda"))
    x, dh = randn_(1, T, W).to(BF16), randn_(1, T, W).to(BF16)
    g = randn_(1, T, W).abs_().neg_().mul_(rate).to(g_type)
    initial, dfinal = randn_(n, W), randn_(n, W)

    def step(x, g, initial, dh, dfinal):
        leaves = [t.detach().requires_grad_(True) for t in (x, g, initial)]
        h, final = gated_scan_call(leaves[0], leaves[1], cu, initial_state=leaves[2], output_final_state=True)
        return (h.detach(), final.detach(), *torch.autograd.grad((h, final), leaves, (dh, dfinal)))

    whole, part = step(x, g, initial, dh, dfinal), [t[..., lo:lo + D] for t in (x, g, initial, dh, dfinal)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = step(*part)
    narrow = step(*part)
    torch.cuda.current_stream().wait_stream(side)
    for name, a, b, c in zip(("h", "final", "dx", "dg", "dinitial"), whole, narrow, beside):
        assert torch.equal(a[..., lo:lo + D], b) and torch.equal(b, c), name
    assert _lib.device_status() == 0


@pytest.mark.parametrize("shape,x_type,r_type", [((300, 8200), BF16, F32), ((300, 12001), BF16, F32), ((300, 16384), BF16, BF16), ((300, 16384), F32, F32),
                                                 ((300, 16383), F16, F32), ((300, 12001), F32, F32)])
def test_wide_rows_in_several_rounds(shape, x_type, r_type):
    N = shape[-1]
    x, z, r = randn(*shape, dtype=x_type), randn(*shape, dtype=x_type, seed=1), randn(*shape, dtype=r_type, seed=2)
    dy, ds = randn(*shape, dtype=x_type, seed=3), randn(*shape, dtype=r_type, seed=4)
    w, c = 1 + 0.2 * randn(N, seed=5), 0.5 + 0.2 * randn(N, seed=6)
    check_residual(x, r, w, c, dy, ds)
    check_gated(x, z, w, r, c, "silu", ds)


def shifted(t):
    return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)


def padded(t, more=8):
    """Rows `more` elements longer than they are read, the last of which ends with its tensor's memory."""
    *outer, N = t.shape
    rows = t[..., 0].numel()
    flat = torch.full((rows * (N + more) - more,), float("nan"), dtype=t.dtype, device="cuda")
    strides, step = [1], N + more
    for n in reversed(outer):
        strides.insert(0, step)
        step *= n
    return flat.as_strided(t.shape, strides).copy_(t)


def inside(t):
    """Heads in the middle of wider rows."""
    n = t.shape[-1] * t.shape[-2]
    wide = torch.full((*t.shape[:-2], 2 * n + 9), float("nan"), dtype=t.dtype, device="cuda")
    return wide[..., 5:5 + n].view(t.shape).copy_(t)


@pytest.mark.parametrize("view,shape", [(shifted, (40, 128)), (shifted, (700, 33)), (shifted, (20, 2000)), (shifted, (9, 4096)), (shifted, (5, 16384)), (padded, (50, 33)),
                                        (padded, (21, 201)), (padded, (340, 2001)), (padded, (3, 9001)), (padded, (3, 5, 40)), (inside, (5, 9, 7, 33)),
                                        (inside, (5, 9, 3, 128)), (inside, (2, 7, 3, 1001))])
@pytest.mark.parametrize("x_type,r_type", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_rows_that_lie_apart(view, shape, x_type, r_type):
    N = shape[-1]
    x, z, r = view(randn(*shape, dtype=x_type)), view(randn(*shape, dtype=x_type, seed=1)), view(randn(*shape, dtype=r_type, seed=2))
    dy, ds = view(randn(*shape, dtype=x_type, seed=3)), view(randn(*shape, dtype=r_type, seed=4))
    w, c = 1 + 0.2 * randn(N, seed=5), 0.5 + 0.2 * randn(N, seed=6)
    check_residual(x, r, w, c, dy, ds)
    check_residual(x, randn(*shape, dtype=r_type, seed=2), w, 0.5, dy, None)
    check_gated(x, z, w, r, c, "silu", ds)
    check_gated(x, z, None, None, None, "sigmoid", dy)


@pytest.mark.parametrize("x_type,r_type", [(BF16, BF16), (BF16, F32), (F32, F32)])
@pytest.mark.parametrize("shape", [(30000, 33), (12000, 7, 33), (20011, 128), (3001, 2001)])
def test_many_rows_in_every_pair_of_types(shape, x_type, r_type):
    N = shape[-1]
    x, z, r = randn(*shape, dtype=x_type), randn(*shape, dtype=x_type, seed=1), randn(*shape, dtype=r_type, seed=2)
    dy, ds = randn(*shape, dtype=x_type, seed=3), randn(*shape, dtype=r_type, seed=4)
    w, c = 1 + 0.2 * randn(N, seed=5), 0.5 + 0.2 * randn(N, seed=6)
    check_residual(x, r, w, c, dy, ds)
    check_gated(x, z, w, r, c, "silu", ds)
