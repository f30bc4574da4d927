"""The gated scan with gates above zero: the product of a tile's decays may leave the range of f32 where the states do not.  Against the
recurrence in 64 bits, forward and backward, on both ways over the tiles, by pairs of channels and by single ones, dense and packed."""
import pytest
import torch

from block_reference import documents, scan, within
from cute_triadic_gdn_b200 import _lib, gated_scan_call, gated_scan_decode

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")
SHORT, LONG = 300, 1500                              # tokens of two rows of one slice: walked whole, and split along time


def make(T, D, x_type, sequences=2):
    """Ordinary decays with zeros in x and dh and in the states: what a case sets is what there is."""
    gen = torch.Generator().manual_seed(T + D)
    g = -torch.nn.functional.softplus(torch.randn(2, T, D, generator=gen))
    zeros = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device="cuda")
    return zeros(2, T, D, dtype=x_type), g.cuda(), zeros(sequences, D), zeros(2, T, D, dtype=x_type), zeros(sequences, D)


def underflow(g, cu, h, lam):
    """What f32 states may lose below 2^-126: nothing holds them there, so that each that is not zero may be that far off, and what grows behind
    it takes the error along: F[t] = a[t] F[t-1] + 2^-126.  (A state of 1e-20 that falls by e^-120 and grows by e^120 again is 1e-72 in between;
    no f32 state brings it back.)  F forward, and the same of the reverse recurrence, whose states go from row to row times a."""
    a = g.detach().double().cpu().exp()
    forward, reverse = torch.zeros_like(a), torch.zeros_like(a)
    for b, lo, hi, _ in documents(*a.shape[:2], cu):
        f = r = torch.zeros(a.shape[2], dtype=torch.float64)
        for t in range(lo, hi):
            f = forward[b, t] = a[b, t] * f + 2.0 ** -126 * (h[b, t] != 0)
        for t in range(hi - 1, lo - 1, -1):
            reverse[b, t] = r + 2.0 ** -126 * (lam[b, t] != 0)
            r = a[b, t] * reverse[b, t] + 2.0 ** -126 * (lam[b, t] != 0)
    return forward, reverse


def check(x, g, initial, dh, dfinal, cu=None):
    leaves = [t.detach().requires_grad_(True) for t in (x, g, initial)]
    offsets = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    h, final = gated_scan_call(leaves[0], leaves[1], offsets, initial_state=leaves[2], output_final_state=True)
    grads = torch.autograd.grad((h, final), leaves, (dh, dfinal))
    ref = scan(x, g, cu, initial, dh, dfinal)
    lost, lost_back = underflow(g, cu, ref["h"][0], ref["dx"][0])
    docs, a = documents(*x.shape[:2], cu), g.detach().double().cpu().exp()
    at = lambda t, which: torch.stack([t[b, (lo, hi - 1)[which]] for b, lo, hi, _ in docs])
    before = torch.zeros_like(a)
    before[:, 1:] = ref["h"][0][:, :-1]
    off_before = torch.zeros_like(a)
    off_before[:, 1:] = lost[:, :-1]
    for b, lo, _, d in docs:
        before[b, lo], off_before[b, lo] = initial[d].double().cpu(), 0.0
    lam = ref["dx"][0].abs()
    more = {"h": lost, "final": at(lost, 1), "dx": lost_back, "dinitial": at(a * lost_back, 0),
            "dg": a * (lost_back * before.abs() + (lam + lost_back) * off_before)}
    ref = {name: (ref[name][0], ref[name][1] + more[name]) for name in more}
    for name, got in zip(("h", "final", "dx", "dg", "dinitial"), (h, final, *grads)):
        assert ref[name][0].abs().max() < 3e38 and torch.isfinite(got).all(), name
        within(got, *ref[name], name)


def grow(kind, x, g, initial, dh, dfinal):
    """Every tile's factor passes 2^128 somewhere, no state does."""
    T = x.shape[1]
    if kind == "zeros":                              # nothing there to grow, then a small token; nothing comes back, then a small gradient
        g[:, 3:260] = 1.0
        x[:, 261], dh[:, 1] = 1e-3, 1e-3
    elif kind == "small states":                     # over a whole tile and more
        g[:, 20:148] = 1.0
        initial[:], dfinal[:] = 1e-30, 1e-30
        g[:, :20], g[:, 148:] = -1e-3, -1e-3
    elif kind == "up and down":                      # inside one tile, over its border, and inside the sixteen rows of one warp
        g[:] = -1e-3
        for t in (2, 130):
            g[:, t:t + 60], g[:, t + 60:t + 120] = 2.0, -2.0
        for t in (256, 264):
            g[:, t:t + 4], g[:, t + 4:t + 8] = 25.0, -25.0
        initial[:], dfinal[:] = 1e-20, 1e-20
        x[:, 125], dh[:, 126] = 1e-20, 1e-20
    elif kind == "down and up":                      # the same the other way round, for the reverse recurrence
        g[:] = -1e-3
        for t in (2, 130):
            g[:, t:t + 60], g[:, t + 60:t + 120] = -2.0, 2.0
        initial[:], dfinal[:] = 1e-20, 1e-20
        x[:, 125], dh[:, 126] = 1e-20, 1e-20
    elif kind == "steep":                            # factors of e^120 in twelve tokens of one warp
        g[:] = -1e-3
        g[:, 33:45] = 10.0
        initial[:], dfinal[:], dh[:, 20], x[:, 50] = 1e-30, 1e-30, 1e-10, 1.0
    elif kind == "reset":                            # a gate of minus infinity behind a factor out of range drops the state
        g[:, 2:62], g[:, 62], g[:, 140:200], g[:, 200] = 2.0, -INF, 2.0, -INF
        initial[:], dfinal[:] = 1e-20, 1e-20
        x[:, 70], dh[:, 64] = 1.0, 1.0


KINDS = ("zeros", "small states", "up and down", "down and up", "steep", "reset")


@pytest.mark.parametrize("T", (SHORT, LONG))
@pytest.mark.parametrize("D,x_type", [(64, F32), (33, F32), (64, BF16), (7, BF16)])
@pytest.mark.parametrize("kind", KINDS)
def test_states_in_range_where_factors_are_not(kind, D, x_type, T):
    assert (_lib.lib.tgdn_scan_scratch_floats(2, T, D) > 0) == (T == LONG)
    case = make(T, D, x_type)
    grow(kind, *case)
    check(*case)


@pytest.mark.parametrize("T", (SHORT, 3 * LONG))
@pytest.mark.parametrize("D,x_type", [(64, F32), (33, BF16)])
@pytest.mark.parametrize("kind", KINDS)
def test_packed_documents_of_them(kind, D, x_type, T):
    """One document grows; its neighbours begin and end in the same tiles, with tokens of their own."""
    at, N = 16, T + 90
    cu = [0, 1, at, at + T, at + T + 5, N]
    x, g, initial, dh, dfinal = make(N, D, x_type, sequences=5)
    x, g, dh = (t[:1].contiguous() for t in (x, g, dh))
    gen = torch.Generator(device="cuda").manual_seed(1)
    for lo, hi in ((0, at), (at + T, N)):
        x[:, lo:hi] = torch.randn(1, hi - lo, D, generator=gen, device="cuda").to(x_type)
        dh[:, lo:hi] = torch.randn(1, hi - lo, D, generator=gen, device="cuda").to(x_type)
    one = slice(at, at + T)
    grow(kind, x[:, one], g[:, one], initial[2:3], dh[:, one], dfinal[2:3])
    assert (_lib.lib.tgdn_scan_scratch_floats(1, N, D) > 0) == (T != SHORT)
    check(x, g, initial, dh, dfinal, cu)


@pytest.mark.parametrize("D", (64, 33))
def test_the_same_bits_alone_and_in_a_wide_batch(D):
    """Split along time and walked whole, with factors out of range among ordinary ones."""
    B, T = 120, LONG
    assert _lib.lib.tgdn_scan_scratch_floats(B, T, D) == 0 < _lib.lib.tgdn_scan_scratch_floats(2, T, D)
    gen = torch.Generator(device="cuda").manual_seed(2)
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, g, initial, dh, dfinal = randn(B, T, D), -torch.nn.functional.softplus(randn(B, T, D)), randn(B, D), randn(B, T, D), randn(B, D)
    for t in (40, 300, 700, 1290):
        g[:, t - 1] = -60.0                          # what grows has become small before
        g[:, t:t + 50, ::2], g[:, t + 50:t + 60, ::2] = 2.0, -10.0
        x[:, t - 1:t + 60] *= 1e-25
        dh[:, t - 2:t + 60] *= 1e-25
        g[:, t + 60] = -60.0

    def step(lo, hi):
        leaves = [t[lo:hi].clone().requires_grad_(True) for t in (x, g, initial)]
        h, final = gated_scan_call(leaves[0], leaves[1], initial_state=leaves[2], output_final_state=True)
        return (h.detach(), final.detach(), *torch.autograd.grad((h, final), leaves, (dh[lo:hi], dfinal[lo:hi])))

    for wide, alone in zip(step(0, B), step(7, 9)):
        assert torch.isfinite(alone).all() and torch.equal(wide[7:9], alone)


def test_the_scan_gives_what_the_steps_of_decode_give():
    T, D = 200, 48
    x, g, initial, _, _ = make(T, D, F32)
    g[:, 3:150] = 1.0
    x[:, 151] = 1e-3
    h, final = gated_scan_call(x, g, initial_state=initial, output_final_state=True)
    state = initial.clone()
    steps = torch.cat([gated_scan_decode(x[:, t:t + 1], g[:, t:t + 1], state) for t in range(T)], 1)
    assert torch.isfinite(h).all() and torch.equal(h == 0, steps == 0)
    assert torch.allclose(h, steps, rtol=1e-4, atol=0) and torch.allclose(final, state, rtol=1e-4, atol=0)
