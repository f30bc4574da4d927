"""The gated scan against the recurrence in 64 bits, token by token: types, lengths around the tiles' borders, odd channel counts, strides,
packed documents with states of their own, gates that reset, infinities and NaN in a neighbour, gradients by the formula and by differences."""
import pytest
import torch

from block_reference import scan, within
from cute_triadic_gdn_b200 import _lib, gated_scan_call, gated_scan_decode

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
PAIRS = [(BF16, F32), (BF16, BF16), (F16, F32), (F16, F16), (F32, F32)]


def make(B, T, D, x_type=F32, g_type=F32, sequences=None, seed=0, memory=0.1):
    gen = torch.Generator().manual_seed(1000 * T + 10 * D + seed)
    randn = lambda *s: torch.randn(*s, generator=gen)
    rate = memory ** (2 * torch.rand(D, generator=gen))
    x, g = randn(B, T, D).to(x_type), (-torch.nn.functional.softplus(randn(B, T, D)) * rate).to(g_type)
    return [t.cuda() for t in (x, g, randn(sequences or B, D), randn(B, T, D).to(x_type), randn(sequences or B, D))]


def offsets(cu):
    return None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")


def run_and_check(x, g, initial, dh, dfinal, cu=None):
    leaves = [t.detach().requires_grad_(True) for t in (x, g)] + ([] if initial is None else [initial.detach().requires_grad_(True)])
    h, final = gated_scan_call(leaves[0], leaves[1], offsets(cu), initial_state=leaves[2] if len(leaves) > 2 else None, output_final_state=True)
    grads = torch.autograd.grad((h, final), leaves, (dh, dfinal))
    ref = scan(x, g, cu, initial, dh, dfinal)
    assert h.dtype == x.dtype and final.dtype == F32 and grads[0].dtype == x.dtype and grads[1].dtype == g.dtype
    for name, got in zip(("h", "final", "dx", "dg", "dinitial"), (h, final, *grads)):
        within(got, *ref[name], name)
    with torch.no_grad():
        assert torch.equal(gated_scan_call(x, g, offsets(cu), initial_state=initial), h)
    return h, final, grads


@pytest.mark.parametrize("x_type,g_type", PAIRS)
@pytest.mark.parametrize("B,T,D", [(1, 1, 1), (2, 16, 2), (1, 17, 63), (2, 128, 64), (1, 129, 66), (3, 300, 5), (1, 1025, 130), (2, 200, 8), (1, 260, 24)])
def test_dense_against_the_definition(B, T, D, x_type, g_type):
    x, g, initial, dh, dfinal = make(B, T, D, x_type, g_type)
    run_and_check(x, g, initial, dh, dfinal)


@pytest.mark.parametrize("x_type,g_type,D", [(BF16, F32, 64), (F16, F16, 33), (F32, F32, 70)])
@pytest.mark.parametrize("cu", [[0, 1], [0, 1, 2, 3], [0, 16, 32, 128, 144, 256, 257], [0, 15, 127, 128, 129, 400], [0, 1000], [0, 255, 511, 512, 700]])
def test_packed_documents(cu, x_type, g_type, D):
    x, g, initial, dh, dfinal = make(1, cu[-1], D, x_type, g_type, sequences=len(cu) - 1)
    run_and_check(x, g, initial, dh, dfinal, cu)
    run_and_check(x, g, None, dh, dfinal, cu)


def test_every_token_a_document_and_64_bit_offsets():
    T, D = 300, 48
    x, g, initial, dh, dfinal = make(1, T, D, BF16, F32, sequences=T)
    run_and_check(x, g, initial, dh, dfinal, list(range(T + 1)))
    cu = torch.tensor([0, 7, T], device="cuda")
    assert torch.equal(gated_scan_call(x, g, cu), gated_scan_call(x, g, cu.int()))


def test_long_memory_stays_exact():
    """Decays of 1 - 1e-3: an exponential that leans to one side would be off by a thousand times its error (see the bound)."""
    T, D = 8192, 64
    gen = torch.Generator().manual_seed(5)
    x, g = torch.randn(1, T, D, generator=gen).cuda(), (-1e-3 * torch.rand(1, T, D, generator=gen)).cuda()
    h = gated_scan_call(x, g)
    ref, _ = scan(x, g)["h"]
    # roundings to nearest, of random sign: a walk of 1 / (1 - a) = 2000 tokens, 0.65 u each (the decay's 0.3 and the sum's 0.6), is 29 u
    # long; four times that for the products of the tiles.  Errors of one unit to one side would be 2000 u
    assert ((h.double().cpu() - ref).norm() / ref.norm()).item() < 128 * 2.0 ** -24


def test_gates_of_minus_infinity_reset_and_positive_gates_grow():
    x, g, initial, dh, dfinal = make(2, 200, 40)
    g[:, 50] = -float("inf")
    g[:, 199] = -float("inf")
    g[:, 100:110] = 0.5
    g[:, 120] = 0.0
    g[0, 130] = -200.0
    run_and_check(x, g, initial, dh, dfinal)


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_a_document_does_not_see_its_neighbours(value):
    cu, D = [0, 40, 130, 200, 333], 36
    x, g, initial, dh, dfinal = make(1, cu[-1], D, sequences=4)
    clean = run_and_check(x, g, initial, dh, dfinal, cu)
    x[:, 40:130], g[:, 60], initial[1], dfinal[1] = value, value, value, value
    dh[:, 40:130] = value
    leaves = [t.requires_grad_(True) for t in (x, g, initial)]
    h, final = gated_scan_call(*leaves[:2], offsets(cu), initial_state=initial, output_final_state=True)
    grads = torch.autograd.grad((h, final), leaves, (dh, dfinal))
    keep_rows, keep_docs = torch.tensor([*range(40), *range(130, 333)]), torch.tensor([0, 2, 3])
    for got, want, keep, axis in [(h, clean[0], keep_rows, 1), (final, clean[1], keep_docs, 0), (grads[0], clean[2][0], keep_rows, 1),
                                  (grads[1], clean[2][1], keep_rows, 1), (grads[2], clean[2][2], keep_docs, 0)]:
        assert torch.equal(got.index_select(axis, keep.cuda()), want.index_select(axis, keep.cuda()))


def test_strides_are_read_in_place_and_change_nothing():
    B, T, D = 2, 150, 64
    x, g, initial, dh, dfinal = make(B, T, D, BF16, F32)

    def step(x, g, dh):
        x, g = x.detach().requires_grad_(True), g.detach().requires_grad_(True)
        h = gated_scan_call(x, g, initial_state=initial)
        return (h.detach(), *torch.autograd.grad(h, (x, g), dh))

    ref = step(x, g, dh)
    wide = lambda t, at: torch.cat([torch.full_like(t, float("nan"))[..., :at], t, t], -1)[..., at:at + D]
    by_channel = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    by_time = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    shifted = lambda t: torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)
    for view in (lambda t: wide(t, 8), lambda t: wide(t, 7), by_channel, by_time, shifted):
        for a, b in zip(step(view(x), view(g), view(dh)), ref):
            assert torch.equal(a, b)
    # windows that overlap: rows that start eight channels after one another
    flat = torch.cat([x.flatten(), x.flatten()])
    windows = flat.as_strided((B, T, D), (T * 8, 8, 1))
    assert torch.equal(gated_scan_call(windows, g), gated_scan_call(windows.contiguous(), g))
    # gates per batch row, expanded over tokens, and per token, expanded over channels; the gradient of a sum is an expanded number
    for shape in ((B, 1, D), (1, T, 1), (1, 1, 1)):
        small = g[:shape[0], :shape[1], :shape[2]].clone().requires_grad_(True)
        h = gated_scan_call(x, small.expand(B, T, D))
        whole = small.detach().expand(B, T, D).contiguous().requires_grad_(True)
        h2 = gated_scan_call(x, whole)
        assert torch.equal(h, h2)
        h.float().sum().backward()
        h2.float().sum().backward()
        assert torch.allclose(small.grad, whole.grad.sum_to_size(shape), rtol=1e-4, atol=1e-3)


def test_results_do_not_depend_on_the_batch_or_on_the_widths_around():
    x, g, initial, dh, dfinal = make(5, 700, 130, BF16, F32)
    leaves = [t.requires_grad_(True) for t in (x, g, initial)]
    h, final = gated_scan_call(x, g, initial_state=initial, output_final_state=True)
    grads = torch.autograd.grad((h, final), leaves, (dh, dfinal))
    for b in (0, 3):
        part = [t.detach()[b:b + 1].clone().requires_grad_(True) for t in leaves]
        hb, fb = gated_scan_call(part[0], part[1], initial_state=part[2], output_final_state=True)
        for a, r in zip((hb, fb, *torch.autograd.grad((hb, fb), part, (dh[b:b + 1], dfinal[b:b + 1]))), (h, final, *grads)):
            assert torch.equal(a, r[b:b + 1])
    narrow = gated_scan_call(x[..., :33], g[..., :33], initial_state=initial[:, :33].contiguous())
    assert torch.equal(narrow, h[..., :33])


@pytest.mark.parametrize("D,x_type,g_type", [(64, BF16, F32), (72, F16, F16), (33, F32, F32)])
def test_long_sequences_alone_and_in_a_wide_batch(D, x_type, g_type):
    """Few slices of a long sequence are split along time, many are walked whole: the same bits, and those of the definition."""
    B, T = 120, 1500
    x, g, initial, dh, dfinal = make(B, T, D, x_type, g_type)
    assert _lib.lib.tgdn_scan_scratch_floats(B, T, D) == 0 < _lib.lib.tgdn_scan_scratch_floats(2, T, D)                # (the two ways)
    leaves = [t.requires_grad_(True) for t in (x, g, initial)]
    h, final = gated_scan_call(x, g, initial_state=initial, output_final_state=True)
    grads = torch.autograd.grad((h, final), leaves, (dh, dfinal))
    part = [t.detach()[7:9].clone() for t in (x, g, initial, dh, dfinal)]
    hb, fb, gb = run_and_check(*part)
    for a, r in zip((hb, fb, *gb), (h, final, *grads)):
        assert torch.equal(a, r[7:9])


@pytest.mark.parametrize("x_type,g_type,D", [(BF16, F32, 40), (F16, F16, 7), (F32, F32, 66), (BF16, BF16, 128)])
def test_long_packed_rows(x_type, g_type, D):
    cu = [0, 1, 128, 129, 1000, 1024, 1500, 2047, 2048, 2300]
    x, g, initial, dh, dfinal = make(1, cu[-1], D, x_type, g_type, sequences=len(cu) - 1)
    run_and_check(x, g, initial, dh, dfinal, cu)
    run_and_check(x, g, None, dh, dfinal, cu)


def test_segments_and_decode_continue_a_sequence():
    B, T, D = 2, 384 + 40, 66
    x, g, initial, dh, dfinal = make(B, T, D, BF16, F32)
    whole = [t.clone().requires_grad_(True) for t in (x, g, initial)]
    h, final = gated_scan_call(whole[0], whole[1], initial_state=whole[2], output_final_state=True)
    ref = torch.autograd.grad((h, final), whole, (dh, dfinal))
    parts, state, outs = [t.clone().requires_grad_(True) for t in (x, g, initial)], None, []
    state = parts[2]
    for lo, hi in ((0, 128), (128, 384), (384, T)):                     # at whole tiles the same bits
        o, state = gated_scan_call(parts[0][:, lo:hi], parts[1][:, lo:hi], initial_state=state, output_final_state=True)
        outs.append(o)
    assert torch.equal(torch.cat(outs, 1), h) and torch.equal(state, final)
    for a, r in zip(torch.autograd.grad((torch.cat(outs, 1), state), parts, (dh, dfinal)), ref):
        assert torch.equal(a, r)
    with torch.no_grad():
        _, state = gated_scan_call(x[:, :384], g[:, :384], initial_state=initial, output_final_state=True)
        steps = [gated_scan_decode(x[:, t:t + 1], g[:, t:t + 1], state) for t in range(384, T)]
    want = scan(x, g, None, initial)
    within(torch.cat(steps, 1), want["h"][0][:, 384:], want["h"][1][:, 384:], "decode")
    within(state, *want["final"], "decoded state")


@pytest.mark.parametrize("x_type,g_type", PAIRS)
@pytest.mark.parametrize("B,D", [(1, 1), (3, 7), (2, 64), (130, 257)])
def test_decode_against_the_definition(B, D, x_type, g_type):
    x, g, state, _, _ = make(B, 1, D, x_type, g_type)
    ref = scan(x, g, None, state)
    for forms in ((x, g), (x[:, 0], g[:, 0]), (torch.cat([x, x], -1)[..., :D], torch.cat([g, g], -1)[..., :D])):
        s = state.clone()
        h = gated_scan_decode(*forms, s)
        assert h.shape == forms[0].shape and h.dtype == x_type
        within(h.reshape(B, 1, D), *ref["h"], "h")
        within(s, *ref["final"], "state")


def test_gradients_against_differences():
    """Central differences of the f32 forward along random directions.  Linear in x and in the initial state; in g the step e leaves
    e^2 / 6 of the third derivative, which is no larger than the loss's terms times the memory cubed."""
    x, g, initial, dh, dfinal = make(1, 96, 34, memory=1.0)             # memories of a few tokens
    leaves = [t.requires_grad_(True) for t in (x, g, initial)]
    cu = offsets([0, 40, 96])
    initial2 = torch.cat([initial, initial + 1]).detach().requires_grad_(True)
    leaves[2] = initial2
    dfinal = torch.cat([dfinal, -dfinal])

    def loss(x, g, s):
        h, final = gated_scan_call(x, g, cu, initial_state=s, output_final_state=True)
        return (h.double() * dh.double()).sum() + (final.double() * dfinal.double()).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for i, step in ((0, 0.5), (1, 2.0 ** -7), (2, 0.5)):
        way = torch.randn(leaves[i].shape, generator=gen, device="cuda")
        with torch.no_grad():
            moved = lambda s: loss(*[t + s * way if j == i else t for j, t in enumerate(leaves)])
            slope = (moved(step) - moved(-step)) / (2 * step)
        want = (grads[i].double() * way.double()).sum()
        size = (grads[i].double() * way.double()).abs().sum()
        # 96 * 34 terms of the loss, each a few u of about one off, over the step; the truncation 2^-14 / 6 times a few of the size
        assert abs(slope - want) < 100 * 2.0 ** -24 * 96 * 34 ** 0.5 / step + 1e-3 * size, (i, slope.item(), want.item())


def test_captured_in_a_graph_and_on_another_stream():
    x, g, initial, dh, dfinal = make(1, 500, 96, BF16, F32, sequences=3)
    cu = offsets([0, 100, 228, 500])

    def step(x, g, initial):
        h, final = gated_scan_call(x, g, cu, initial_state=initial, output_final_state=True)
        return (h, final, *torch.autograd.grad((h, final), (x, g, initial), (dh, dfinal)))

    leaves = [t.clone().requires_grad_(True) for t in (x, g, initial)]
    ref = [t.detach().clone() for t in step(*leaves)]        # (no eager graph of the leaves outlives its step: torch cannot capture beside one)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*leaves)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*leaves)
    with torch.no_grad():
        for t, fresh in zip(leaves, make(1, 500, 96, BF16, F32, sequences=3, seed=1)):
            t.copy_(fresh)
    graph.replay()
    again = [t.clone() for t in out]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(again, out))
    assert all(torch.equal(a, b) for a, b in zip(again, step(*leaves))) and not torch.equal(again[0], ref[0])


def test_decode_counts_as_a_change_of_its_state():
    x, g, initial, _, _ = make(2, 32, 8)
    x.requires_grad_(True)
    h = gated_scan_call(x, g, initial_state=initial)
    before = initial._version
    with torch.no_grad():
        gated_scan_decode(x[:, :1].detach(), g[:, :1], initial)
    assert initial._version == before + 1
    with pytest.raises(RuntimeError, match="inplace"):                          # the backward of h would read the state of later
        h.sum().backward()
    with torch.inference_mode():
        state = gated_scan_call(x.detach(), g, output_final_state=True)[1]
        first = gated_scan_decode(x[:, :1].detach(), g[:, :1], state)
    with torch.no_grad():
        second = gated_scan_decode(x[:, :1].detach(), g[:, :1], state)          # a state of inference mode carries no count
    assert first.shape == second.shape and not torch.equal(first, second)


def test_unused_outputs_and_partial_gradients():
    x, g, initial, dh, dfinal = make(2, 70, 32)
    leaves = [t.requires_grad_(True) for t in (x, g, initial)]
    h, final = gated_scan_call(x, g, initial_state=initial, output_final_state=True)
    only_final = torch.autograd.grad(final, leaves, dfinal)
    ref = scan(x, g, None, initial, torch.zeros_like(dh), dfinal)
    for name, got in zip(("dx", "dg", "dinitial"), only_final):
        within(got, *ref[name], name)
    with torch.no_grad():
        frozen = gated_scan_call(x, g, initial_state=initial)
    assert not frozen.requires_grad
    s, = torch.autograd.grad(gated_scan_call(x.detach(), g.detach(), initial_state=initial), initial, dh)
    within(s, *scan(x, g, None, initial, dh)["dinitial"], "dinitial alone")


def test_more_than_two_to_the_31_elements():
    """Offsets pass 32 bits: the last batch row and the last channels are those of a call of their own."""
    B, T, D = 3, 70000, 11000
    x = torch.zeros(B, T, D, dtype=BF16, device="cuda")
    assert x.numel() > 2 ** 31
    g = torch.full((1, 1, D), -0.25, dtype=BF16, device="cuda").expand(B, T, D)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x[-1, -300:, -64:] = torch.randn(300, 64, generator=gen, device="cuda").to(BF16)
    x.requires_grad_(True)
    h = gated_scan_call(x, g)
    tail = x.detach()[-1:, -300:, -64:].clone().requires_grad_(True)
    small = gated_scan_call(tail, g[-1:, -300:, -64:])
    within(h[-1:, -300:, -64:], *scan(tail, g[-1:, -300:, -64:])["h"], "h")
    assert not h[0].any() and not h[-1, :-300].any()
    del small
    dh = torch.zeros_like(h)
    dh[-1, -1, -1] = 1.0
    dx, = torch.autograd.grad(h, x, dh)
    assert dx[-1, -1, -1] == 1 and abs(dx[-1, -2, -1].item() - 0.7788) < 4e-3 and not dx[:2].any()


def test_refusals():
    x, g, initial, dh, dfinal = make(2, 32, 8)
    cu = offsets([0, 32])
    for bad in (lambda: gated_scan_call(x, g[:, :16]), lambda: gated_scan_call(x[0], g[0]), lambda: gated_scan_call(x, g.half()),
                lambda: gated_scan_call(x.double(), g), lambda: gated_scan_call(x, g.cpu()), lambda: gated_scan_call(x, g, initial_state=initial[:1]),
                lambda: gated_scan_call(x, g, initial_state=initial.half()), lambda: gated_scan_call(x, g, cu),
                lambda: gated_scan_call(x[:1], g[:1], cu.cpu()), lambda: gated_scan_call(x[:1], g[:1], cu.float()),
                lambda: gated_scan_call(x[:1], g[:1], cu[:1]), lambda: gated_scan_call(x[:1], g[:1], cu, initial_state=initial),
                lambda: gated_scan_decode(x, g, initial), lambda: gated_scan_decode(x[:, :1], g[:, :1], initial.half()),
                lambda: gated_scan_decode(x[:, :1], g[:, :1], initial[:1]), lambda: gated_scan_decode(x[:, :1], g[:, :1], initial.t().contiguous().t()),
                lambda: gated_scan_decode(x[:, :1].clone().requires_grad_(True), g[:, :1], initial)):
        with pytest.raises(ValueError):
            bad()
    for shape in ((0, 8, 4), (2, 0, 4), (2, 8, 0)):
        with pytest.raises(_lib.TgdnError):
            gated_scan_call(torch.empty(shape, device="cuda"), torch.empty(shape, device="cuda"))
    for B, D in ((0, 4), (2, 0)):
        with pytest.raises(_lib.TgdnError):
            gated_scan_decode(torch.empty(B, D, device="cuda"), torch.empty(B, D, device="cuda"), torch.empty(B, D, device="cuda"))
