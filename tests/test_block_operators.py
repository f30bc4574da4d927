"""The operators around the core without a GPU (registrations, shapes, refusals, the reference of the tests itself) and, on one, a block that
is put together from them."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from block_reference import gated_norm, residual_norm, scan
from cute_triadic_gdn_b200 import (_lib, conv_split_norm_call, gated_norm_call, gated_scan_call, gated_scan_decode, gdn_joint_call,
                                   residual_norm_call)

BF16, F32 = torch.bfloat16, torch.float32


def test_fake_kernels_give_the_real_shapes():
    ops = torch.ops.tgdn_b200
    with FakeTensorMode():
        like = lambda *shape, dtype=BF16: torch.empty(*shape, dtype=dtype, device="cuda")
        x, g = like(2, 300, 40), like(2, 300, 40, dtype=F32)
        h, final, carry = ops.gated_scan_fwd(x, g, None, None, 0, True, True)
        assert h.shape == x.shape and h.dtype == BF16 and final.shape == (2, 40) and final.dtype == F32
        assert carry.numel() == _lib.lib.tgdn_scan_carry_floats(2, 300, 40) == 2 * 3 * 40
        assert [t.numel() for t in ops.gated_scan_fwd(x, g)[1:]] == [0, 0]
        dx, dg, dinitial = ops.gated_scan_bwd(x, g, x, carry, final)
        assert dx.shape == dg.shape == x.shape and dg.dtype == F32 and dinitial.shape == (2, 40)
        doc_map, valid = ops.gated_scan_map(like(5, dtype=torch.int32), 300)
        assert doc_map.shape == (300,) and valid.shape == (1,)
        assert ops.gated_scan_fwd(x[:1], g[:1], None, doc_map, 4, True)[1].shape == (4, 40)
        r, w = like(2, 300, 40, dtype=F32), like(40)
        y, stream, rstd = ops.residual_norm_fwd(x, r, w, w, 1.0, 1e-6, True)
        assert y.dtype == BF16 and stream.dtype == F32 and y.shape == stream.shape == x.shape and rstd.shape == (600,)
        dr, dxr, dw, dc = ops.residual_norm_bwd(stream, x, BF16, y, stream, w, w, 1.0, rstd, True, True)
        assert dr.dtype == F32 and dxr.dtype == BF16 and dw.shape == dc.shape == (40,)
        assert [t.numel() for t in ops.residual_norm_bwd(y, None, BF16, y, None, None, None, 1.0, rstd, False, False)[1:]] == [0, 0, 0]
        out, rstd = ops.gated_norm_fwd(x, x, w, r, w, 1.0, 1, 1e-6, True)
        assert out.dtype == F32 and rstd.shape == (600,)
        dx, dz, dw, dc = ops.gated_norm_bwd(x, x, out, w, w, 1.0, 1, rstd, True, False)
        assert dx.shape == dz.shape == x.shape and dw.shape == (40,) and dc.numel() == 0


def test_calls_without_a_gpu_are_refused():
    x, w = torch.ones(2, 8, 16), torch.ones(16)
    for call in (lambda: gated_scan_call(x, x), lambda: residual_norm_call(x, x, w), lambda: gated_norm_call(x, x, w)):
        with pytest.raises(NotImplementedError, match="CPU"):
            call()
    with pytest.raises(ValueError, match="CUDA device"):
        gated_scan_decode(x[:, :1], x[:, :1], torch.zeros(2, 16))
    with pytest.raises(ValueError, match="activation"):
        gated_norm_call(x, x, w, activation="tanh")
    with pytest.raises(ValueError, match="cu_seqlens"):
        gated_scan_call(x[:1], x[:1], torch.tensor([0.0, 8.0]))
    with pytest.raises(ValueError, match="packed row"):
        gated_scan_call(x, x, torch.tensor([0, 8]))


def test_arguments_of_the_c_abi_are_checked_before_a_launch():
    L, fake, null = _lib.lib, ctypes.c_void_p(4096), None
    rows = lambda t=1, data=4096, inner=8: ctypes.byref(_lib.Rows(data, inner, 64, 8, t))
    vec = lambda t=1, data=4096: ctypes.byref(_lib.Vector(data, t))
    assert L.tgdn_scan_fwd(null, rows(), null, 0, 1, 8, 8, null, fake, null, null, null, 0, null) == -2
    assert L.tgdn_scan_fwd(rows(), rows(), null, 0, 1, 8, 8, null, null, null, null, null, 0, null) == -2
    assert L.tgdn_scan_fwd(rows(), rows(7), null, 0, 1, 8, 8, null, fake, null, null, null, 0, null) == -8
    assert L.tgdn_scan_fwd(rows(), rows(), null, 0, 1, 0, 8, null, fake, null, null, null, 0, null) == -1
    assert L.tgdn_scan_fwd(rows(), rows(), fake, 2, 2, 8, 8, null, fake, null, null, null, 0, null) == -1          # a packed row of two batch rows
    assert L.tgdn_scan_bwd(rows(), rows(), rows(), null, 0, 1, 8, 8, null, null, null, fake, fake, null, null, 0, null) == -2
    assert L.tgdn_scan_bwd(rows(), rows(), rows(0), null, 0, 1, 8, 8, null, fake, null, fake, fake, null, null, 0, null) == -8
    assert L.tgdn_scan_fwd(rows(), rows(), null, 0, 1, 4096, 8, null, fake, null, null, null, 0, null) == -5
    assert L.tgdn_scan_step(rows(), rows(), 1, 8, null, fake, null) == -2
    assert L.tgdn_scan_map(fake, 0, 0, 8, fake, fake, null) == -1 and L.tgdn_scan_map(null, 0, 1, 8, fake, fake, null) == -2
    assert L.tgdn_residual_norm_fwd(rows(), rows(), null, null, 1.0, 8, 16385, 1e-6, fake, fake, null, null) == -1
    assert L.tgdn_residual_norm_fwd(rows(), rows(), vec(9), null, 1.0, 8, 8, 1e-6, fake, fake, null, null) == -8
    assert L.tgdn_residual_norm_fwd(rows(), null, null, null, 1.0, 8, 8, 1e-6, fake, fake, null, null) == -2
    assert L.tgdn_residual_norm_fwd(rows(), rows(1, 4096, 0), null, null, 1.0, 8, 8, 1e-6, fake, fake, null, null) == -1
    assert L.tgdn_residual_norm_bwd(fake, 1, null, 1, rows(), null, null, vec(), 1.0, fake, 8, 8, fake, fake, null, vec(), null, 0, null) == -2
    assert L.tgdn_gated_norm_fwd(rows(), null, 1, null, null, null, 1.0, 8, 8, 1e-6, fake, 1, null, null) == -2
    assert L.tgdn_gated_norm_fwd(rows(), rows(), 5, null, null, null, 1.0, 8, 8, 1e-6, fake, 1, null, null) == -1
    assert L.tgdn_gated_norm_fwd(rows(), rows(2), 1, null, null, null, 1.0, 8, 8, 1e-6, fake, 1, null, null) == -8
    assert L.tgdn_gated_norm_bwd(rows(), null, 0, rows(), null, null, 1.0, null, 8, 8, fake, null, null, null, null, 0, null) == -2
    assert L.tgdn_norm_scratch_floats(0, 8) == 0 and L.tgdn_norm_scratch_floats(8, 16385) == 0
    for code in (-8,):
        assert b"type" in L.tgdn_error_string(code)


def test_the_reference_of_the_tests_is_the_gradient_of_its_own_forward():
    """Its backward formulas against autograd and against differences, in 64 bits."""
    gen = torch.Generator().manual_seed(1)
    randn = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    x, g, s0, dh, dfin, cu = randn(1, 9, 3), -randn(1, 9, 3).abs(), randn(2, 3), randn(1, 9, 3), randn(2, 3), [0, 4, 9]

    def scan_loss(x, g, s0):
        loss = 0.0
        for d, (lo, hi) in enumerate(zip(cu[:-1], cu[1:])):
            h = s0[d]
            for t in range(lo, hi):
                h = g[0, t].exp() * h + x[0, t]
                loss = loss + (h * dh[0, t]).sum()
            loss = loss + (h * dfin[d]).sum()
        return loss

    leaves = [t.clone().requires_grad_(True) for t in (x, g, s0)]
    ref = scan(x, g, cu, s0, dh, dfin)
    assert torch.autograd.gradcheck(scan_loss, leaves)
    for name, grad in zip(("dx", "dg", "dinitial"), torch.autograd.grad(scan_loss(*leaves), leaves)):
        assert torch.allclose(ref[name][0], grad, rtol=1e-12, atol=1e-12), name

    x, r, z, w, c, d1, d2 = randn(4, 6), randn(4, 6), randn(4, 6), randn(6), randn(6), randn(4, 6), randn(4, 6)
    norm = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-3).sqrt()

    def before(x, r, w, c):
        s = r + c * x
        return (norm(s) * w * d1).sum() + (s * d2).sum()

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w, c)]
    ref = residual_norm(x, r, w, c, 1e-3, d1, d2)
    assert torch.autograd.gradcheck(before, leaves)
    for name, grad in zip(("dx", "dresidual", "dweight", "dscale"), torch.autograd.grad(before(*leaves), leaves)):
        assert torch.allclose(ref[name][0], grad, rtol=1e-12, atol=1e-12), name
    for act, f in (("silu", torch.nn.functional.silu), ("sigmoid", torch.sigmoid)):
        after = lambda x, z, w, r, c: ((r + c * norm(x) * w * f(z)) * d1).sum()
        leaves = [t.clone().requires_grad_(True) for t in (x, z, w, r, c)]
        ref = gated_norm(x, z, w, r, c, act, 1e-3, d1)
        assert torch.autograd.gradcheck(after, leaves)
        for name, grad in zip(("dx", "dgate", "dweight", None, "dscale"), torch.autograd.grad(after(*leaves), leaves)):
            assert name is None or torch.allclose(ref[name][0], grad, rtol=1e-12, atol=1e-12), name


# ---- a block put together from them -------------------------------------------------------------------------------------
H, E, N = 2, 4, 256


def block(x, stream, p, cu, call):
    """Two layers of a hybrid stack: the residual stream and its norm, projections, the Triadic GDN core behind its pre-pass, the gated norm
    per head; then the gated scan between the same norms, its output normed into the stream."""
    y, stream = call["residual"](x, stream, p["w1"], p["c1"])
    q, k, v, k2, q2 = conv_split_norm_call((y @ p["qkv"]), p["conv"], H, E, cu)
    g, beta = -torch.nn.functional.softplus((y @ p["g"]).float()).view(1, -1, H, E), torch.sigmoid((y @ p["beta"]).float()).view(1, -1, H)
    o = gdn_joint_call(q, k, v, k2, q2, g, beta, cu_seqlens=cu)
    o = call["gated"](o, (y @ p["gate"]).view(o.shape), p["w2"])
    y, stream = call["residual"](o.flatten(2) @ p["out"], stream, p["w3"], 0.5)
    z = y @ p["scan"]
    h = call["scan"](z[..., :N], -torch.nn.functional.softplus(z[..., N:2 * N].float()), cu)
    return call["gated"](h, z[..., 2 * N:], p["w4"], stream, p["c2"], "sigmoid")


def plain_calls():
    """The same calls in f32 torch operations, differentiated by autograd."""
    norm = lambda t: t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6)

    def residual(x, stream, w, scale):
        s = stream.float() + (scale.float() if torch.is_tensor(scale) else scale) * x.float()
        return (norm(s) * w.float()).to(x.dtype), s.to(stream.dtype)

    def gated(x, gate, w, stream=None, scale=None, activation="silu"):
        y = norm(x.float()) * w.float() * (torch.nn.functional.silu if activation == "silu" else torch.sigmoid)(gate.float())
        return y.to(x.dtype) if stream is None else (stream.float() + scale.float() * y).to(stream.dtype)

    def recurrence(x, g, cu):
        out, starts, h = [], set(cu.tolist()), None
        for t in range(x.shape[1]):
            h = x[:, t].float() + (0 if t in starts else g[:, t].exp() * h)
            out.append(h)
        return torch.stack(out, 1).to(x.dtype)

    return {"residual": residual, "gated": gated, "scan": recurrence}


def make_block(T):
    gen = torch.Generator().manual_seed(9)
    C = H * (3 * 128 + 2 * E)
    randn = lambda *s, std=1.0, dtype=BF16: (std * torch.randn(*s, generator=gen)).to(dtype).cuda()
    p = {"w1": 1 + randn(N, std=0.1), "c1": 1 + randn(N, std=0.1), "qkv": randn(N, C, std=N ** -0.5), "conv": randn(C, 4, std=0.5),
         "g": randn(N, H * E, std=N ** -0.5), "beta": randn(N, H, std=N ** -0.5), "gate": randn(N, H * 128, std=N ** -0.5), "w2": 1 + randn(128, std=0.1),
         "out": randn(H * 128, N, std=(H * 128) ** -0.5), "w3": 1 + randn(N, std=0.1), "scan": randn(N, 3 * N, std=N ** -0.5),
         "w4": 1 + randn(N, std=0.1), "c2": 1 + randn(N, std=0.1)}
    return randn(1, T, N), randn(1, T, N, dtype=F32), p, randn(1, T, N, dtype=F32)


@pytest.mark.gpu
def test_a_block_of_them_forward_and_backward():
    T, cu = 300, torch.tensor([0, 17, 150, 300], dtype=torch.int32).cuda()
    x, stream, p, dout = make_block(T)
    own = {"residual": residual_norm_call, "gated": gated_norm_call, "scan": gated_scan_call}
    results = []
    for call in (own, plain_calls()):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, stream, *p.values())]
        out = block(leaves[0], leaves[1], dict(zip(p, leaves[2:])), cu, call)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    assert _lib.device_status() == 0
    # both run bf16 between the operators, rounded at the same places: what differs are last places of f32 that flip a rounding now and then
    # (2^-8 of a value each), and the backward's norm of the stream, which is f32 here
    for name, a, b in zip(["out", "x", "stream", *p], *results):
        assert a.dtype == b.dtype and ((a.double() - b.double()).norm() / b.double().norm()).item() < 2e-2, name


@pytest.mark.gpu
def test_one_node_per_call_under_torch_compile():
    x, stream, p, _ = make_block(200)
    cu = torch.tensor([0, 60, 200], dtype=torch.int32).cuda()

    def step(x, stream, w, cu):
        y, s = residual_norm_call(x, stream, w, 0.5)
        h = gated_scan_call(y, -stream.abs(), cu)
        return gated_norm_call(h, y, w, s)

    seen = []

    def backend(gm, example_inputs):
        seen.extend(str(n.target) for n in gm.graph.nodes if n.op == "call_function" and "tgdn_b200" in str(n.target))
        return gm.forward

    with torch.no_grad():
        assert torch.equal(torch.compile(step, backend=backend, fullgraph=True)(x, stream, p["w1"], cu), step(x, stream, p["w1"], cu))
    assert len(seen) == 4 and all(any(name in t for t in seen) for name in ("residual_norm_fwd", "gated_scan_map", "gated_scan_fwd", "gated_norm_fwd"))
    results = []
    for fn in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, stream, p["w1"])]
        out = fn(*leaves, cu)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out))])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_c_abi_entries_give_the_packages_bits():
    """The entries as include/tgdn.h declares them, on the caller's buffers, against the operators that reach them through the package."""
    L, p, ops = _lib.lib, _lib.ptr, torch.ops.tgdn_b200
    gen = torch.Generator().manual_seed(4)
    randn = lambda *s, dtype=F32: torch.randn(*s, generator=gen).to(dtype).cuda()
    nan = lambda *s, dtype=F32: torch.full(s, float("nan"), dtype=dtype, device="cuda")
    ids = {F32: 0, BF16: 1, torch.float16: 2}
    rows = lambda t: ctypes.byref(_lib.Rows(t.data_ptr(), t.shape[-2] if t.dim() > 2 else t.shape[0], t.stride(0), t.stride(-2), ids[t.dtype]))
    vec = lambda t: ctypes.byref(_lib.Vector(t.data_ptr(), ids[t.dtype]))

    def call(name, *args):
        _lib.check(getattr(L, name)(*[p(a) if torch.is_tensor(a) else a for a in args], _lib.stream_of(randn(1))), name)

    for T, D, cu in ((200, 24, [0, 50, 51, 200]), (3000, 40, [0, 1000, 3000]), (3000, 33, None)):
        x, g, dh, docs = randn(1, T, D, dtype=BF16), -randn(1, T, D).abs(), randn(1, T, D, dtype=BF16), len(cu) - 1 if cu else 0
        initial, dfinal = randn(docs or 1, D), randn(docs or 1, D)
        doc_map = None
        if cu:
            doc_map, valid = torch.full((T,), -1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.bool, device="cuda")
            call("tgdn_scan_map", torch.tensor(cu, device="cuda"), 1, docs, T, doc_map, valid)
            assert bool(valid) and doc_map.nonzero().flatten().tolist() == cu[:-1] and doc_map[cu[:-1]].tolist() == list(range(1, docs + 1))
        floats = L.tgdn_scan_scratch_floats(1, T, D)
        scratch = nan(floats) if floats else None
        h, final, carry = nan(1, T, D, dtype=BF16), nan(docs or 1, D), nan(L.tgdn_scan_carry_floats(1, T, D))
        call("tgdn_scan_fwd", rows(x), rows(g), doc_map, docs, 1, T, D, initial, h, final, carry, scratch, floats)
        dx, dg, dinitial = nan(1, T, D, dtype=BF16), nan(1, T, D), nan(docs or 1, D)
        call("tgdn_scan_bwd", rows(x), rows(g), rows(dh), doc_map, docs, 1, T, D, initial, carry, dfinal, dx, dg, dinitial, scratch, floats)
        want = (*ops.gated_scan_fwd(x, g, initial, doc_map, docs, True, True), *ops.gated_scan_bwd(x, g, dh, carry, initial, doc_map, docs, dfinal))
        assert all(torch.equal(a, b) for a, b in zip((h, final, carry, dx, dg, dinitial), want))
        # without what is optional
        h2 = nan(1, T, D, dtype=BF16)
        call("tgdn_scan_fwd", rows(x), rows(g), doc_map, docs, 1, T, D, initial, h2, None, None, scratch, floats)
        assert torch.equal(h, h2)
    state, token = randn(3, 40), nan(3, 1, 40, dtype=BF16)
    x, g, kept = randn(3, 1, 40, dtype=BF16), -randn(3, 1, 40).abs(), state.clone()
    call("tgdn_scan_step", rows(x), rows(g), 3, 40, state, token)
    assert torch.equal(gated_scan_decode(x, g, kept), token) and torch.equal(kept, state)

    for R, N in ((70, 96), (9, 2001)):
        x, r, z, dy, w, c = randn(R, N, dtype=BF16), randn(R, N), randn(R, N, dtype=BF16), randn(R, N, dtype=BF16), randn(N), randn(N, dtype=BF16)
        y, stream, rstd = nan(R, N, dtype=BF16), nan(R, N), nan(R)
        call("tgdn_residual_norm_fwd", rows(x), rows(r), vec(w), vec(c), 1.0, R, N, 1e-6, y, stream, rstd)
        assert all(torch.equal(a, b) for a, b in zip((y, stream, rstd), ops.residual_norm_fwd(x, r, w, c, 1.0, 1e-6, True)))
        floats = L.tgdn_norm_scratch_floats(R, N)
        scratch, dr, dx, dw, dc = nan(floats), nan(R, N), nan(R, N, dtype=BF16), nan(N), nan(N, dtype=BF16)
        call("tgdn_residual_norm_bwd", stream, 0, rows(x), 1, rows(dy), rows(r), vec(w), vec(c), 1.0, rstd, R, N, dr, dx, vec(dw), vec(dc), scratch, floats)
        want = ops.residual_norm_bwd(stream, x, BF16, dy, r, w, c, 1.0, rstd, True, True)
        assert all(torch.equal(a, b) for a, b in zip((dr, dx, dw, dc), want))
        out, rstd = nan(R, N), nan(R)
        call("tgdn_gated_norm_fwd", rows(x), rows(z), 1, vec(w), rows(r), vec(c), 1.0, R, N, 1e-6, out, 0, rstd)
        assert all(torch.equal(a, b) for a, b in zip((out, rstd), ops.gated_norm_fwd(x, z, w, r, c, 1.0, 1, 1e-6, True)))
        dx, dz, dw, dc = nan(R, N, dtype=BF16), nan(R, N, dtype=BF16), nan(N), nan(N, dtype=BF16)
        call("tgdn_gated_norm_bwd", rows(x), rows(z), 1, rows(r), vec(w), vec(c), 1.0, rstd, R, N, dx, dz, vec(dw), vec(dc), scratch, floats)
        want = ops.gated_norm_bwd(x, z, r, w, c, 1.0, 1, rstd, True, True)
        assert all(torch.equal(a, b) for a, b in zip((dx, dz, dw, dc), want))
        assert L.tgdn_residual_norm_bwd(p(stream), 0, rows(x), 1, rows(dy), None, vec(w), vec(c), 1.0, p(rstd), R, N, p(dr), p(dx), vec(dw), vec(dc),
                                        p(scratch), 1, None) == -5
    assert _lib.device_status() == 0
