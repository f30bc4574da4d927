"""The operators around the core in 64 bits, with a bound on what f32 arithmetic may make of them.

u = 2^-24 is half a step of f32.  A bound counts the roundings that a term of a sum goes through on the longest way, times the sum of the
terms' absolute values (first order); the rounding of a result to its type, half a step of that, comes on top in `within`."""
import torch

U = 2.0 ** -24
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -126}   # half a step of the smallest numbers; f32: flushed


def within(got, ref, bound, name=""):
    """|got - ref| is at most the bound and half a step of got's type; the same values where ref is not finite."""
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    got64, ref, bound = got.detach().double().cpu(), ref.detach().double().cpu(), bound.detach().double().cpu()
    half = torch.finfo(got.dtype).eps / 2
    off = (got64 - ref).abs() - (half * (ref.abs() + bound) + bound + SMALLEST[got.dtype])
    bad = ~(off <= 0) & torch.isfinite(ref)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}, " \
                          f"got {got64[bad][0].item()!r}, expected {ref[bad][0].item()!r}, bound {bound[bad][0].item():.3e}"
    same = torch.isfinite(ref) | (got64 == ref) | (torch.isnan(got64) & torch.isnan(ref))
    assert same.all(), f"{name}: infinities or NaN elsewhere than expected"


def documents(B, T, cu):
    return [(b, 0, T, b) for b in range(B)] if cu is None else [(0, lo, hi, d) for d, (lo, hi) in enumerate(zip(cu[:-1], cu[1:]))]


def scan(x, g, cu=None, initial=None, dh=None, dfinal=None):
    """{name: (value, bound)} of h, final and, with dh, of dx, dg, dinitial.

    A term of h[t] that came in s tokens before has passed s decays, each with the error of exp (four roundings of the hardware's power of
    two, and the rounding of g's product with log2 e, |g| of them), a product and a sum; putting tiles together costs it twenty more."""
    x, g = x.detach().double().cpu(), g.detach().double().cpu()
    B, T, D = x.shape
    a, cost = g.exp(), 6 + 2 * torch.where(torch.isfinite(g), g.abs(), torch.zeros_like(g))
    seqs = documents(B, T, cu)
    zero = torch.zeros(len(seqs), D, dtype=torch.float64)
    start = zero if initial is None else initial.detach().double().cpu()
    out = {n: torch.zeros_like(x) for n in ("h", "before", "h_abs", "h_steps", "dx", "dg", "dx_abs", "dx_steps", "dg_bound")}
    final, final_bound, dinit, dinit_bound = (torch.zeros_like(zero) for _ in range(4))
    for b, lo, hi, d in seqs:
        h, H, W = start[d], start[d].abs(), torch.zeros(D, dtype=torch.float64)
        for t in range(lo, hi):
            out["before"][b, t] = h
            W = a[b, t] * (W + cost[b, t] * H)
            h, H = torch.where(a[b, t] == 0, torch.zeros_like(h), a[b, t] * h) + x[b, t], a[b, t] * H + x[b, t].abs()
            out["h"][b, t], out["h_abs"][b, t], out["h_steps"][b, t] = h, H, W
        final[d], final_bound[d] = h, U * (20 * H + W)
    res = {"h": (out["h"], U * (20 * out["h_abs"] + out["h_steps"])), "final": (final, final_bound)}
    if dh is None:
        return res
    dh = dh.detach().double().cpu()
    for b, lo, hi, d in seqs:
        mu = zero[d] if dfinal is None else dfinal.detach().double().cpu()[d]
        M, W = mu.abs(), torch.zeros(D, dtype=torch.float64)
        for t in range(hi - 1, lo - 1, -1):
            lam, L = dh[b, t] + mu, dh[b, t].abs() + M
            out["dx"][b, t], out["dx_abs"][b, t], out["dx_steps"][b, t] = lam, L, W
            before, B_ = out["before"][b, t].abs(), out["h_abs"][b, t - 1] if t > lo else start[d].abs()
            steps = out["h_steps"][b, t - 1] if t > lo else torch.zeros(D, dtype=torch.float64)
            out["dg"][b, t] = lam * a[b, t] * out["before"][b, t]
            out["dg_bound"][b, t] = a[b, t] * U * ((20 * L + W) * B_ + L * (20 * B_ + steps) + (4 + cost[b, t]) * L * B_)
            W = a[b, t] * (W + cost[b, t] * L)
            mu, M = a[b, t] * lam, a[b, t] * L
        dinit[d], dinit_bound[d] = mu, U * (20 * M + W)
    res["dx"] = (out["dx"], U * (20 * out["dx_abs"] + out["dx_steps"]))
    res["dg"] = (out["dg"], out["dg_bound"])
    res["dinitial"] = (dinit, dinit_bound)
    return res


def _rows(t):
    return None if t is None else t.detach().double().cpu().reshape(-1, t.shape[-1])


def _vector(v, N):
    return torch.ones(N, dtype=torch.float64) if v is None else v.detach().double().cpu() if torch.is_tensor(v) else torch.full((N,), float(v), dtype=torch.float64)


# A sum of N products over a row's threads takes at most 16 roundings in a thread, ten over its lanes and warps (32 in order); its root
# halves them; the power -1/2 takes four, the products around it six.
ROW = 64


def residual_norm(x, residual, weight, scale, eps, dy=None, dstream=None):
    shape, N = x.shape, x.shape[-1]
    stream_half = torch.finfo(residual.dtype).eps / 2 + U
    x, r0, dy, ds = _rows(x), _rows(residual), _rows(dy), _rows(dstream)
    w, c = _vector(weight, N), _vector(scale, N)
    r, r_abs = r0 + c * x, r0.abs() + (c * x).abs()
    inv = (r.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = r * inv
    back = lambda t: t.reshape(shape)
    # the sum is rounded once or twice (a fused product); its error is one of the sum, not of the terms, and passes through the norm
    near = 2 * U * (r_abs * inv + n.abs() * (r_abs * r.abs()).mean(-1, keepdim=True) * inv.square())
    res = {"stream": (back(r), back(2 * U * r_abs)), "y": (back(n * w), back(w.abs() * (near + ROW * U * n.abs())))}
    if dy is None and ds is None:
        return res
    dy, ds = torch.zeros_like(r) if dy is None else dy, torch.zeros_like(r) if ds is None else ds
    v = dy * w
    s = (v * n).mean(-1, keepdim=True)
    dr = ds + inv * (v - n * s)
    # the backward's n comes from the stream as stored: half a step of that type off, in the product and in the mean
    n_off = stream_half * n.abs() + near
    s_abs = (v * n).abs().mean(-1, keepdim=True)
    dr_off = inv * (n_off * s.abs() + n.abs() * (v.abs() * n_off).mean(-1, keepdim=True) + ROW * U * (v.abs() + n.abs() * s_abs)) + U * ds.abs()
    R = r.shape[0]
    depth = (R + 64) * U
    res["dresidual"] = (back(dr), back(dr_off))
    res["dx"] = (back(dr * c), back((dr_off + U * dr.abs()) * c.abs()))
    res["dweight"] = ((dy * n).sum(0), (dy.abs() * n_off).sum(0) + (depth + ROW * U) * (dy * n).abs().sum(0))
    res["dscale"] = ((dr * x).sum(0), (dr_off * x.abs()).sum(0) + depth * (dr * x).abs().sum(0))
    return res


def gated_norm(x, gate, weight, residual, scale, activation, eps, dout=None):
    shape, N = x.shape, x.shape[-1]
    x, z, r, dout = _rows(x), _rows(gate), _rows(residual), _rows(dout)
    w, c = _vector(weight, N), _vector(scale, N)
    inv = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = x * inv
    if z is None:
        act, slope, cost, slope_abs = torch.ones_like(x), torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    else:
        sig = torch.sigmoid(z)
        act = z * sig if activation == "silu" else sig
        slope = sig * (1 + z * (1 - sig)) if activation == "silu" else sig * (1 - sig)
        # terms of the slope by their absolute values: 1 - sig is formed from sig, whose error is one of sig
        slope_abs = sig * (1 + z.abs() * (1 + sig)) if activation == "silu" else sig * (1 + sig)
        cost = 16 + 2 * z.abs()                      # the exponential's product with log2 e, itself, the quotient, the products
    y = c * n * w * act
    out = y if r is None else r + y
    back = lambda t: t.reshape(shape)
    res = {"out": (back(out), back(U * ((ROW + cost) * y.abs() + 2 * out.abs())))}
    if dout is None:
        return res
    v = c * dout * w * act
    s = (v * n).mean(-1, keepdim=True)
    s_off = ((ROW + cost) * (v * n).abs()).mean(-1, keepdim=True)
    res["dx"] = (back(inv * (v - n * s)), back(U * inv * ((ROW + cost) * v.abs() + n.abs() * (s_off + 2 * ROW * s.abs()))))
    res["dgate"] = (back(c * dout * n * w * slope), back(U * (c * dout * n * w).abs() * (ROW + cost) * slope_abs))
    depth = x.shape[0] + 64 + ROW
    S, S_off = (dout * n * act).sum(0), U * ((depth + cost) * (dout * n * act).abs()).sum(0)
    res["dweight"], res["dscale"] = (c * S, c.abs() * S_off), (w * S, w.abs() * S_off)
    return res
