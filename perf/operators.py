"""Performance cases of the operators that stand around the Triadic GDN core in a block: the per-channel gated recurrence and its decode
step, and the norms before and after a block.

    listed()            the named cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, made from the seed
    run(state)          one pass: through the package's entry points where `own` is true, in elementary torch operations otherwise
    exact(case, seed)   the outputs of that pass in 64 bits, from the definitions
    work(case)          bytes and FLOPs of one pass that no implementation can do without

A case is a dict of plain values.  `kind` selects the operator and the direction:

    scan_train     gated_scan_call, forward and backward:  h[t] = exp(g[t]) h[t-1] + x[t] per channel
    scan_prefill   gated_scan_call without gradients; the final state is handed out for the decode that follows
    scan_decode    gated_scan_decode, one token per sequence on a resident f32 state
    residual       residual_norm_call:  stream = residual + scale x,  y = rmsnorm(stream) weight
    gated          gated_norm_call:  y = rmsnorm(x) weight act(gate),  or  residual + scale y

`strided`: the inputs are slices of wider rows, as a fused projection leaves them.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def _scan(kind, B, T, D, x="bf16", g="f32", docs="", states=False, strided=False):
    return {"kind": kind, "B": B, "T": T, "D": D, "x": x, "g": g, "docs": docs, "states": states, "strided": strided}


def _residual(B, T, N, x="bf16", stream="bf16", scale="", train=True, strided=False):
    return {"kind": "residual", "B": B, "T": T, "N": N, "x": x, "stream": stream, "scale": scale, "train": train, "strided": strided}


def _gated(B, T, H, N, x="bf16", gate="silu", stream="", scale="", train=True, strided=False):
    return {"kind": "gated", "B": B, "T": T, "H": H, "N": N, "x": x, "gate": gate, "stream": stream, "scale": scale, "train": train,
            "strided": strided}


def listed():
    cases = {
        # a short batch of a small model, where launches and host work are what counts
        "scan_small": _scan("scan_train", 2, 256, 512),
        # the training step of a layer of width 2048, gates in 16 bits like the rest
        "scan_train": _scan("scan_train", 8, 4096, 2048, g="bf16"),
        # documents of lognormal length packed into one long row, every one with a state of its own handed in and out
        "scan_packed": _scan("scan_train", 1, 131072, 1024, docs="lognormal:2048", states=True),
        # a channel count and a length that no tile divides, all in 32 bits
        "scan_odd": _scan("scan_train", 3, 1000, 333, x="f32"),
        # inference over prompts, both operands slices of a fused projection
        "scan_prefill": _scan("scan_prefill", 4, 4096, 4096, x="f16", states=True, strided=True),
        # one user, and a full batch of them
        "scan_decode_one": _scan("scan_decode", 1, 1, 4096, g="bf16"),
        "scan_decode_batch": _scan("scan_decode", 512, 1, 4096),
        # before a block while decoding: one token of each of 32 sequences
        "residual_decode": _residual(32, 1, 4096, train=False),
        # before a block while training: residual stream in 32 bits, a learned scale per channel
        "residual_train": _residual(8, 4096, 4096, stream="f32", scale="channel"),
        # after the core of the headline training step: 32 heads of 128, the gate a slice of a projection
        "gated_heads": _gated(8, 8192, 32, 128, strided=True),
        # after a block of odd width, into the residual stream
        "gated_odd": _gated(3, 1000, 1, 2001, x="f16", gate="sigmoid", stream="f16", scale="channel"),
        # after the core while one user decodes
        "gated_decode": _gated(1, 1, 32, 128, train=False),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["scan_train", "scan_train", "scan_train", "scan_prefill", "scan_decode", "residual", "residual", "gated", "gated"])
    x = rng.choice(["bf16", "bf16", "f16", "f32"])
    strided = rng.random() < 0.3
    if kind.startswith("scan"):
        g = rng.choice([x, "f32"])
        D = _log_int(rng, 1, 8192)
        if rng.random() < 0.6:                           # widths of real layers are mostly multiples of 64
            D = 64 * max(1, D // 64)
        if kind == "scan_decode":
            return _scan(kind, _log_int(rng, 1, 512), 1, D, x, g, strided=strided)
        tokens = _log_int(rng, 1, max(1, min(131072, (1 << 25) // D)))
        if rng.random() < 0.4:
            docs = rng.choice(["equal:%d" % max(1, min(tokens, _log_int(rng, 1, 64))), "lognormal:%d" % _log_int(rng, 20, 4000)])
            return _scan(kind, 1, tokens, D, x, g, docs, rng.random() < 0.5, strided)
        B = min(tokens, _log_int(rng, 1, 16))
        return _scan(kind, B, tokens // B, D, x, g, "", rng.random() < 0.5, strided)
    stream = rng.choice([x, "f32"])
    scale = rng.choice(["", "number", "channel"])
    train = rng.random() < 0.7
    if kind == "residual":
        N = _log_int(rng, 1, 16384)
        if rng.random() < 0.6:
            N = 64 * max(1, N // 64)
        tokens = _log_int(rng, 1, max(1, min(131072, (1 << 25) // N)))
        B = min(tokens, _log_int(rng, 1, 32))
        return _residual(B, tokens // B, N, x, stream, scale, train, strided)
    heads = rng.random() < 0.5                           # a norm per head, or over the whole row
    H = _log_int(rng, 1, 32) if heads else 1
    N = rng.choice([64, 128, 128, 256, 96, 80, 33]) if heads else _log_int(rng, 1, 16384)
    tokens = _log_int(rng, 1, max(1, min(131072, (1 << 25) // (H * N))))
    B = min(tokens, _log_int(rng, 1, 32))
    if rng.random() < 0.5:
        stream = scale = ""
    return _gated(B, tokens // B, H, N, x, rng.choice(["silu", "silu", "sigmoid", ""]), stream, scale, train, strided)


def _offsets(case):
    T = case["T"]
    how, n = case["docs"].split(":")
    if how == "equal":
        n = int(n)
        return [i * T // n for i in range(n + 1)]
    rng, cu = np.random.default_rng(31), [0]
    while cu[-1] < T:
        cu.append(min(T, cu[-1] + max(1, int(round(float(rng.lognormal(math.log(int(n)), 1.0)))))))
    return cu


class _State:
    pass


def prepare(case, seed):
    s = _State()
    s.case = case
    kind, B, T = case["kind"], case["B"], case["T"]
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev)
    x_type = TYPES[case["x"]]

    def rows(values, dtype):
        """The values in the type, as a tensor of its own or as the middle of wider rows."""
        values = values.to(dtype)
        if not case["strided"]:
            return values
        n = values.shape[-1] * (values.shape[-2] if values.dim() == 4 else 1)
        wide = torch.zeros(B, T, 2 * n + 64, dtype=dtype, device=dev)
        view = wide[..., n:2 * n].view(values.shape) if values.dim() == 4 else wide[..., n:2 * n]
        return view.copy_(values)

    if kind.startswith("scan"):
        D = case["D"]
        rate = 10.0 ** (-3.0 * torch.rand(D, generator=gen, device=dev))     # memories of one to a thousand tokens
        s.x = rows(randn(B, T, D), x_type)
        s.g = rows(-torch.nn.functional.softplus(randn(B, T, D)) * rate, TYPES[case["g"]])
        s.cu = torch.tensor(_offsets(case), dtype=torch.int32, device=dev) if case["docs"] else None
        sequences = s.cu.numel() - 1 if case["docs"] else B
        if kind == "scan_decode":
            s.resident = randn(B, D)
            return s
        s.initial = randn(sequences, D) if case["states"] else None
        if kind == "scan_train":
            s.dh = randn(B, T, D).to(x_type)
            s.dfinal = randn(sequences, D) if case["states"] else None
            for t in (s.x, s.g, s.initial):
                if t is not None:
                    t.requires_grad_()
        return s
    N = case["N"]
    shape = (B, T, N) if kind == "residual" or case["H"] == 1 else (B, T, case["H"], N)
    s.x = rows(randn(*shape), x_type)
    s.weight = (1.0 + 0.1 * randn(N)).to(x_type)
    out_type = TYPES[case["stream"]] if case["stream"] else x_type
    s.scale = {"": None, "number": 0.7071, "channel": (0.5 + 0.1 * randn(N)).to(x_type)}[case["scale"]]
    s.residual = (2.0 * randn(*shape)).to(out_type) if case["stream"] else None
    if kind == "gated":
        s.gate = rows(randn(*shape), x_type) if case["gate"] else None
    if case["train"]:
        s.dy = randn(*shape).to(out_type if kind == "gated" else x_type)
        if kind == "residual":
            s.dstream = randn(*shape).to(out_type)
        for t in _leaves(s):
            t.requires_grad_()
    return s


def _leaves(s):
    """What the pass is differentiated in, in the order of the gradients among its outputs."""
    names = {"scan_train": ("x", "g", "initial"), "residual": ("x", "residual", "weight", "scale"),
             "gated": ("x", "gate", "weight", "residual", "scale")}[s.case["kind"]]
    return [t for t in (getattr(s, n) for n in names) if torch.is_tensor(t)]


def run(s):
    kind = s.case["kind"]
    if kind == "scan_train":
        out = (_own_scan if own else _plain_scan_train)(s)
    elif kind == "scan_prefill":
        out = (_own_prefill if own else _plain_prefill)(s)
    elif kind == "scan_decode":
        out = (_own_decode if own else _plain_decode)(s)
    else:
        call = (_own_residual if own else _plain_residual) if kind == "residual" else (_own_gated if own else _plain_gated)
        if not s.case["train"]:
            with torch.no_grad():
                return call(s)
        y = call(s)
        grads = (s.dy, s.dstream) if kind == "residual" else (s.dy,)
        out = (*(t.detach() for t in y), *torch.autograd.grad(y, _leaves(s), grads))
    return out


# ---- through the package ----------------------------------------------------------------------------------------------
def _own_scan(s):
    from cute_triadic_gdn_b200 import gated_scan_call
    if s.initial is None:
        h = gated_scan_call(s.x, s.g, s.cu)
        return (h.detach(), *torch.autograd.grad(h, (s.x, s.g), s.dh))
    h, final = gated_scan_call(s.x, s.g, s.cu, initial_state=s.initial, output_final_state=True)
    return (h.detach(), final.detach(), *torch.autograd.grad((h, final), (s.x, s.g, s.initial), (s.dh, s.dfinal)))


def _own_prefill(s):
    from cute_triadic_gdn_b200 import gated_scan_call
    with torch.no_grad():
        return gated_scan_call(s.x, s.g, s.cu, initial_state=s.initial, output_final_state=True)


def _own_decode(s):
    from cute_triadic_gdn_b200 import gated_scan_decode
    with torch.no_grad():
        return gated_scan_decode(s.x, s.g, s.resident), s.resident


def _own_residual(s):
    from cute_triadic_gdn_b200 import residual_norm_call
    return residual_norm_call(s.x, s.residual, s.weight, scale=s.scale, eps=EPS)


def _own_gated(s):
    from cute_triadic_gdn_b200 import gated_norm_call
    return (gated_norm_call(s.x, s.gate, s.weight, residual=s.residual, scale=s.scale, activation=s.case["gate"] or "silu", eps=EPS),)


# ---- the plain forms: elementary operations in 32 bits, rounded once at the end ----------------------------------------
def _solve(a, x):
    """h[t] = a[t] h[t-1] + x[t] along axis 1 from zero, by doubling: after the step of width s every h[t] holds the sum over the 2s
    tokens up to t and a[t] the product of their decays.  Overwrites a and x."""
    width, T = 1, x.shape[1]
    while width < T:
        x = torch.cat([x[:, :width], x[:, width:] + a[:, width:] * x[:, :-width]], 1)
        a = torch.cat([a[:, :width], a[:, width:] * a[:, :-width]], 1)
        width *= 2
    return x


def _decays(g):
    """exp(g), formed in 64 bits: near one, an error that leans to one side adds up over the thousand tokens that a state remembers."""
    return torch.exp(g.double()).float()


def _bounds(s):
    """(batch row, first token, last token) of every sequence, as index tensors."""
    B, T = s.x.shape[:2]
    if s.cu is None:
        rows = torch.arange(B, device=s.x.device)
        return rows, torch.zeros_like(rows), torch.full_like(rows, T - 1)
    cu = s.cu.long()
    return torch.zeros_like(cu[:-1]), cu[:-1], cu[1:] - 1


def _plain_forward(s):
    rows, first, last = _bounds(s)
    a, x = _decays(s.g), s.x.float().clone()
    if s.initial is not None:
        x[rows, first] += a[rows, first] * s.initial
    inside = a.clone()
    inside[rows, first] = 0.0                            # nothing comes into a sequence from the token before it
    h = _solve(inside, x)
    return a, h, h[rows, last]


def _plain_prefill(s):
    with torch.no_grad():
        _, h, final = _plain_forward(s)
        return h.to(s.x.dtype), final


def _plain_scan_train(s):
    with torch.no_grad():
        rows, first, last = _bounds(s)
        a, h, final = _plain_forward(s)
        before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
        before[rows, first] = 0.0 if s.initial is None else s.initial.detach()
        dh = s.dh.float().clone()
        if s.dfinal is not None:
            dh[rows, last] += s.dfinal
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)       # exp(g[t+1]), and zero behind a sequence's end
        after[rows, last] = 0.0
        lam = _solve(after.flip(1), dh.flip(1)).flip(1)
        mu = lam * a
        out = (h.to(s.x.dtype), lam.to(s.x.dtype), (mu * before).to(s.g.dtype))
        return out if s.initial is None else (out[0], final, *out[1:], mu[rows, first])


def _plain_decode(s):
    with torch.no_grad():
        s.resident.copy_(_decays(s.g[:, 0]) * s.resident + s.x[:, 0].float())
        return s.resident[:, None].to(s.x.dtype), s.resident


def _plain_residual(s):
    stream = s.x.float() if s.scale is None else s.x.float() * (s.scale.float() if torch.is_tensor(s.scale) else s.scale)
    stream = s.residual.float() + stream
    y = stream * torch.rsqrt((stream * stream).mean(-1, keepdim=True) + EPS) * s.weight.float()
    return y.to(s.x.dtype), stream.to(s.residual.dtype)


def _plain_gated(s):
    x = s.x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s.weight.float()
    if s.gate is not None:
        z = s.gate.float()
        y = y * ((z if s.case["gate"] == "silu" else 1.0) / (1.0 + torch.exp(-z)))
    if s.residual is None:
        return ((y if s.scale is None else y * (s.scale.float() if torch.is_tensor(s.scale) else s.scale)).to(s.x.dtype),)
    if s.scale is not None:
        y = y * (s.scale.float() if torch.is_tensor(s.scale) else s.scale)
    return ((s.residual.float() + y).to(s.residual.dtype),)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "scan_decode":
            state = s.g[:, 0].double().exp().mul(s.resident.double()).add(s.x[:, 0].double())
            return state.unsqueeze(1), state
        if case["kind"].startswith("scan"):
            return _exact_scan(s)
        return _exact_residual(s) if case["kind"] == "residual" else _exact_gated(s)


def _exact_scan(s):
    """Token by token, all channels of all batch rows at once."""
    B, T, D = s.x.shape
    cu = s.cu.tolist() if s.cu is not None else [0, T]
    begins, ends = {t: d for d, t in enumerate(cu[:-1])}, {t - 1: d for d, t in enumerate(cu[1:])}
    pick = (lambda states, d: states) if s.cu is None else (lambda states, d: states[d:d + 1])
    a = s.g.detach().double().exp().transpose(0, 1).contiguous()           # (T, B, D)
    x = s.x.detach().double().transpose(0, 1).contiguous()
    h, finals = torch.empty_like(x), []
    state = torch.zeros(B, D, dtype=torch.float64, device=x.device)
    for t in range(T):
        if t in begins:
            state = torch.zeros_like(state) if s.initial is None else pick(s.initial.detach(), begins[t]).double().clone()
        state = torch.addcmul(x[t], a[t], state, out=h[t])
        if t in ends:
            finals.append(state)
    final = torch.cat(finals)
    if s.case["kind"] == "scan_prefill":
        return h.transpose(0, 1), final
    lam, dinits = s.dh.double().transpose(0, 1).contiguous(), []
    dg = torch.empty_like(a)
    for t in range(T - 1, -1, -1):
        if t in ends:
            if s.dfinal is not None:
                lam[t] += pick(s.dfinal, ends[t])
        else:
            lam[t].addcmul_(a[t + 1], lam[t + 1])
        if t in begins:
            dinits.append(a[t] * lam[t])
            if s.initial is None:
                dg[t] = 0.0
            else:
                torch.mul(dinits[-1], pick(s.initial.detach(), begins[t]).double(), out=dg[t])
        else:
            torch.mul(lam[t], h[t - 1], out=dg[t]).mul_(a[t])
    out = (h.transpose(0, 1), lam.transpose(0, 1), dg.transpose(0, 1))
    return out if s.initial is None else (out[0], final, *out[1:], torch.cat(dinits[::-1]))


def _by_rows(tensors, body, columns):
    """body over slices of rows: the results of `columns` rows-wise put together, those behind them added up."""
    N = tensors[0].shape[-1]
    flat = [None if t is None else t.detach().reshape(-1, N) for t in tensors]
    step, parts, sums = max(1, (1 << 25) // N), [], None
    for lo in range(0, flat[0].shape[0], step):
        got = body(*[None if t is None else t[lo:lo + step].double() for t in flat])
        parts.append(got[:columns])
        sums = list(got[columns:]) if sums is None else [u + v for u, v in zip(sums, got[columns:])]
    return [torch.cat(p).reshape(tensors[0].shape) for p in zip(*parts)], sums


def _factors(s):
    N = s.x.shape[-1]
    one = torch.ones(N, dtype=torch.float64, device=s.x.device)
    return s.weight.detach().double(), one * (1.0 if s.scale is None else s.scale.detach().double() if torch.is_tensor(s.scale) else s.scale)


def _exact_residual(s):
    w, c = _factors(s)
    train = s.case["train"]

    def body(x, residual, dy, dstream):
        r = residual + c * x
        inv = (r.square().mean(-1, keepdim=True) + EPS).pow(-0.5)
        n = r * inv
        if not train:
            return n * w, r
        v = dy * w
        dr = dstream + inv * (v - n * (v * n).mean(-1, keepdim=True))
        return n * w, r, dr * c, dr, (dy * n).sum(0), (dr * x).sum(0)

    rows, sums = _by_rows([s.x, s.residual, s.dy if train else None, s.dstream if train else None], body, 4 if train else 2)
    if not train:
        return tuple(rows)
    return (*rows, sums[0], *([sums[1]] if torch.is_tensor(s.scale) else []))


def _exact_gated(s):
    w, c = _factors(s)
    train, silu = s.case["train"], s.case["gate"] == "silu"

    def body(x, z, residual, dy):
        inv = (x.square().mean(-1, keepdim=True) + EPS).pow(-0.5)
        n = x * inv
        if z is None:
            act, slope = torch.ones_like(x), torch.zeros_like(x)
        else:
            sig = torch.sigmoid(z)
            act = z * sig if silu else sig
            slope = sig * (1 + z * (1 - sig)) if silu else sig * (1 - sig)
        y = c * n * w * act
        out = y if residual is None else residual + y
        if not train:
            return (out,)
        u = c * dy * w * act
        dx = inv * (u - n * (u * n).mean(-1, keepdim=True))
        return out, dx, c * dy * n * w * slope, (c * dy * n * act).sum(0), (dy * n * w * act).sum(0)

    rows, sums = _by_rows([s.x, s.gate, s.residual, s.dy if train else None], body, 3 if train else 1)
    if not train:
        return tuple(rows)
    return (rows[0], rows[1], *([rows[2]] if s.gate is not None else []), sums[0], *([s.dy.double()] if s.residual is not None else []),
            *([sums[1]] if torch.is_tensor(s.scale) else []))


# ---- floors ---------------------------------------------------------------------------------------------------------------
def work(case):
    kind, B, T = case["kind"], case["B"], case["T"]
    xb = SIZE[case["x"]]
    if kind.startswith("scan"):
        n, gb = B * T * case["D"], SIZE[case["g"]]
        if kind == "scan_decode":
            return {"bytes": n * (2 * xb + gb + 8), "flops": 3 * n}
        sequences = len(_offsets(case)) - 1 if case["docs"] else B
        state = 4 * sequences * case["D"]
        if kind == "scan_prefill":
            return {"bytes": n * (2 * xb + gb) + state * (2 if case["states"] else 1), "flops": 3 * n}
        # forward: x, g -> h; backward: x, g, dh -> dx, dg; a state in and out and the gradients of both
        return {"bytes": n * (5 * xb + 3 * gb) + (4 * state if case["states"] else 0), "flops": 10 * n}
    n = B * T * case["N"] * case.get("H", 1)
    sb = SIZE[case["stream"]] if case["stream"] else 0
    learned = case["scale"] == "channel"
    if kind == "residual":
        forward = n * (2 * xb + 2 * sb)
        # dy, dstream, stream (and x where the scale is learned) -> the gradient of the stream (and of x where it is another)
        backward = n * (xb + 3 * sb + (xb if learned else 0) + (0 if case["scale"] == "" and sb == xb else xb))
        return {"bytes": forward + (backward if case["train"] else 0), "flops": n * (22 if case["train"] else 7)}
    gate = xb if case["gate"] else 0
    forward = n * (xb + gate + (2 * sb if sb else xb))
    backward = n * (2 * xb + 2 * gate + (sb or xb))
    return {"bytes": forward + (backward if case["train"] else 0), "flops": n * (32 if case["train"] else 12)}
