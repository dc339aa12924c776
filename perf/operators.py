"""Operators of serving with 4-bit weights, from one token to whole prompts: their plain forms
in elementary torch operations, and the calls a user makes of this framework's kernels.

  gemv     y[m] = D(W x[m] + b), W = D(code * scale) in groups along K, 1 .. 64 rows
           (a decoding step of a W4 linear)
  route    the k largest logits of every token (ties: the lowest index; a logit of -inf is never
           chosen), their softmax weights, and the stable order of the chosen (token, expert)
           pairs by expert
  experts  z[s] = D(W_e(s) x[row(s)]) over the pairs in expert order (ragged sizes per expert);
           gated: D(silu(gate) * up) of the two halves of W_e
  combine  y[t] = D(sum_j w[t, j] z[slot(t, j)])

`own` selects the framework's kernels; `run` takes what `prepare` gives either way.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token through a 4096 x 4096 projection in groups of 128: the latency of decoding
        dict(name="gemv_1", op="gemv", M=1, N=4096, K=4096, G=128, dtype="fp16", bias=False),
        # a small decoding batch through the gate projection of a 4096 / 11008 MLP, groups of 64
        dict(name="gemv_8", op="gemv", M=8, N=11008, K=4096, G=64, dtype="bf16", bias=False),
        # the most rows one call takes (many sequences, or drafted tokens), a down projection
        dict(name="gemv_64", op="gemv", M=64, N=4096, K=11008, G=128, dtype="fp16", bias=True),
        # odd sizes in fp32: K is no whole group, N no whole tile, rows not 16-byte aligned
        dict(name="gemv_odd", op="gemv", M=3, N=2051, K=2047, G=32, dtype="fp32", bias=True),
        # a decoding batch picks 2 of 8 experts
        dict(name="route_8", op="route", T=8, E=8, k=2, dtype="fp16", normalize=True, masked=0.0),
        # a batch of padded prompts (an eighth of the tokens are padding) picks 6 of 64
        dict(name="route_65537", op="route", T=65537, E=64, k=6, dtype="bf16", normalize=False,
             masked=0.125),
        # a decoding batch through gate and up of 8 experts (4096 / 11008), activation fused
        dict(name="experts_gate_up_8", op="experts", T=8, E=8, k=2, K=4096, N=11008, G=128,
             dtype="fp16", gated=True, slots=False),
        # a 2048-token prompt through the same
        dict(name="experts_gate_up_2048", op="experts", T=2048, E=8, k=2, K=4096, N=11008, G=128,
             dtype="fp16", gated=True, slots=False),
        # the way back down, rows already in expert order
        dict(name="experts_down_2048", op="experts", T=2048, E=8, k=2, K=11008, N=4096, G=128,
             dtype="bf16", gated=False, slots=True),
        # many small experts, ragged: 509 tokens pick 6 of 64
        dict(name="experts_ragged_509", op="experts", T=509, E=64, k=6, K=2048, N=1408, G=64,
             dtype="bf16", gated=True, slots=False),
        # the expert outputs of a decoding batch, and of prompts, back to their tokens
        dict(name="combine_8", op="combine", T=8, E=8, k=2, H=4096, dtype="fp16"),
        dict(name="combine_16384", op="combine", T=16384, E=64, k=6, H=2048, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gemv", "gemv", "route", "experts", "experts", "combine"])
    dt = rng.choice(["fp16", "bf16"])
    if op == "gemv":
        return dict(op=op, M=_log(rng, 1, 64), N=_log(rng, 64, 11008),
                    K=rng.choice([_log(rng, 64, 11008), 64 * _log(rng, 1, 172)]),
                    G=rng.choice([32, 64, 128, 256]), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    bias=rng.random() < 0.5)
    if op == "route":
        E = _log(rng, 2, 128)
        return dict(op=op, T=_log(rng, 1, 32768), E=E, k=rng.randint(1, min(E, 8)),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]), normalize=rng.random() < 0.5,
                    masked=rng.choice([0.0, 0.0, 0.125, 0.5]))
    if op == "combine":
        E = _log(rng, 2, 64)
        k, H = rng.randint(1, min(E, 6)), _log(rng, 64, 4096)
        return dict(op=op, T=_log(rng, 1, min(16384, (6 * 16384 * 2048) // (k * H))), E=E, k=k, H=H,
                    dtype=dt)
    E = _log(rng, 2, 64)
    k = rng.randint(1, min(E, 6))
    # all experts' weights together stay below those of 8 x 22016 x 4096
    K = rng.choice([_log(rng, 64, 4096), 64 * _log(rng, 1, 64)])
    gated = rng.random() < 0.5
    N = _log(rng, 64, max(65, min(8192, (1 << 29) // (E * K * (2 if gated else 1)))))
    return dict(op=op, T=_log(rng, 1, 1024), E=E, k=k, K=K, N=N, G=rng.choice([64, 128]),
                dtype=dt, gated=gated, slots=rng.random() < 0.5)


def _active(c):
    """Expected number of experts that at least one token picks."""
    return c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** c["T"])


def work(c):
    eb = 4 if c.get("dtype") == "fp32" else 2
    if c["op"] == "gemv":
        M, N, K = c["M"], c["N"], c["K"]
        ng = -(-K // c["G"])
        return {"bytes": N * K / 2 + eb * (N * ng + M * K + M * N + (N if c["bias"] else 0)),
                "flops": 2.0 * M * N * K}
    T, E, k = c["T"], c["E"], c["k"]
    if c["op"] == "route":
        return {"bytes": eb * T * E + 16.0 * T * k + 4 * (E + 1), "flops": 4.0 * T * E}
    if c["op"] == "combine":
        return {"bytes": eb * (T * k + T) * c["H"] + 8.0 * T * k, "flops": 2.0 * T * k * c["H"]}
    N = c["N"] * (2 if c["gated"] else 1)
    K = c["K"]
    x_rows = T * k if c["slots"] else T
    return {"bytes": _active(c) * (N * K / 2 + eb * N * (-(-K // c["G"]))) + eb * x_rows * K
            + eb * T * k * c["N"], "flops": 2.0 * T * k * N * K}


# ---------------------------------------------------------------------------------- inputs
def _codes(shape, g, dev):
    """4-bit codes in -7 .. 7, more of them near 0, as rounding to the group's maximum leaves."""
    a = torch.randint(-4, 4, shape, generator=g, device=dev, dtype=torch.int8)
    return a.add_(torch.randint(-3, 4, shape, generator=g, device=dev, dtype=torch.int8)).clamp_(-7, 7)


def _scales(shape, g, dev, dt):
    return (0.004 + 0.006 * torch.rand(shape, generator=g, device=dev)).to(dt)


def _rows(M, K, g, dev, dt):
    """Activations with a few outlier channels."""
    x = torch.randn(M, K, generator=g, device=dev)
    hot = torch.randint(0, K, (max(1, K // 64),), generator=g, device=dev)
    x[:, hot] *= 8.0
    return x.to(dt)


def _logits(c, g, dev):
    """Router logits: some experts are liked better, so that the loads are ragged."""
    T, E = c["T"], c["E"]
    l = torch.randn(T, E, generator=g, device=dev) + torch.randn(E, generator=g, device=dev)
    return l


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    st = {"case": c}
    if c["op"] == "gemv":
        M, N, K = c["M"], c["N"], c["K"]
        st["x"] = _rows(M, K, g, dev, dt)
        st["codes"] = _codes((N, K), g, dev)
        st["scales"] = _scales((N, -(-K // c["G"])), g, dev, dt)
        st["bias"] = torch.randn(N, generator=g, device=dev).to(dt) if c["bias"] else None
        if own:
            from smoothquant import ops
            st["w"] = ops.pack_codes(st.pop("codes"), st.pop("scales"), c["G"])
        return st
    logits = _logits(c, g, dev)
    if c["op"] == "route":
        logits = logits.to(dt)
        if c["masked"] > 0:
            pad = torch.rand(c["T"], generator=g, device=dev) < c["masked"]
            logits[pad] = float("-inf")
        st["logits"] = logits
        return st
    T, E, k = c["T"], c["E"], c["k"]
    wts, ids = torch.sort(logits, dim=1, descending=True, stable=True)
    ids = ids[:, :k].to(torch.int32).contiguous()
    wts = torch.softmax(wts[:, :k], dim=1).contiguous()
    if c["op"] == "combine":
        st["z"] = torch.randn(T * k, c["H"], generator=g, device=dev).to(dt)
    else:
        N = c["N"] * (2 if c["gated"] else 1)
        st["x"] = _rows(T * k if c["slots"] else T, c["K"], g, dev, dt)
        st["codes"] = _codes((E, N, c["K"]), g, dev)
        st["scales"] = _scales((E, N, -(-c["K"] // c["G"])), g, dev, dt)
    if own:
        from smoothquant import experts
        st["routing"] = experts.plan_routes(ids, wts, E)
        if c["op"] == "experts":
            st["w"] = experts.pack_expert_codes(st.pop("codes"), st.pop("scales"), c["G"],
                                                gated=c["gated"])
    else:
        flat = ids.reshape(-1).long()
        order = torch.sort(flat, stable=True)[1]
        st["order"], st["weights"] = order, wts
        st["slots"] = torch.empty_like(order).scatter_(0, order, torch.arange(T * k, device=dev))
        st["counts"] = torch.bincount(flat, minlength=E).tolist()
    return st


# ---------------------------------------------------------------------------------- one pass
def run(st):
    c = st["case"]
    if own:
        return _run_own(st, c)
    dt = DTYPES[c["dtype"]]
    if c["op"] == "gemv":
        y = st["x"].float() @ _w_hat(st["codes"], st["scales"], c["G"], torch.float32).T
        if st["bias"] is not None:
            y = y + st["bias"].float()
        return y.to(dt)
    if c["op"] == "route":
        return _route(st["logits"].float(), c)
    if c["op"] == "combine":
        z = st["z"].float()[st["slots"]].view(c["T"], c["k"], c["H"])
        return (z * st["weights"][:, :, None]).sum(1).to(dt)
    return _experts(st["x"], st["codes"], st["scales"], st["order"], st["counts"], c,
                    torch.float32).to(dt)


def _run_own(st, c):
    from smoothquant import experts, ops
    if c["op"] == "gemv":
        return ops.gemv(st["x"], st["w"], st["bias"])
    if c["op"] == "route":
        r = experts.route(st["logits"], c["k"], normalize=c["normalize"])
        return r.weights, r.ids, r.offsets, r.rows, r.slots
    if c["op"] == "combine":
        return experts.combine(st["z"], st["routing"])
    return experts.expert_linear(st["x"], st["w"], st["routing"],
                                 act="silu" if c["gated"] else None,
                                 rows="slot" if c["slots"] else "token")


def _w_hat(codes, scales, G, acc):
    """The weight the codes stand for, rounded to the scales' type, in `acc`."""
    s = scales.to(acc).repeat_interleave(G, dim=-1)[..., :codes.shape[-1]]
    return (codes.to(acc) * s).to(scales.dtype).to(acc)


def _experts(x, codes, scales, order, counts, c, acc):
    out, at = [], 0
    for e, n in enumerate(counts):
        if n == 0:
            continue
        idx = slice(at, at + n) if c["slots"] else order[at:at + n] // c["k"]
        y = x[idx].to(acc) @ _w_hat(codes[e], scales[e], c["G"], acc).T
        if c["gated"]:
            a, b = y[:, :c["N"]], y[:, c["N"]:]
            y = a / (1 + torch.exp(-a)) * b
        out.append(y)
        at += n
    return torch.cat(out)


def _route(l, c):
    """l: logits in the type the sums are held in."""
    T, E, k = c["T"], c["E"], c["k"]
    dev = l.device
    v, idx = torch.sort(l, dim=1, descending=True, stable=True)
    v, idx, top = v[:, :k], idx[:, :k], v[:, :1]
    sel = v != float("-inf")
    e = torch.where(sel, torch.exp(v - top), 0.0)
    den = e.sum(1, keepdim=True) if c["normalize"] else torch.exp(l - top).sum(1, keepdim=True)
    weights = torch.where(sel, e / den, 0.0).float()
    ids = torch.where(sel, idx, -1)
    key = torch.where(sel, idx, E).reshape(-1)
    skey, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(skey, torch.arange(E + 1, device=dev))
    at = torch.arange(T * k, device=dev)
    rows = torch.where(at < offsets[E], order, -1)
    slots = torch.where(key < E, torch.empty_like(order).scatter_(0, order, at), -1)
    i32 = torch.int32
    return weights, ids.to(i32), offsets.to(i32), rows.to(i32), slots.to(i32)


# ---------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits (one output element at a time is a dot
    product over K of the inputs and the weights' values; whole numbers have no such value)."""
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    c, f64 = case, torch.float64

    def values(codes, scales):
        col = torch.arange(codes.shape[1], device=codes.device) // c["G"]
        return codes.to(f64).mul_(scales.to(f64)[:, col]).to(scales.dtype).to(f64)

    if c["op"] == "gemv":
        y = torch.matmul(values(st["codes"], st["scales"]), st["x"].to(f64).T).T
        return y if st["bias"] is None else y + st["bias"].to(f64)[None]
    if c["op"] == "route":
        l = st["logits"].to(f64)
        top = l.max(dim=1, keepdim=True).values
        p = torch.exp(l - torch.where(torch.isinf(top), 0.0, top))
        chosen = torch.topk(p, c["k"], dim=1).values
        den = (chosen if c["normalize"] else p).sum(1, keepdim=True)
        return torch.where(den > 0, chosen / torch.where(den > 0, den, 1.0), 0.0), None, None, None, None
    if c["op"] == "combine":
        y = torch.zeros(c["T"], c["H"], dtype=f64, device=st["z"].device)
        for j in range(c["k"]):
            at = st["slots"].view(c["T"], c["k"])[:, j]
            y += st["weights"][:, j, None].to(f64) * st["z"][at].to(f64)
        return y
    z = torch.empty(c["T"] * c["k"], c["N"], dtype=f64, device=st["x"].device)
    at = 0
    for e, n in enumerate(st["counts"]):
        if n:
            w = values(st["codes"][e], st["scales"][e])
            src = torch.arange(at, at + n, device=z.device)
            x = st["x"][src if c["slots"] else torch.div(st["order"][src], c["k"], rounding_mode="floor")]
            y = torch.matmul(w, x.to(f64).T)
            if c["gated"]:
                y = torch.sigmoid(y[:c["N"]]) * y[:c["N"]] * y[c["N"]:]
            z[at:at + n] = y.T
        at += n
    return z
