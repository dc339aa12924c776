"""Routing, the products grouped by expert and their combination against their definitions in 64
bits: whole numbers and exact sums bit for bit."""
import pytest
import torch

from smoothquant import experts, ops
from w4_cases import DT, HALF, gen, int_rows, int_weight, tolerance, values

pytestmark = pytest.mark.gpu
INF = float("inf")


# ------------------------------------------------------------------ routing
def plain_plan(ids, E):
    """offsets, rows, slots of ids (CPU, int64)."""
    flat = ids.reshape(-1).tolist()
    per = [[f for f, e in enumerate(flat) if e == x] for x in range(E)]
    rows = [f for p in per for f in p]
    offsets = [0]
    for p in per:
        offsets.append(offsets[-1] + len(p))
    slots = [-1] * len(flat)
    for s, f in enumerate(rows):
        slots[f] = s
    return offsets, rows + [-1] * (len(flat) - len(rows)), slots


def plain_route(logits, k, normalize):
    l = logits.double().cpu()
    T, E = l.shape
    ids = torch.full((T, k), -1, dtype=torch.long)
    w = torch.zeros(T, k, dtype=torch.float64)
    key = torch.where(l.isnan(), torch.full_like(l, INF), l)
    for t in range(T):
        # NaN before +inf before the rest; ties: the lowest index
        order = sorted(range(E), key=lambda e: (not bool(l[t, e].isnan()), -float(key[t, e]), e))
        sel = [e for e in order[:k] if float(key[t, e]) != -INF]
        if not sel:
            continue
        top = l[t, sel[0]]
        ex = torch.exp(l[t] - top)
        den = ex[sel].sum() if normalize else ex.sum()
        for j, e in enumerate(sel):
            ids[t, j], w[t, j] = e, ex[e] / den
    return ids, w


def check_routing(r, ids, E):
    offsets, rows, slots = plain_plan(ids, E)
    assert r.offsets.tolist() == offsets
    assert r.rows.tolist() == rows
    assert r.slots.tolist() == slots


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 5, 5), (255, 64, 6), (256, 256, 16),
                                   (257, 200, 3), (600, 65, 8), (2, 256, 1)])
def test_route(T, E, k, normalize, dt):
    g = gen(T + E)
    logits = (2 * torch.randn(T, E, generator=g, device="cuda")).to(DT[dt])
    if T > 4:
        logits[1] = -INF                     # padding: nothing to choose
        logits[2, 1:] = -INF                 # one expert left
        logits[3] = 1.5                      # ties all along
        logits[4, : E // 2] = -INF
    r = experts.route(logits, k, normalize)
    ids, w = plain_route(logits, k, normalize)
    assert torch.equal(r.ids.cpu().long(), ids)
    # exp of a rounded difference d (|d| <= 32: 2^-24 * 32 of the value, + 2 steps of expf), the
    # sum of E such terms and one division
    tol = (32 * 2 + 4 + E) * 2.0 ** -24 * w + 1e-38
    assert ((r.weights.cpu().double() - w).abs() <= tol).all()
    check_routing(r, ids, E)


def test_route_special_values():
    nan = float("nan")
    logits = torch.tensor([[nan, 1.0, 2.0, INF], [0.0, -0.0, 0.0, -0.0], [INF, INF, 0.0, -INF],
                           [-INF, nan, -INF, -INF], [3e38, -3e38, 0.0, 1.0]], device="cuda")
    r = experts.route(logits, 3)
    assert r.ids.tolist() == [[0, 3, 2], [0, 1, 2], [0, 1, 2], [1, -1, -1], [0, 3, 2]]
    assert r.weights[0].isnan().all() and r.weights[2].isnan().all()
    assert torch.allclose(r.weights[1].cpu(), torch.full((3,), 1 / 3))
    assert r.weights[3].isnan().tolist() == [True, False, False]
    assert r.weights[4].tolist() == [1.0, 0.0, 0.0]
    check_routing(r, r.ids.cpu(), 4)


@pytest.mark.parametrize("T,E,k", [(70001, 17, 4), (131072 + 300, 64, 2), (5000, 1, 1), (3000, 256, 3)])
def test_route_many_blocks(T, E, k):
    """Up to 512 blocks of 256 tokens add up the counts before them themselves, more take a scan."""
    g = gen(3)
    logits = torch.randn(T, E, generator=g, device="cuda").to(torch.bfloat16)
    logits[torch.rand(T, generator=g, device="cuda") < 0.3] = -INF
    r = experts.route(logits, k)
    v, idx = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    ids = torch.where(v[:, :k] > -INF, idx[:, :k], -1)
    assert torch.equal(r.ids.long(), ids)
    key = torch.where(ids < 0, E, ids).reshape(-1)
    skey, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(skey, torch.arange(E + 1, device="cuda"))
    assert torch.equal(r.offsets.long(), offsets)
    n = int(offsets[-1])
    assert torch.equal(r.rows[:n].long(), order[:n]) and (r.rows[n:] == -1).all()
    back = torch.full_like(order, -1)
    back[order[:n]] = torch.arange(n, device="cuda")
    assert torch.equal(r.slots.long(), back)


@pytest.mark.parametrize("idt", [torch.int32, torch.int64, torch.int16])
def test_plan_of_given_ids(idt):
    g = gen(5)
    T, E, k = 300, 12, 3
    ids = torch.randint(-2, E + 2, (T, k), generator=g, device="cuda").to(idt)  # some out of range
    ids[7] = 4                                                                  # the same thrice
    w = torch.rand(T, k, generator=g, device="cuda").half()
    r = experts.plan_routes(ids, w, E)
    check_routing(r, ids.cpu(), E)
    assert torch.equal(r.weights, w.float())
    if idt == torch.int64:
        ids[0] = 2 ** 32 + 1                  # would wrap to expert 1
        assert experts.plan_routes(ids, w, E).slots[:k].tolist() == [-1] * k


def test_routing_strides_empty_and_refusals():
    logits = torch.randn(10, 40, device="cuda")
    a = experts.route(logits[:, 3:11], 2)
    b = experts.route(logits[:, 3:11].contiguous(), 2)
    c = experts.route(logits[:, 3:11].t().contiguous().t(), 2)
    d = experts.route(logits[4:5, :8].expand(10, 8), 2)
    for n in ("ids", "weights", "offsets", "rows", "slots"):
        assert torch.equal(getattr(a, n), getattr(b, n)) and torch.equal(getattr(a, n), getattr(c, n))
    assert torch.equal(d.ids, experts.route(logits[4:5, :8], 2).ids.expand(10, 2))
    e = experts.route(logits[:0, :8], 2)
    assert e.offsets.tolist() == [0] * 9 and e.rows.numel() == 0 and e.tokens == 0
    p = experts.plan_routes(torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                            torch.empty(0, 2, device="cuda"), 8)
    assert p.offsets.tolist() == [0] * 9
    for bad in (lambda: experts.route(logits[:, :4], 5), lambda: experts.route(logits[0], 1),
                lambda: experts.route(logits, 0), lambda: experts.route(logits.repeat(1, 7), 2),
                lambda: experts.route(logits, 17), lambda: experts.route(logits.double(), 2),
                lambda: experts.plan_routes(logits, logits, 8),
                lambda: experts.plan_routes(a.ids, a.weights[:, :1], 8),
                lambda: experts.plan_routes(a.ids, a.weights, 257)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ products
def _ids(T, k, E, g, dropped=0.0):
    """Distinct experts per token, some of them liked better; some pairs go nowhere."""
    l = torch.randn(T, E, generator=g, device="cuda") + 1.5 * torch.randn(E, generator=g, device="cuda")
    ids = l.topk(k, dim=1).indices.to(torch.int32)
    if dropped:
        ids[torch.rand(T, k, generator=g, device="cuda") < dropped] = -1
    return ids


def plain_experts(x, w, r, by_slot):
    """z in 64 bits, rows in expert order, of the pairs that go somewhere."""
    off, rows = r.offsets.tolist(), r.rows.long()
    z = []
    for e in range(r.num_experts):
        at = torch.arange(off[e], off[e + 1], device=x.device)
        z.append((x[at] if by_slot else x[rows[at] // r.top_k]).double() @ w[e].T)
    return torch.cat(z)


SHAPES = [(1, 8, 2, 64, 128, 64), (9, 3, 1, 33, 100, 32), (130, 5, 3, 96, 256, 64),
          (300, 40, 6, 50, 192, 64), (40, 2, 2, 300, 1000, 8), (1100, 4, 2, 264, 384, 128),
          (500, 2, 1, 130, 256, 32), (256, 1, 1, 257, 128, 64), (777, 3, 3, 512, 640, 640),
          (260, 256, 4, 16, 128, 128), (330, 3, 1, 512, 2048, 128), (64, 8, 2, 96, 4096, 64), (300, 2, 1, 64, 64, 64),
          (700, 3, 2, 288, 1344, 64), (9, 4, 2, 64, 448, 32), (400, 2, 1, 130, 4160, 128)]


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("by_slot", [False, True])
@pytest.mark.parametrize("T,E,k,N,K,G", SHAPES)
def test_products_exact_sums(T, E, k, N, K, G, by_slot, dt):
    D, g = DT[dt], gen(T + N)
    codes, scales = int_weight((E, N, K), G, D, g)
    pe = experts.pack_expert_codes(codes, scales, G)
    ids = _ids(T, k, E, g, 0.1)
    r = experts.plan_routes(ids, torch.ones(T, k, device="cuda"), E)
    x = int_rows(T * k if by_slot else T, K, D, g)
    out = torch.full((T * k, N), 7.0, device="cuda", dtype=D)
    z = experts.expert_linear(x, pe, r, rows="slot" if by_slot else "token", out=out)
    assert z is out
    n = int(r.offsets[-1])
    want = plain_experts(x, values(codes, scales, G), r, by_slot).float().to(D)
    assert torch.equal(z[:n], want)
    assert (z[n:] == 7.0).all()                       # rows behind the last pair: as they were


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("height", [64, 128, 256])
def test_tile_heights_agree(height, dt, monkeypatch):
    """Every tile height, on segments of 0, 1, and the sizes around a tile's, with salient columns and
    an odd number of outputs: the same bits."""
    from smoothquant import _lib
    monkeypatch.setenv("SQMP_EXPERT_ROWS", str(height))
    _lib.reload_knobs()
    D, g = DT[dt], gen(height)
    sizes = [0, 1, 63, 64, 65, 127, 0, 129, 192, 193, 255, 256, 257, 320, 513]
    ids = torch.repeat_interleave(torch.arange(len(sizes), device="cuda"),
                                  torch.tensor(sizes, device="cuda"))
    ids = ids[torch.randperm(len(ids), generator=g, device="cuda")].view(-1, 1)
    E, T, N, K, G = len(sizes), len(ids), 283, 1152, 64   # (18 stages: up to two parts)
    codes, scales = int_weight((E, N, K), G, D, g)
    pe = experts.pack_expert_codes(codes, scales, G)
    r = experts.plan_routes(ids, torch.ones(T, 1, device="cuda"), E)
    x = int_rows(T, K, D, g)
    want = plain_experts(x, values(codes, scales, G), r, False).float().to(D)
    assert torch.equal(experts.expert_linear(x, pe, r), want)
    # whole 8-column outputs and salient columns: small whole numbers quantize exactly
    w = torch.randint(-7, 8, (E, 48, 256), generator=g, device="cuda").to(D)
    w[:, :, :4] = 7
    sal = torch.tensor([5, 9, 200], device="cuda")
    w[:, :, sal] *= 3
    ps = experts.pack_experts(w, "per_group_unsorted", 64, sal)
    x = int_rows(T, 256, D, g)
    w_hat = torch.stack([ops.dequant_weight(ops.pack_weight(w[e], "per_group_unsorted", 4, 64, sal))
                         for e in range(E)]).double()
    z = experts.expert_linear(x, ps, r).double()
    y = plain_experts(x, w_hat, r, False)
    assert (z - y).abs().max() <= HALF[D] * y.abs().max() * 1.01


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("T,E,k,I,K,G", [(4, 8, 2, 40, 128, 64), (150, 4, 2, 257, 320, 64),
                                         (700, 6, 1, 128, 512, 128)])
def test_gated(T, E, k, I, K, G, act, dt):
    D, g = DT[dt], gen(I)
    codes = torch.randint(-7, 8, (E, 2 * I, K), generator=g, device="cuda", dtype=torch.int8)
    ng = (K + G - 1) // G
    scales = (0.02 * torch.rand(E, 2 * I, ng, generator=g, device="cuda") + 0.002).to(D)
    pe = experts.pack_expert_codes(codes, scales, G, gated=True)
    r = experts.plan_routes(_ids(T, k, E, g), torch.ones(T, k, device="cuda"), E)
    x = torch.randn(T, K, generator=g, device="cuda").to(D)
    h = experts.expert_linear(x, pe, r, act=act)
    w = values(codes, scales, G)
    y = plain_experts(x, w, r, False)
    gate, up = y[:, :I], y[:, I:]
    a = torch.nn.functional.silu(gate) if act == "silu" else torch.nn.functional.gelu(gate)
    want = a * up
    # errors of the two sums (tolerance without the rounding), through |act'| <= 1.13 and the
    # product; 8 steps of the fp32 activation itself; one rounding to D
    s = plain_experts(x.abs(), w.abs(), r, False) * ((K / 4 + 65) * 2.0 ** -23)
    tol = 1.13 * s[:, :I] * (up.abs() + s[:, I:]) + (a.abs() + 1.13 * s[:, :I]) * s[:, I:] \
        + 8 * 2.0 ** -24 * (want.abs() + gate.abs() * 2.0 ** -20) + HALF[D] * want.abs() * 1.01 \
        + torch.finfo(D).smallest_normal * HALF[D] * 2
    assert h.shape == (T * k, I)
    assert ((h.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("wq,p,gated", [("per_channel", 0.0, True), ("per_group", 0.1, False),
                                        ("per_group", 0.0, True), ("per_tensor", 0.05, False),
                                        ("per_group_unsorted", 0.0, False)])
@pytest.mark.parametrize("by_slot", [False, True])
def test_quantized_experts(wq, p, gated, by_slot, dt):
    """Weights quantized here, every expert in a column order of its own, salient columns."""
    D, g = DT[dt], gen(2)
    T, E, k, N, K, G = 37, 4, 2, 64, 200, 32
    w = (0.02 * torch.randn(E, N, K, generator=g, device="cuda")).to(D)
    sal = torch.randperm(K, generator=g, device="cuda")[:int(p * K)] if p else None
    pe = experts.pack_experts(w, wq, G, sal, gated)
    r = experts.plan_routes(_ids(T, k, E, g, 0.2), torch.ones(T, k, device="cuda"), E)
    x = torch.randn(T * k if by_slot else T, K, generator=g, device="cuda").to(D)
    z = experts.expert_linear(x, pe, r, act="silu" if gated else None, rows="slot" if by_slot else "token")
    w_hat = torch.stack([ops.dequant_weight(ops.pack_weight(w[e], wq, 4, G, sal)) for e in range(E)])
    y = plain_experts(x, w_hat.double(), r, by_slot)
    n = y.shape[0]
    if gated:
        y = torch.nn.functional.silu(y[:, :N // 2]) * y[:, N // 2:]
    # 1 % of the largest output: an element of another column or expert is off by far more
    err = (z[:n].double() - y).abs().max() / y.abs().max()
    assert err < (3e-3 if dt == "fp16" else 1e-2)


def test_products_strides_empty_and_refusals():
    g = gen(1)
    D = torch.float16
    codes, scales = int_weight((3, 48, 128), 64, D, g)
    pe = experts.pack_expert_codes(codes, scales, 64)
    pg = experts.pack_expert_codes(codes, scales, 64, gated=True)
    r = experts.plan_routes(_ids(6, 2, 3, g), torch.ones(6, 2, device="cuda"), 3)
    x = int_rows(6, 128, D, g)
    want = experts.expert_linear(x, pe, r)
    wide = torch.zeros(6, 136, device="cuda", dtype=D)
    wide[:, :128] = x
    assert torch.equal(experts.expert_linear(wide[:, :128], pe, r), want)
    odd = torch.zeros(6, 129, device="cuda", dtype=D)
    odd[:, 1:] = x
    assert torch.equal(experts.expert_linear(odd[:, 1:], pe, r), want)
    assert torch.equal(experts.expert_linear(x.t().contiguous().t(), pe, r), want)
    one = x[2:3].expand(6, 128)
    assert torch.equal(experts.expert_linear(one, pe, r), experts.expert_linear(one.contiguous(), pe, r))
    nothing = experts.plan_routes(torch.full((6, 2), -1, device="cuda"), torch.ones(6, 2, device="cuda"), 3)
    out = torch.full((12, 48), 3.0, device="cuda", dtype=D)
    assert (experts.expert_linear(x, pe, nothing, out=out) == 3.0).all()
    none = experts.plan_routes(torch.empty(0, 2, dtype=torch.int64, device="cuda"),
                               torch.empty(0, 2, device="cuda"), 3)
    assert experts.expert_linear(x[:0], pe, none).shape == (0, 48)
    assert experts.combine(want[:0], none).shape == (0, 48)
    for bad in (lambda: experts.expert_linear(x, pe, r, act="silu"),
                lambda: experts.expert_linear(x, pg, r),
                lambda: experts.expert_linear(x, pg, r, act="relu"),
                lambda: experts.expert_linear(x, pe, r, rows="slot"),
                lambda: experts.expert_linear(x, pe, r, rows="row"),
                lambda: experts.expert_linear(x[:, :64], pe, r),
                lambda: experts.expert_linear(x, pe, r, out=out[:6]),
                lambda: experts.expert_linear(x, pe, experts.plan_routes(r.ids, r.weights, 4)),
                lambda: experts.combine(want[:6], r),
                lambda: experts.pack_expert_codes(codes, scales[:2], 64),
                lambda: experts.pack_expert_codes(codes[:, :47], scales[:, :47], 64, gated=True)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="dtype"):
        experts.expert_linear(x.float(), pe, r)


# ------------------------------------------------------------------ combine
@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("T,E,k,H", [(1, 4, 2, 8), (50, 8, 3, 513), (33, 16, 6, 1024), (5, 2, 1, 1),
                                     (9, 16, 16, 72)])
def test_combine(T, E, k, H, dt):
    D, g = DT[dt], gen(H)
    ids = _ids(T, min(k, E), E, g, 0.2)
    w = torch.rand(T, k, generator=g, device="cuda")
    r = experts.plan_routes(ids, w, E)
    z = torch.randn(T * k, H, generator=g, device="cuda").to(D)
    z[int(r.offsets[-1]):] = float("nan")                 # rows that no pair has
    y = experts.combine(z, r)
    sl = r.slots.view(T, k).long()
    terms = torch.where((sl >= 0)[..., None], z[sl.clamp(min=0)].double() * w.double()[..., None], 0.0)
    want = terms.sum(1)
    # k additions in fp32, one rounding to D
    tol = (k + 1) * 2.0 ** -24 * terms.abs().sum(1) + HALF[D] * want.abs() * 1.01 \
        + torch.finfo(D).smallest_normal * HALF[D] * 2
    assert ((y.double() - want).abs() <= tol).all()
    assert (y[(sl < 0).all(1)] == 0).all()
    out = torch.empty_like(y)
    assert experts.combine(z, r, out=out) is out and torch.equal(out, y)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("T", [1, 9, 200])
def test_block_captured_and_replayed(T):
    """Routing, both products and the combination as one block: captured once, replayed on other
    inputs with eager work between, against the eager block and the 64-bit one."""
    g = gen(T)
    D, E, k, H, I = torch.float16, 8, 2, 128, 96
    cu, su = int_weight((E, 2 * I, H), 64, D, g)
    cd, sd = int_weight((E, H, I), 32, D, g)
    up = experts.pack_expert_codes(cu, su / 64, 64, gated=True)
    down = experts.pack_expert_codes(cd, sd / 64, 32)

    def block(x, logits):
        r = experts.route(logits, k)
        h = experts.expert_linear(x, up, r, act="silu")
        return experts.combine(experts.expert_linear(h, down, r, rows="slot"), r), r

    x = torch.randn(T, H, generator=g, device="cuda").to(D)
    logits = torch.randn(T, E, generator=g, device="cuda")
    y0, r = block(x, logits)
    w = r.weights.double()
    wu, wd = values(cu, su / 64, 64), values(cd, sd / 64, 32)
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for j in range(k):
        for t in range(T):
            e = int(r.ids[t, j])
            u = x[t].double() @ wu[e].T
            want[t] += w[t, j] * ((torch.nn.functional.silu(u[:I]) * u[I:]) @ wd[e].T)
    assert ((y0.double() - want).norm() / want.norm()) < 2e-3   # two roundings to fp16 in a row
    xs, ls = x.clone(), logits.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, _ = block(xs, ls)
    for i in range(4):
        xs.copy_(x.roll(i, 1)), ls.copy_(logits.roll(i, 1))
        graph.replay()
        eager, _ = block(x.roll(i, 1), logits.roll(i, 1))
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
    assert torch.equal(block(x, logits)[0], y0)                 # the same bits again


def test_offsets_beyond_32_bits():
    """Operands and outputs of more than 4 GiB: rows and weights on either side of the border."""
    D, g = torch.float16, gen(8)
    # a weight whose codes take 4.3 GB
    N, K = 1_050_000, 8192
    codes = torch.randint(-8, 8, (N, K), generator=g, device="cuda", dtype=torch.int8)
    scales = torch.ones(N, K // 256, device="cuda", dtype=D)
    scales[::2] = 0.5
    pw = ops.pack_codes(codes, scales, 256)
    for M in (1, 20):
        x = int_rows(M, K, D, g)
        y = ops.gemv(x, pw)
        pick = torch.cat([torch.arange(64), torch.arange(N // 2, N // 2 + 64), torch.arange(N - 64, N)]).cuda()
        want = x.double() @ values(codes[pick], scales[pick], 256).T
        assert torch.equal(y[:, pick], want.float().to(D))
    del codes, scales, pw
    # rows in expert order, 4.9 GB of them; then the same rows picked by token
    T, K, N = 600_000, 4096, 40
    codes, scales = int_weight((3, N, K), 128, D, g)
    pe = experts.pack_expert_codes(codes, scales, 128)
    x = torch.randint(-4, 5, (T, K), generator=g, device="cuda", dtype=torch.int8).to(D)
    ids = torch.randint(0, 3, (T, 1), generator=g, device="cuda")
    r = experts.plan_routes(ids, torch.ones(T, 1, device="cuda"), 3)
    pick = torch.cat([torch.arange(50), torch.arange(T // 2, T // 2 + 50), torch.arange(T - 50, T)]).cuda()
    e_of = ids.view(-1)[r.rows.long()]
    w = values(codes, scales, 128)
    for by_slot in (True, False):
        z = experts.expert_linear(x, pe, r, rows="slot" if by_slot else "token")
        src = pick if by_slot else r.rows.long()[pick]
        want = torch.einsum("sk,snk->sn", x[src].double(), w[e_of[pick]])
        assert torch.equal(z[pick], want.float().to(D))
    y = experts.combine(z, r)
    assert torch.equal(y[r.rows.long()[pick]], z[pick])
