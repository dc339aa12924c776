"""The expert and few-row kernels where their sums are exact whatever the order, with derived bounds for
what is rounded: every tile height with the gated epilogue, joined parts, bias, salient columns and
column orders; the module, a token alone and in a batch."""
import pytest
import torch

from smoothquant import _lib, experts, ops
from test_gpu_experts import _ids, plain_experts
from w4_cases import DT, HALF, gen, int_rows, int_weight, values

pytestmark = pytest.mark.gpu


def whole_weight(shape, unit, D, g):
    """Weights that 4 bits hold exactly: multiples -7 .. 7 of `unit` (a power of two), a 7 in every
    eighth column, so that each row's group of 32 columns or more has the scale `unit`."""
    w = torch.randint(-7, 8, shape, generator=g, device="cuda")
    w[..., ::8] = 7
    return (w.double() * unit).to(D)


def salient_columns(w, p, unit, g):
    """A share p of the odd columns (those of 7 stay in the groups), with half units in them: exact there,
    between two codes anywhere else, and below their groups' maxima."""
    K = w.shape[-1]
    if not p:
        return None
    odd = torch.arange(1, K, 2, device="cuda")
    sal = odd[torch.randperm(len(odd), generator=g, device="cuda")[:int(p * K)]]
    half = torch.randint(-7, 7, (*w.shape[:-1], len(sal)), generator=g, device="cuda").double() + 0.5
    w[..., sal] = (half * unit).to(w.dtype)
    return sal


def check_exact(w, wq, G, sal, D):
    for e in range(w.shape[0]):
        assert torch.equal(ops.dequant_weight(ops.pack_weight(w[e], wq, 4, G, sal)), w[e])


def gated(u, I, act):
    """(act(gate) * up, the bound of one evaluation in fp32 and one rounding) for exact gate and up.
    silu: expf within 1 step, an addition, a division, a product: under 8 half steps of the value.
    gelu: 1 + erf(t) for t < 0 cancels, so its error is absolute: 2 steps of erff, the rounding of t
    (|t erf'(t)| < 0.43 of a half step) and of the addition, times |gate / 2| |up|; then the same 8.
    Results below the normal range of fp32 (|gate| > 87) or of D are off by a step of its least."""
    gate, up = u[:, :I], u[:, I:]
    a = gate * torch.sigmoid(gate) if act == "silu" else 0.5 * gate * torch.special.erfc(-gate * 0.5 ** 0.5)
    want = a * up
    tol = 8 * 2.0 ** -24 * want.abs() + 2.0 ** -126 * (1 + up.abs()) * (1 + gate.abs())
    if act == "gelu":
        tol = tol + 4 * 2.0 ** -24 * gate.abs() * up.abs()
    return want, tol


def rounded(tol, want, D):
    return tol * (1 + HALF[D]) + HALF[D] * want.abs() + torch.finfo(D).smallest_normal * HALF[D] * 2


# sizes around the pieces of a tile; then 2048 rows and more per expert on average, where tiles of 256
# rows are the rule's own choice: one of them whole rounds of workgroups and a split rest
RAGGED = [0, 1, 63, 64, 65, 127, 0, 129, 192, 193, 255, 256, 257, 320, 513]


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("sizes,I,K,G,height", [
    (RAGGED, 141, 1152, 64, 256), (RAGGED, 48, 192, 32, 256), (RAGGED, 141, 1152, 32, 128),
    ([2500, 1800], 203, 1152, 64, None), ([2500, 1800], 72, 320, 32, None), ([4300], 4000, 1088, 64, None)])
def test_gated_tiles(sizes, I, K, G, height, act, dt, monkeypatch):
    if height:
        monkeypatch.setenv("SQMP_EXPERT_ROWS", str(height))
        _lib.reload_knobs()
    D, g = DT[dt], gen(I + K)
    E, T = len(sizes), sum(sizes)
    ids = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(sizes, device="cuda"))
    ids = ids[torch.randperm(T, generator=g, device="cuda")].view(-1, 1)
    codes, scales = int_weight((E, 2 * I, K), G, D, g)
    scales = scales / 64                                      # gates of a few units
    pe = experts.pack_expert_codes(codes, scales, G, gated=True)
    r = experts.plan_routes(ids, torch.ones(T, 1, device="cuda"), E)
    x = int_rows(T, K, D, g)
    u = plain_experts(x, values(codes, scales, G), r, False)
    want, tol = gated(u, I, act)
    h = experts.expert_linear(x, pe, r, act=act).double()
    assert h.shape == (T, I) and ((h - want).abs() <= rounded(tol, want, D)).all()
    # rows in expert order: the same products
    assert torch.equal(experts.expert_linear(x[r.rows.long()], pe, r, act=act, rows="slot").double(), h)


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("wq,p", [("per_group_unsorted", 0.05), ("per_group", 0.05), ("per_group", 0.0)])
@pytest.mark.parametrize("sizes,I,K,G,height", [
    (RAGGED, 72, 1216, 64, 256), (RAGGED, 40, 320, 32, 128), ([2100, 2200], 96, 704, 64, None)])
def test_gated_tiles_with_salient_columns(sizes, I, K, G, height, wq, p, dt, monkeypatch):
    if height:
        monkeypatch.setenv("SQMP_EXPERT_ROWS", str(height))
        _lib.reload_knobs()
    D, g = DT[dt], gen(I + K)
    E, T = len(sizes), sum(sizes)
    ids = torch.repeat_interleave(torch.arange(E, device="cuda"), torch.tensor(sizes, device="cuda"))
    ids = ids[torch.randperm(T, generator=g, device="cuda")].view(-1, 1)
    w = whole_weight((E, 2 * I, K), 2.0 ** -6, D, g)
    sal = salient_columns(w, p, 2.0 ** -6, g)
    check_exact(w, wq, G, sal, D)
    pe = experts.pack_experts(w, wq, G, sal, gated=True)
    assert pe.S == (0 if sal is None else len(sal))
    r = experts.plan_routes(ids, torch.ones(T, 1, device="cuda"), E)
    x = int_rows(T, K, D, g)
    want, tol = gated(plain_experts(x, w.double(), r, False), I, "silu")
    h = experts.expert_linear(x, pe, r, act="silu").double()
    assert ((h - want).abs() <= rounded(tol, want, D)).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("wq,p", [("per_group", 0.05), ("per_group_unsorted", 0.1), ("per_group", 0.0),
                                  ("per_channel", 0.03)])
@pytest.mark.parametrize("T,E,k,N,K,G,by_slot", [(37, 4, 2, 72, 200, 32, False), (37, 4, 2, 72, 200, 32, True),
                                                 (500, 3, 2, 203, 1200, 64, False), (300, 2, 1, 96, 320, 64, True),
                                                 (5, 3, 1, 40, 128, 64, False)])
def test_quantized_orders_exact(T, E, k, N, K, G, by_slot, wq, p, dt):
    """Column orders of every expert's own and salient columns, few rows and tiles: bit for bit."""
    D, g = DT[dt], gen(T + N)
    w = whole_weight((E, N, K), 2.0 ** -2, D, g)
    sal = salient_columns(w, p, 2.0 ** -2, g)
    check_exact(w, wq, G, sal, D)
    pe = experts.pack_experts(w, wq, G, sal)
    r = experts.plan_routes(_ids(T, k, E, g, 0.2), torch.ones(T, k, device="cuda"), E)
    x = int_rows(T * k if by_slot else T, K, D, g)
    z = experts.expert_linear(x, pe, r, rows="slot" if by_slot else "token")
    n = int(r.offsets[-1])
    assert torch.equal(z[:n], plain_experts(x, w.double(), r, by_slot).float().to(D))


@pytest.mark.parametrize("dt", ["fp16", "bf16"])
@pytest.mark.parametrize("M", [33, 64])
@pytest.mark.parametrize("N,K,G,p", [(22501, 192, 64, 0.0), (22504, 1088, 32, 0.0), (22501, 1088, 64, 0.03),
                                     (22528, 2048, 128, 0.0), (22498, 2112, 32, 0.05)])
def test_wide_weights_of_many_rows_with_bias(N, K, G, p, M, dt):
    """More than 32 rows of a wide weight run on the tiles: bias, salient columns, parts along K."""
    D, g = DT[dt], gen(N + K)
    w = whole_weight((1, N, K), 2.0 ** -2, D, g)
    sal = salient_columns(w, p, 2.0 ** -2, g)
    check_exact(w, "per_group_unsorted", G, sal, D)
    pw = ops.pack_weight(w[0], "per_group_unsorted", 4, G, sal)
    x = int_rows(M, K, D, g)
    bias = (torch.randint(-200, 201, (N,), generator=g, device="cuda").double() / 4).to(D)
    y = x.double() @ w[0].double().T
    assert torch.equal(ops.gemv(x, pw), y.float().to(D))
    want = (y + bias.double()).float().to(D)
    assert torch.equal(ops.gemv(x, pw, bias), want)
    a = ops.pack_rows(x, pw.amap, pw.Kp, pw.salient, pw.S, pw.S_pad)
    assert torch.equal(ops.gemv(a, pw, bias, packed=True), want)
    # the same rows on the few-row kernel (a narrower weight): the same sums
    few = ops.pack_weight(w[0][:1000].contiguous(), "per_group_unsorted", 4, G, sal)
    assert torch.equal(ops.gemv(x, few, bias[:1000]), want[:, :1000])


class FusedExperts(torch.nn.Module):
    """What W4A4Experts takes over: two 3-D parameters and an activation."""
    def __init__(self, gate_up, down, act):
        super().__init__()
        self.gate_up_proj, self.down_proj = torch.nn.Parameter(gate_up), torch.nn.Parameter(down)
        self.act_fn = act


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("aq,p", [(None, 0.0), (None, 0.05), ("per_token", 0.0), ("per_token", 0.05)])
@pytest.mark.parametrize("T", [3, 70, 400])
def test_module(T, aq, p, dt):
    """W4A4Experts of weights and rows that 4 bits hold exactly: gate and up sums are exact, so h is the
    same bits for a token alone (few rows) and in its batch (tiles), and the output is the same within
    the additions of the second product; without activation quantization also against 64 bits."""
    D, g = DT[dt], gen(T)
    E, k, H, I, G = 4, 2, 320, 88, 64
    gu, dn = whole_weight((E, 2 * I, H), 2.0 ** -6, D, g), whole_weight((E, H, I), 2.0 ** -4, D, g)
    sal = salient_columns(gu, p, 2.0 ** -6, g)
    imp = torch.zeros(H)
    if p:
        imp[sal.cpu()] = 1 + torch.arange(len(sal), dtype=torch.float32)
    mod = experts.W4A4Experts.from_float(FusedExperts(gu, dn, torch.nn.SiLU()), "per_group_unsorted", aq, imp, p, 4, G)
    assert (mod.gate_up_salient is None) == (p == 0) and (p == 0 or set(mod.gate_up_salient.tolist()) == set(sal.tolist()))
    x = torch.randint(-7, 8, (T, H), generator=g, device="cuda").to(D)
    x[:, 0] = 7                                               # (a quantizer's scale of 1)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices
    wt = torch.rand(T, k, generator=g, device="cuda")
    y = mod(x, ids, wt)
    up, down, maps = mod.packed()
    r = experts.plan_routes(ids, wt, E)
    h = experts.expert_linear(x, up, r, act="silu")
    u = plain_experts(x, gu.double(), r, False)
    want, tol = gated(u, I, "silu")
    assert ((h.double() - want).abs() <= rounded(tol, want, D)).all()
    hq = mod._quant(h.clone(), down, maps[1])
    s, z64 = (plain_experts(t, m, r, True) for t, m in ((hq.abs(), dn.double().abs()), (hq, dn.double())))
    # the second product's additions (chains of at most I / 4 + 64), its rounding, the weighted sum's
    # two terms, the output's rounding
    tiny = torch.finfo(D).smallest_normal * HALF[D] * 2
    dz = (I / 4 + 65) * 2.0 ** -23 * s + HALF[D] * z64.abs() * (1 + 2.0 ** -8) + tiny
    sl, wd = r.slots.view(T, k).long(), wt.double()[..., None]
    y64 = (z64[sl] * wd).sum(1)
    bound = (dz[sl] * wd).sum(1) * (1 + 2.0 ** -8) + (k + 1) * 2.0 ** -24 * (z64[sl].abs() * wd).sum(1)
    bound = bound + HALF[D] * (y64.abs() + bound) + tiny
    assert ((y.double() - y64).abs() <= bound).all()
    for t in {0, T // 2, T - 1}:
        ra = experts.plan_routes(ids[t:t + 1], wt[t:t + 1], E)
        ha = experts.expert_linear(x[t:t + 1], up, ra, act="silu")
        assert torch.equal(ha[ra.slots.long()], h[sl[t]])     # the very rows of the batch
        alone = mod(x[t:t + 1], ids[t:t + 1], wt[t:t + 1])
        assert ((alone.double() - y64[t]).abs() <= bound[t]).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("T", [1, 8, 13])
@pytest.mark.parametrize("E,N,K,G", [(64, 512, 320, 64), (8, 4102, 192, 32), (3, 11006, 1088, 64), (40, 864, 200, 8),
                                     (2, 4096, 704, 128)])
def test_few_rows_of_many_blocks(E, N, K, G, T, act, dt):
    """Experts of a few rows: on either side of 1024 blocks of 32 weight rows, from which on workgroups have
    4 waves; up to 8 rows of an expert, and more."""
    D, g = DT[dt], gen(N + T)
    codes, scales = int_weight((E, N, K), G, D, g)
    scales = scales / 64 if act else scales
    pe = experts.pack_expert_codes(codes, scales, G, gated=act is not None)
    ids = torch.randint(0, E, (T, 1), generator=g, device="cuda")
    ids[T // 2:] = 1                                          # an expert of most of the tokens
    r = experts.plan_routes(ids, torch.ones(T, 1, device="cuda"), E)
    x = int_rows(T, K, D, g)
    u = plain_experts(x, values(codes, scales, G), r, False)
    z = experts.expert_linear(x, pe, r, act=act)
    if act is None:
        assert torch.equal(z, u.float().to(D))
    else:
        want, tol = gated(u, N // 2, act)
        assert ((z.double() - want).abs() <= rounded(tol, want, D)).all()
