"""ops.gemv (few rows times a packed 4-bit weight) against its definition in 64 bits: bit for bit
where the sums are exact whatever their order, else within the accumulation's bound."""
import pytest
import torch

from smoothquant import ops
from smoothquant.fake_quant import W4A4Linear, use_gemv
from w4_cases import DT, gen, int_rows, int_weight, tolerance, values

pytestmark = pytest.mark.gpu


def _int_case(M, N, K, G, dt, seed):
    g = gen(seed)
    codes, scales = int_weight((N, K), G, dt, g)
    x = int_rows(M, K, dt, g)
    return x, codes, scales, ops.pack_codes(codes, scales, G)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 49, 64])
@pytest.mark.parametrize("N,K,G", [(32, 128, 64), (40, 192, 32), (257, 1000, 8), (1, 64, 64),
                                   (33, 1, 128), (96, 2304, 256), (2600, 256, 64), (22500, 192, 64),
                                   (64, 64, 64), (70, 448, 32), (40, 1344, 192)])
def test_exact_sums(M, N, K, G, dt):
    x, codes, scales, pw = _int_case(M, N, K, G, DT[dt], M * 1000 + N)
    want = (x.double() @ values(codes, scales, G).T).float().to(DT[dt])
    assert torch.equal(ops.gemv(x, pw), want)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("M,N,K,G", [(1, 4096, 4096, 128), (3, 500, 11008, 64), (64, 300, 2047, 32),
                                     (20, 1030, 100, 16)])
def test_random_values_and_bias(M, N, K, G, dt):
    D, g = DT[dt], gen(7)
    codes = torch.randint(-7, 8, (N, K), generator=g, device="cuda", dtype=torch.int8)
    scales = (0.01 * torch.rand(N, (K + G - 1) // G, generator=g, device="cuda") + 0.001).to(D)
    x = torch.randn(M, K, generator=g, device="cuda").to(D)
    bias = torch.randn(N, generator=g, device="cuda").to(D)
    y = ops.gemv(x, ops.pack_codes(codes, scales, G), bias)
    w = values(codes, scales, G)
    want = x.double() @ w.T + bias.double()
    # (+ the addition of the bias in fp32: half a step of the sum)
    tol = tolerance(x, w, want, D, extra=2.0 ** -24 * want.abs())
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("wq,p,G", [("per_group", 0.1, 64), ("per_channel", 0.0, 128),
                                    ("per_tensor", 0.05, 128), ("per_group_unsorted", 0.3, 32),
                                    ("per_group_mean3std", 0.02, 16)])
def test_packed_orders_and_salient_columns(dt, wq, p, G):
    """Weights packed in an order of their own, with exact salient columns: x in the columns' order
    and the operand of the activation quantizer's layout give the same bits."""
    D, g = DT[dt], gen(11)
    N, K, M = 72, 320, 5
    w = (torch.randn(N, K, generator=g, device="cuda") * 0.02).to(D)
    sal = torch.randperm(K, generator=g, device="cuda")[:int(p * K)] if p else None
    pw = ops.pack_weight(w, wq, 4, G, sal)
    x = torch.randn(M, K, generator=g, device="cuda").to(D)
    y = ops.gemv(x, pw)
    w_hat = ops.dequant_weight(pw).double()
    want = x.double() @ w_hat.T
    assert ((y.double() - want).abs() <= tolerance(x, w_hat, want, D)).all()
    a = ops.pack_rows(x, pw.amap, pw.Kp, pw.salient, pw.S, pw.S_pad)
    assert torch.equal(ops.gemv(a, pw, packed=True), y)


@pytest.mark.parametrize("dt", ["fp16", "fp32"])
def test_strides_and_alignment(dt):
    D = DT[dt]
    x, codes, scales, pw = _int_case(6, 64, 256, 64, D, 3)
    want = ops.gemv(x, pw)
    wide = torch.full((6, 320), 77.0, device="cuda", dtype=D)
    wide[:, 16:272] = x
    odd = torch.full((6, 259), 77.0, device="cuda", dtype=D)
    odd[:, 1:257] = x
    assert torch.equal(ops.gemv(wide[:, 16:272], pw), want)      # a row stride, aligned
    assert torch.equal(ops.gemv(odd[:, 1:257], pw), want)        # rows that are not 16-B aligned
    assert torch.equal(ops.gemv(x.t().contiguous().t(), pw), want)
    assert torch.equal(ops.gemv(wide[3:4, 16:272], pw), want[3:4])
    one = x[2:3].expand(6, 256)                                  # a row stride of 0
    assert torch.equal(ops.gemv(one, pw), want[2:3].expand(6, 64))
    assert torch.equal(ops.gemv(x.flip(0), pw), want.flip(0))
    bias = torch.arange(128, device="cuda").to(D)
    assert torch.equal(ops.gemv(x, pw, bias[::2]), ops.gemv(x, pw, bias[::2].contiguous()))


def test_rows_do_not_meet():
    """A row of NaN or infinity leaves the others' bits alone, and rows past M are never read into
    the result."""
    x, codes, scales, pw = _int_case(9, 48, 384, 128, torch.bfloat16, 5)
    want = ops.gemv(x, pw)
    bad = x.clone()
    bad[3] = float("nan")
    bad[7, 11] = float("inf")
    got = ops.gemv(bad, pw)
    keep = [0, 1, 2, 4, 5, 6, 8]
    assert torch.equal(got[keep], want[keep])
    assert got[3].isnan().all()
    nz = codes[:, 11] != 0
    assert not got[7][nz].isfinite().any() and torch.equal(got[7][~nz].isnan(), torch.ones(int((~nz).sum()), dtype=torch.bool, device="cuda"))


def test_empty_and_refusals():
    x, codes, scales, pw = _int_case(2, 32, 128, 64, torch.float16, 1)
    assert ops.gemv(x[:0], pw).shape == (0, 32)
    with pytest.raises(ValueError, match="at most 64"):
        ops.gemv(torch.zeros(65, 128, device="cuda", dtype=torch.float16), pw)
    with pytest.raises(ValueError, match="columns"):
        ops.gemv(x[:, :64], pw)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.gemv(x.float(), pw)
    with pytest.raises(RuntimeError, match="bias"):
        ops.gemv(x, pw, torch.zeros(31, device="cuda", dtype=torch.float16))
    w8 = ops.pack_weight(torch.randn(32, 128, device="cuda").half(), "per_group", 8, 64, None)
    with pytest.raises(ValueError, match="4-bit"):
        ops.gemv(x, w8)
    fine = ops.pack_weight(torch.randn(32, 128, device="cuda").half(), "per_group", 4, 4, None)
    with pytest.raises(ValueError, match="multiple of 8"):
        ops.gemv(x, fine)
    with pytest.raises(ValueError, match="scales"):
        ops.pack_codes(codes, scales, 32)


@pytest.mark.parametrize("M", [1, 40])
def test_captured_and_on_another_stream(M):
    x, codes, scales, pw = _int_case(M, 200, 1024, 128, torch.float16, 9)
    want = ops.gemv(x, pw)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert torch.equal(ops.gemv(x, pw), want)
    torch.cuda.current_stream().wait_stream(s)
    xs = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.gemv(xs, pw)
    for i in range(4):
        xs.copy_(x.roll(i, 1))
        graph.replay()
        eager = ops.gemv(x.roll(i, 1), pw)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
    # first used inside a capture: nothing of the capture is kept
    fresh = ops.pack_codes(codes, scales, 128)
    graph2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph2):
        y2 = ops.gemv(x, fresh)
    assert torch.equal(ops.gemv(x, fresh), want)
    graph2.replay()
    torch.cuda.synchronize()
    assert torch.equal(y2, want)


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("aq,wq,p", [("per_group", "per_group", 0.1), ("per_token", "per_channel", 0.0),
                                     ("per_tensor", "per_group", 0.05)])
def test_linear_module(dt, aq, wq, p):
    """W4A4Linear with kernel "gemv": the packed-order kernel's result (the same operands) within
    the accumulation's bound on few rows, its very bits on more."""
    D = DT[dt]
    torch.manual_seed(2)
    K, N = 256, 96
    lin = torch.nn.Linear(K, N).to("cuda", D)
    x0 = torch.randn(3, K, device="cuda").to(D)
    imp = x0.float().abs().mean(0).cpu()
    q = W4A4Linear.from_float(lin, weight_quant=wq, act_quant=aq, importance=imp, salient_prop=p,
                              group_size=32)
    pw = q.packed()
    for M in (1, 5, 64, 65):
        x = torch.randn(M, K, device="cuda").to(D)
        q.kernel = "fq"
        xa = x.clone()
        want = q(xa)
        q.kernel = "gemv"
        xb = x.clone()
        got = q(xb)
        assert torch.equal(xa, xb)            # the same in-place effect on the input
        if M > 64:
            q.kernel = "auto"
            assert torch.equal(got, q(x.clone()))
            continue
        a = ops.quant_act_fp(x.clone(), pw, aq, 4, 32)
        w = torch.cat([ops.dequant_weight_packed(pw), pw.wsal], 1).double()
        exact = a.double() @ w.T + q.bias.reshape(-1).double()
        tol = tolerance(a, w, exact, D, extra=2.0 ** -24 * exact.abs())
        assert ((got.double() - exact).abs() <= tol).all()
        # (fp32 layers on "fq" run split fp16 planes: 2^-21 of sum |a w|)
        tol2 = 2 * tol + (2.0 ** -21 * (a.double().abs() @ w.abs().T) if dt == "fp32" else 0)
        assert ((got.double() - want.double()).abs() <= tol2).all()


def test_linear_module_quantized_output_and_model_switch():
    torch.manual_seed(4)
    m = torch.nn.Sequential(torch.nn.Linear(128, 128), torch.nn.Linear(128, 64)).to("cuda", torch.float16)
    q0 = W4A4Linear.from_float(m[0], weight_quant="per_group", act_quant="per_group",
                               quantize_output=True, group_size=64)
    q1 = W4A4Linear.from_float(m[1], weight_quant="per_channel", act_quant="per_token")
    m = torch.nn.Sequential(q0, q1)
    x = torch.randn(2, 4, 128, device="cuda").half()
    assert use_gemv(m) == 2 and q0.kernel == q1.kernel == "gemv"
    y = m(x)
    assert y.shape == (2, 4, 64) and y.isfinite().all()
    assert use_gemv(m, False) == 2 and q0.kernel == q1.kernel == "auto"
    assert m(x[:0]).shape == (0, 4, 64)
