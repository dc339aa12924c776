"""The expert calls in the company of the framework's other layers, and the calls around the tested
ones: buffers used again, overlapping ones, routings by hand."""
import pytest
import torch

from smoothquant import experts, ops
from smoothquant.fake_quant import W4A4Linear
from w4_cases import DT, gen, int_rows, int_weight, tolerance

pytestmark = pytest.mark.gpu


def _layers(n, K, N, D, **kw):
    """Sorted per_group layers of one input width, whose statistics and operands are kept per input."""
    torch.manual_seed(6)
    return [W4A4Linear.from_float(torch.nn.Linear(K, N).to("cuda", D), weight_quant="per_group",
                                  act_quant="per_group", group_size=64, **kw) for _ in range(n)]


@pytest.mark.parametrize("linked", [False, True])
def test_a_buffer_written_again_between_two_layers(linked):
    """combine / expert_linear into one buffer, a layer on it, again, another layer on it: the second
    layer quantizes the new contents."""
    from smoothquant.fake_quant import link_siblings
    D, g = torch.float16, gen(1)
    T, E, k, H = 24, 4, 2, 128
    a, b = _layers(2, H, 96, D)
    if linked:
        link_siblings(a, b)
    r = experts.route(torch.randn(T, E, generator=g, device="cuda"), k)
    z = [torch.randn(T * k, H, generator=g, device="cuda").to(D) for _ in range(2)]
    buf = torch.empty(T, H, device="cuda", dtype=D)
    a(experts.combine(z[0], r, out=buf))
    got = b(experts.combine(z[1], r, out=buf))
    assert torch.equal(got, b(buf.clone()))
    codes, scales = int_weight((E, H, 64), 64, D, g)
    pe = experts.pack_expert_codes(codes, scales, 64)
    x = [int_rows(T, 64, D, g) for _ in range(2)]
    buf = torch.empty(T * k, H, device="cuda", dtype=D)
    a(experts.expert_linear(x[0], pe, r, out=buf))
    got = b(experts.expert_linear(x[1], pe, r, out=buf))
    assert torch.equal(got, b(buf.clone()))


def test_copies_of_a_layer_after_its_original_is_gone(tmp_path):
    """Layers copied and saved after they ran on few rows, from a state dict too: each computes from its
    own weight (the original's is overwritten, then freed)."""
    import copy
    D = torch.float16
    src, = _layers(1, 128, 96, D)
    loaded, = _layers(1, 128, 96, D)
    loaded.load_state_dict(src.state_dict())
    x = torch.randn(3, 128, device="cuda").to(D)
    for q in (src, loaded):
        q.kernel = "gemv"
        want = q(x.clone())
        pw = q.packed()
        assert pw.gemv_args is not None
        f = str(tmp_path / "q.pt")
        torch.save(q, f)
        others = [copy.deepcopy(q), torch.load(f, weights_only=False), copy.deepcopy(pw)]
        for t in pw.gemv:
            t.zero_()
        assert torch.equal(q(x.clone()), q.bias.reshape(1, -1).expand(3, -1).to(D))   # (what a copy must not see)
        del q, pw
        a = ops.quant_act_fp(x, others[2], "per_group", 4, 64)
        y = ops.gemv(a, others[2], others[0].bias, packed=True)
        for got in (others[0](x.clone()), others[1](x.clone()), y):
            assert torch.equal(got, want)


@pytest.mark.parametrize("linked", [False, True])
def test_layers_first_used_in_a_capture(linked):
    """A prompt captured before any eager call, then a decoding step: the step does not take the
    operands that only the graph's replays write."""
    from smoothquant.fake_quant import link_siblings
    D = torch.float16
    warm, cold = _layers(2, 128, 96, D), _layers(2, 128, 96, D)
    if linked:
        link_siblings(*warm), link_siblings(*cold)
    x = torch.randn(300, 128, device="cuda").to(D)
    for q in warm:                                            # (the quantizers' workspaces)
        q(x)
    want = [q(x) for q in warm]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = [q(x) for q in cold]
    step = x[:3].clone()
    for a, b in zip(warm, cold):
        a.kernel = b.kernel = "gemv"
        assert torch.equal(b(step), a(step))
        a.kernel = b.kernel = "auto"
        assert torch.equal(b(step), a(step))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(y, want))
        assert all(torch.equal(q(x), w) for q, w in zip(cold, want))


def _captured(fn):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fn()
    return graph, y


@pytest.mark.parametrize("kernel", ["gemv", "auto"])
def test_graphs_of_decoding_steps_share_nothing(kernel):
    """Graphs of two batch sizes, captured one after the other without a warm-up on the capture's
    stream: replayed in the other order, in turns, and side by side on two streams."""
    D, g = torch.float16, gen(4)
    a, b = _layers(2, 256, 96, D)
    for q in (a, b):
        q.kernel = kernel
    ins = [torch.randn(M, 256, generator=g, device="cuda").to(D) for M in (1, 7)]
    want = [[(a(x.roll(i, 1)), b(x.roll(i, 1))) for x in ins] for i in range(4)]
    xs = [x.clone() for x in ins]
    graphs = [_captured(lambda x=x: (a(x), b(x))) for x in xs]

    def check(i, picks, streams=None):
        for p in picks:
            xs[p].copy_(ins[p].roll(i, 1))
        torch.cuda.synchronize()
        for n, p in enumerate(picks):
            with torch.cuda.stream(streams[n] if streams else torch.cuda.current_stream()):
                graphs[p][0].replay()
        torch.cuda.synchronize()
        for p in picks:
            for got, w in zip(graphs[p][1], want[i][p]):
                assert torch.equal(got, w)
    check(1, [1])                                             # the second graph before the first
    a(ins[0])
    check(2, [0, 1])
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        check(3, [0, 1], side)
        check(0, [1, 0], side)


def test_a_graph_does_not_take_statistics_from_outside_of_it():
    """A layer captured alone, after eager calls (and another capture) of its sibling on the same
    tensor: its graph computes its own statistics and operand of new contents."""
    D, g = torch.float16, gen(5)
    a, b = _layers(2, 128, 96, D)
    x = torch.randn(5, 128, generator=g, device="cuda").to(D)
    xs = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a(xs), b(xs)
        a.kernel = b.kernel = "gemv"
        a(xs), b(xs)
    torch.cuda.synchronize()
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, stream=s):
        ya = a(xs)
    with torch.cuda.graph(second, stream=s):
        yb = b(xs)
    for i in range(3):
        new = x.roll(i + 1, 1) * (1 + i)
        xs.copy_(new)
        second.replay()
        torch.cuda.synchronize()
        assert torch.equal(yb, b(new.clone()))
        first.replay()
        torch.cuda.synchronize()
        assert torch.equal(ya, a(new.clone()))


def test_siblings_captured_one_by_one():
    """Linked layers, each captured in a graph of its own on the same tensor: every graph computes its
    layer's output."""
    from smoothquant.fake_quant import link_siblings
    D, g = torch.float16, gen(6)
    a, b = _layers(2, 128, 96, D)
    link_siblings(a, b)
    x = torch.randn(300, 128, generator=g, device="cuda").to(D)
    a(x), b(x)
    xs = x.clone()
    a(xs)                                                     # (b's output of it is kept for b)
    graphs = [_captured(lambda q=q: q(xs)) for q in (a, b)]
    assert torch.equal(a(xs), a(x.clone()))                   # not the graph's, which has not run
    for i in range(3):
        new = x.roll(i + 1, 1)
        xs.copy_(new)
        for (graph, y), q in zip(reversed(graphs), (b, a)):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, q(new.clone()))


@pytest.mark.parametrize("p", [0.0, 0.05])
def test_graphs_of_expert_modules_side_by_side(p):
    """Two expert modules with salient columns of their own, captured without a warm-up, replayed on two
    streams at once."""
    import copy
    from test_gpu_mixtral import _model
    base = copy.deepcopy(_model(3).model.layers[0].mlp.experts).to("cuda", torch.float16)
    H, g = base.hidden_dim, gen(7)
    mods, ins = [], []
    for i in range(2):
        imp = torch.rand(H, generator=g, device="cuda").cpu()
        mods.append(experts.W4A4Experts.from_float(base, "per_channel", "per_token", imp, p, 4, 32))
        T = 40 + 30 * i
        ins.append((torch.randn(T, H, generator=g, device="cuda").half(),
                    torch.rand(T, base.num_experts, generator=g, device="cuda").topk(2, dim=1).indices,
                    torch.rand(T, 2, generator=g, device="cuda")))
    want = [m(*i) for m, i in zip(mods, ins)]
    graphs = [_captured(lambda m=m, i=i: m(*i)) for m, i in zip(mods, ins)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        torch.cuda.synchronize()
        for s, (graph, _y) in zip(side, reversed(graphs)):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_g, y), w in zip(graphs, want):
            assert torch.equal(y, w)


# ------------------------------------------------------------------ routings by hand
@pytest.mark.parametrize("T", [5, 300])
def test_router_weights_cast_by_the_caller(T):
    """routing.weights in the model's type, as a model's own router casts them, and strided: the sums
    of the converted weights."""
    D, g = torch.bfloat16, gen(T)
    E, k, H = 8, 2, 96
    r = experts.route(torch.randn(T, E, generator=g, device="cuda"), k)
    z = torch.randn(T * k, H, generator=g, device="cuda").to(D)
    w16 = r.weights.to(D)
    want = experts.combine(z, experts.plan_routes(r.ids, w16, E))
    for w in (w16, w16.double(), w16.t().contiguous().t(), w16.float()[:, None, :].expand(T, 3, k)[:, 1]):
        r.weights = w
        assert torch.equal(experts.combine(z, r), want)
    r.weights = w16.cpu()
    with pytest.raises(RuntimeError, match="weights"):
        experts.combine(z, r)
    codes, scales = int_weight((E, 32, 64), 64, D, g)
    pe = experts.pack_expert_codes(codes, scales, 64)
    x = int_rows(T, 64, D, g)
    good, wide = r.rows, r.rows.long()
    for bad in (wide, good[:-1], good.cpu()):
        r.rows = bad
        with pytest.raises((ValueError, RuntimeError), match="rows"):
            experts.expert_linear(x, pe, r)
    r.rows = good
    assert experts.expert_linear(x, pe, r).shape == (T * k, 32)


# ------------------------------------------------------------------ gated weights
def unpacked(pe, e):
    """W_hat of expert e's packed rows [rows, K] from the operands' documented layout (csrc/sqmp_w4.h):
    32-row blocks, 64-position stages, lane (r, q) holding rows r and 16 + r, chunk 4 (q & 1) + 2 s + q / 2."""
    nb, nk = (pe.N + 255) // 256 * 8, pe.Kp // 64
    words = pe.codes_t[e].cpu().view(torch.int32).view(nb, nk, 4, 16, 2, 2)       # block, stage, q, r, j, s
    nib = torch.stack([(words >> ((16 if v & 1 else 0) + 4 * (v >> 1))) & 15 for v in range(8)], -1) - 8
    codes = torch.zeros(nb, 2, 16, nk, 8, 8, dtype=torch.int32)                   # block, j, r, stage, chunk, element
    sal = None if pe.sal_t is None else pe.sal_t[e].cpu().view(nb, pe.S_pad // 64, 4, 16, 2, 2, 8)
    exact = None if sal is None else torch.zeros(nb, 2, 16, pe.S_pad // 64, 8, 8, dtype=pe.dtype)
    for q in range(4):
        for s in range(2):
            c = 4 * (q & 1) + 2 * s + (q >> 1)
            codes[:, :, :, :, c] = nib[:, :, q, :, :, s].permute(0, 3, 2, 1, 4)
            if sal is not None:
                exact[:, :, :, :, c] = sal[:, :, q, :, :, s].permute(0, 3, 2, 1, 4)
    group = torch.clamp(torch.arange(pe.Kp) // pe.Gw, max=pe.ngw - 1)
    scale = pe.scale_t[e].cpu().view(nb, pe.ngw, 16, 2).permute(0, 3, 2, 1).reshape(nb * 32, pe.ngw)[:, group]
    w = (codes.reshape(nb * 32, pe.Kp).double() * scale.double()).to(pe.dtype)
    amap = (pe.amap if pe.amap.dim() == 1 else pe.amap[e]).cpu().long()
    out = torch.zeros(nb * 32, pe.K, dtype=pe.dtype)
    out[:, amap[amap >= 0]] = w[:, amap >= 0]
    if exact is not None:
        out[:, pe.salient.cpu().long()] = exact.reshape(nb * 32, pe.S_pad)[:, :pe.S]
    return out[:pe.N]


@pytest.mark.parametrize("dt", ["fp16", "fp32"])
@pytest.mark.parametrize("wq", ["per_channel", "per_tensor", "per_group", "per_group_unsorted", "per_group_mean3std"])
@pytest.mark.parametrize("I,p", [(5, 0.0), (33, 0.0), (33, 0.06), (48, 0.0)])
def test_gated_weights_are_those_of_their_own_rows(I, p, wq, dt):
    """A gated weight is quantized as one weight of 2 I rows, whatever I is padded to: the very values
    of ops.pack_weight of those rows."""
    D, g = DT[dt], gen(I)
    E, K, G = 3, 192, 32
    # columns whose mean and spread differ: rows of zeros among the statistics change their order
    w = (torch.randn(E, 2 * I, K, generator=g, device="cuda") * 0.02
         * torch.rand(K, generator=g, device="cuda") + 0.02 * torch.rand(K, generator=g, device="cuda")).to(D)
    sal = torch.randperm(K, generator=g, device="cuda")[:int(p * K)] if p else None
    pe = experts.pack_experts(w, wq, G, sal, gated=True)
    assert pe.n_out == I and pe.gated
    n = torch.arange(I)
    gate = 32 * (n // 16) + n % 16
    for e in range(E):
        want = ops.dequant_weight(ops.pack_weight(w[e], wq, 4, G, sal)).cpu()
        got = unpacked(pe, e)
        assert torch.equal(got[gate], want[:I]) and torch.equal(got[gate + 16], want[I:])


@pytest.mark.parametrize("M", [64, 65, 300, 2048])
def test_linked_layers_after_use_gemv(M):
    """A model switched for decoding computes prompts as before: one grouped pass, the bits of "auto"."""
    from smoothquant import fake_quant
    D = torch.float16
    layers = _layers(3, 512, 256, D)
    group = fake_quant.link_siblings(*layers)
    x = torch.randn(M, 512, device="cuda").to(D)
    want = [q(x) for q in layers]
    launches = []
    real = ops.gemm_fq7_group
    fake_quant.use_gemv(torch.nn.ModuleList(layers))
    try:
        ops.gemm_fq7_group = lambda *a: launches.append(len(a[0])) or real(*a)
        got = [q(x) for q in layers]
    finally:
        ops.gemm_fq7_group = real
    assert launches == ([3] if M > 64 else []) and not group._stash
    for y, w, q in zip(got, want, layers):
        if M > 64:
            assert torch.equal(y, w)
            continue
        pw = q.packed()
        a = ops.quant_act_fp(x.clone(), pw, "per_group", 4, 64)
        w_hat = ops.dequant_weight_packed(pw).double()
        exact = a.double() @ w_hat.T + q.bias.reshape(-1).double()
        tol = tolerance(a, w_hat, exact, D, extra=2.0 ** -24 * exact.abs())
        assert ((y.double() - exact).abs() <= tol).all()


def test_scales_that_require_a_gradient():
    """Packed weights of parameters: constants without a graph, that copy as any other."""
    import copy
    D, g = torch.float16, gen(9)
    codes, scales = int_weight((2, 64, 128), 64, D, g)
    want = ops.pack_codes(codes[0], scales[0], 64)
    p = torch.nn.Parameter(scales)
    pw, pe = ops.pack_codes(codes[0], p[0], 64), experts.pack_expert_codes(codes, p, 64, gated=True)
    assert not pw.wscale.requires_grad and not pe.scale_t.requires_grad
    x = int_rows(3, 128, D, g)
    assert torch.equal(ops.gemv(x, copy.deepcopy(pw)), ops.gemv(x, want))
    r = experts.plan_routes(torch.tensor([[0], [1], [1]], device="cuda"), torch.ones(3, 1, device="cuda"), 2)
    assert torch.equal(experts.expert_linear(x, copy.deepcopy(pe), r, act="silu"),
                       experts.expert_linear(x, pe, r, act="silu"))
    dense = ops.pack_codes(codes[0], torch.nn.Parameter(scales[0]).repeat_interleave(16, 1), 4)
    assert not dense.dense.requires_grad
