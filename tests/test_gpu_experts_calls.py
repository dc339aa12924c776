"""The expert calls in the company of the framework's other layers, and the calls around the tested
ones: buffers used again, overlapping ones, routings by hand."""
import pytest
import torch

from smoothquant import experts, ops
from smoothquant.fake_quant import W4A4Linear
from w4_cases import DT, gen, int_rows, int_weight

pytestmark = pytest.mark.gpu


def _layers(n, K, N, D, **kw):
    """Sorted per_group layers of one input width, whose statistics and operands are kept per input."""
    torch.manual_seed(6)
    return [W4A4Linear.from_float(torch.nn.Linear(K, N).to("cuda", D), weight_quant="per_group",
                                  act_quant="per_group", group_size=32, **kw) for _ in range(n)]


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
        a = ops.quant_act_fp(x, others[2], "per_group", 4, 32)
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
