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
