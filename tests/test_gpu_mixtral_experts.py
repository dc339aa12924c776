"""W4A4Experts (the fused experts of a mixture, swapped by quantize_mixtral(quantize_experts=True))
against the same computation from the dequantized weights, and its place in a model."""
import copy

import pytest
import torch

from smoothquant import experts, fake_quant, ops
from smoothquant.checkpoint import load_quantized, save_quantized
from test_gpu_mixtral import _model, _tokens
from w4_cases import DT, gen

pytestmark = pytest.mark.gpu


def _plain(mod, base, x, ids, w, D, act_quant, salient):
    """The module's computation in fp32 from dequantized weights, quantizing activations with the
    framework's own quantizers."""
    E, inter = base.num_experts, base.intermediate_dim
    g = mod.group_size

    def quant(t, sal):
        t = t.clone()
        if act_quant is None:
            return t
        keep = None if sal is None else t[:, sal].clone()
        if sal is not None:
            mask = torch.ones(t.shape[1], dtype=torch.bool, device=t.device)
            mask[sal] = False
            t[:, mask] = fake_quant._ACT_FNS[act_quant](t[:, mask].contiguous(), **(
                dict(n_bits=4, group_size=g) if "group" in act_quant else dict(n_bits=4)))
            t[:, sal] = keep
            return t
        return fake_quant._ACT_FNS[act_quant](t, **(dict(n_bits=4, group_size=g) if "group" in act_quant
                                                    else dict(n_bits=4)))

    def w_hat(t, e, sal=None):
        return ops.dequant_weight(ops.pack_weight(t[e].to(D), mod.weight_quant, 4, g, sal)).float()

    xq = quant(x, salient).float()
    y = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    for e in range(E):
        t, j = torch.where(ids == e)
        if not len(t):
            continue
        u = xq[t] @ w_hat(base.gate_up_proj.data, e, salient).T
        h = (torch.nn.functional.silu(u[:, :inter]) * u[:, inter:]).to(D)
        z = (quant(h, None).float() @ w_hat(base.down_proj.data, e).T).to(D).float()
        y.index_add_(0, t, z * w[t, j, None].float())
    return y


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("wq,aq,p,T", [("per_channel", "per_token", 0.0, 1), ("per_channel", "per_token", 0.05, 70),
                                       ("per_group_unsorted", "per_group_unsorted", 0.0, 300),
                                       ("per_channel", None, 0.0, 33)])
def test_module(wq, aq, p, T, dt):
    D, g = DT[dt], gen(T)
    base = copy.deepcopy(_model(3).model.layers[0].mlp.experts).to("cuda", D)
    H = base.hidden_dim
    x = torch.randn(T, H, generator=g, device="cuda").to(D)
    imp = x.float().abs().mean(0).cpu()
    mod = experts.W4A4Experts.from_float(base, wq, aq, imp, p, 4, 32)
    ids = torch.rand(T, base.num_experts, generator=g, device="cuda").topk(2, dim=1).indices
    w = torch.rand(T, 2, generator=g, device="cuda")
    x0 = x.clone()
    y = mod(x, ids, w)
    assert torch.equal(x, x0) and y.shape == x.shape and y.dtype == D
    sal = None if p == 0 else mod.gate_up_salient.long()
    want = _plain(mod, base, x, ids, w, D, aq, sal)
    # 4-bit codes of h next to a rounding border may fall either way (1 / 7 of a value's range
    # each); everything else is within a few roundings
    rel = float((y.float() - want).norm() / want.norm())
    assert rel < (0.05 if aq else 2e-2), rel
    # each token by itself gives the same bits: nothing of one token reaches another
    if T > 1:
        alone = torch.cat([mod(x[t:t + 1], ids[t:t + 1], w[t:t + 1]) for t in (0, T // 2, T - 1)])
        ref = y[[0, T // 2, T - 1]]
        assert float((alone.float() - ref.float()).norm() / ref.float().norm()) < 0.05
    assert mod(x[:0], ids[:0], w[:0]).shape == (0, H)
    with pytest.raises(RuntimeError):
        mod.to(torch.float64)


@pytest.mark.parametrize("T", [3, 90])
@pytest.mark.parametrize("aq", ["per_token", None])
def test_module_captured(T, aq):
    """The module captured before and after its first eager call: replays equal the eager bits, and
    nothing that a capture built is used outside of it."""
    g = gen(T)
    base = copy.deepcopy(_model(3).model.layers[0].mlp.experts).to("cuda", torch.float16)
    x = torch.randn(T, base.hidden_dim, generator=g, device="cuda").half()
    ids = torch.rand(T, base.num_experts, generator=g, device="cuda").topk(2, dim=1).indices
    w = torch.rand(T, 2, generator=g, device="cuda")
    warm = experts.W4A4Experts.from_float(base, "per_channel", aq, None, 0, 4, 32)
    want = warm(x, ids, w)
    fresh = experts.W4A4Experts.from_float(base, "per_channel", aq, None, 0, 4, 32)
    for mod in (warm, fresh):
        xs = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = mod(xs, ids, w)
        assert torch.equal(mod(x, ids, w), want)          # eager between capture and replay
        for i in range(3):
            xs.copy_(x.roll(i, 0))
            graph.replay()
            eager = mod(x.roll(i, 0), ids, w)
            torch.cuda.synchronize()
            assert torch.equal(y, eager)


@pytest.mark.parametrize("aq,p", [("per_token", 0.0), ("per_token", 0.1)])
def test_quantize_mixtral_experts(tmp_path, aq, p):
    from smoothquant.calibration import get_calib_feat
    base = _model(5).to("cuda")
    feat = get_calib_feat(base, None, samples=[_tokens(1, 32), _tokens(2, 32)])
    x = _tokens(9, 40).to("cuda")
    kw = dict(weight_quant="per_channel", act_quant=aq, input_feat=feat, salient_prop=p, group_size=32)
    plain = fake_quant.quantize_mixtral(copy.deepcopy(base), **kw)
    q = fake_quant.quantize_model(copy.deepcopy(base), quantize_experts=True, **kw)
    layers = [m for m in q.modules() if isinstance(m, experts.W4A4Experts)]
    assert len(layers) == 2 and not any(isinstance(m, experts.W4A4Experts) for m in plain.modules())
    assert (layers[0].gate_up_salient is None) == (p == 0)
    with torch.no_grad():
        ref, y = plain(x).logits.float(), q(x).logits.float()
    assert y.isfinite().all()
    # 4-bit experts move the logits of this random model, but do not replace them
    assert float((y - ref).norm() / ref.norm()) < 0.5
    assert "W4A4Experts(4 experts" in repr(layers[0])
    # one token at a time, few-row kernels: the prompt's logits again
    fake_quant.use_gemv(q)
    with torch.no_grad():
        out = q(x[:, :39], use_cache=True)
        step = q(x[:, 39:], past_key_values=out.past_key_values, use_cache=True).logits[:, -1].float()
    assert float((step - y[:, -1]).norm() / y[:, -1].norm()) < 0.1
    fake_quant.use_gemv(q, False)
    # a checkpoint restores the very layers
    path = str(tmp_path / "m.pt")
    save_quantized(q, path)
    fresh = load_quantized(copy.deepcopy(base), path)
    with torch.no_grad():
        assert torch.equal(fresh(x).logits, q(x).logits)
    with pytest.raises(ValueError, match="row by row"):
        fake_quant.quantize_mixtral(copy.deepcopy(base), act_quant="per_group", quantize_experts=True)
