"""Every decoder of 4-bit codes gives D(code * scale): all 16 codes under scales over the type's range,
read through the kernels by one-hot rows (a product with one term, 1 * W)."""
import pytest
import torch

from smoothquant import experts, ops
from w4_cases import DT, gen, values

pytestmark = pytest.mark.gpu


def _weight(N, K, G, dt, g):
    codes = torch.randint(-8, 8, (N, K), generator=g, device="cuda", dtype=torch.int8)
    codes[:, :16] = torch.arange(-8, 8, device="cuda")
    # mantissas of every kind, exponents from the least normal value / 8 up to the largest / 8
    lo, hi = (-11, 11) if dt == torch.float16 else (-120, 120)
    e = torch.randint(lo, hi, (N, (K + G - 1) // G), generator=g, device="cuda")
    scales = ((1 + torch.rand(e.shape, generator=g, device="cuda").double()) * torch.exp2(e.double())).to(dt)
    return codes, scales


@pytest.mark.parametrize("dt", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_decoders(G, dt):
    D, g = DT[dt], gen(G)
    N, K = 1024, 512
    codes, scales = _weight(N, K, G, D, g)
    if D == torch.float32:
        scales = scales.clamp(max=2.0 ** 100)
    want = values(codes, scales, G).to(D).T.contiguous()                 # [K, N]
    assert want.isfinite().all()
    pw = ops.pack_codes(codes, scales, G)
    eye = torch.eye(K, device="cuda", dtype=D)
    for M in (1, 8, 16, 64):                                             # the few-row kernels
        for at in range(0, K, M if M > 8 else 64):
            n = min(M, K - at)
            assert torch.equal(ops.gemv(eye[at:at + n].contiguous(), pw), want[at:at + n])
    if D != torch.float32:                                               # the packed-order GEMM
        assert torch.equal(ops.gemm_fq(eye, pw, None), want)
    pe = experts.pack_expert_codes(torch.stack([codes, codes.flip(0)]), torch.stack([scales, scales.flip(0)]), G)
    both = torch.stack([want, want.flip(1)])
    for T in (16, K):                                                    # few rows of an expert, its tiles
        ids = (torch.arange(T, device="cuda") % 2).view(-1, 1)
        r = experts.plan_routes(ids, torch.ones(T, 1, device="cuda"), 2)
        z = experts.expert_linear(eye[:T].contiguous(), pe, r)
        pairs = r.rows.long()
        assert torch.equal(z, both[ids.view(-1)[pairs], pairs])
