"""Inputs and 64-bit definitions shared by the few-row and expert tests."""
import torch

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# half a step of each type, relative: the error of one rounding
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def gen(seed, dev="cuda"):
    return torch.Generator(device=dev).manual_seed(seed)


def int_weight(shape, G, dt, g):
    """codes and power-of-two scales: products with small whole numbers, and their sums, are exact
    in fp32 whatever the order (all are multiples of 2^-4, sums below 2^19 of them)."""
    dev = g.device
    codes = torch.randint(-8, 8, shape, generator=g, device=dev, dtype=torch.int8)
    ng = (shape[-1] + G - 1) // G
    scales = 2.0 ** torch.randint(-4, 1, shape[:-1] + (ng,), generator=g, device=dev).float()
    return codes, scales.to(dt)


def int_rows(M, K, dt, g):
    return torch.randint(-4, 5, (M, K), generator=g, device=g.device).to(dt)


def values(codes, scales, G):
    """D(code * scale) in 64 bits."""
    s = scales.double().repeat_interleave(G, dim=-1)[..., :codes.shape[-1]]
    return (codes.double() * s).to(scales.dtype).double()


def tolerance(x, w, y, dt, extra=0.0):
    """|error| of one fp32 accumulation and one rounding to D.  The K products are exact in fp32
    (fp16 / bf16; one rounding each in fp32 -- the + 1) and meet in chains of at most K / 4 + 64
    additions (at least 4 partial sums per output, then their sum), each off by at most one
    step of the running sum, which sum |x w| bounds."""
    K = x.shape[1]
    chain = (K / 4 + 64 + 1) * 2.0 ** -23
    return chain * (x.double().abs() @ w.abs().T) + HALF[dt] * y.abs() * (1 + 2.0 ** -8) + extra \
        + torch.finfo(dt).smallest_normal * HALF[dt] * 2
