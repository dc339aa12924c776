"""Mixture-of-experts blocks with 4-bit expert weights: routing, the products grouped by expert,
the way back, and the module that replaces a model's fused experts.

    r = route(logits, top_k)                     # or plan_routes(ids, weights, num_experts)
    h = expert_linear(x, gate_up, r, act="silu")  # [tokens * top_k, I], rows in expert order
    z = expert_linear(h, down, r, rows="slot")
    y = combine(z, r)                             # [tokens, H]

The reference swaps every expert's w1 / w2 / w3 for a W4A4Linear
(/root/reference/smoothquant/fake_quant.py:564-668); transformers >= 5 holds them as two 3-D
parameters, which `pack_experts` packs and W4A4Experts computes.  Inference only; every function
launches HIP kernels on the current stream of its tensors' device, without host
synchronisation, and raises on host tensors.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch import nn

from . import _lib, ops
from ._lib import check, load

MAX_EXPERTS, MAX_TOP_K = 256, 16
MAX_PAIRS = 2 ** 31 - 4097  # slots and pairs are int32, the kernels' loops run at most a block past them
ACTS = {None: 0, "silu": 1, "gelu": 2}


# ------------------------------------------------------------------ routing
@dataclass
class Routing:
    """Which experts the tokens go to, and the (token, expert) pairs in expert order.  A pair is
    f = token * top_k + j; an id of -1 means that nothing was chosen there.  The three lists are a
    plan as plan_routes makes it: the kernels follow them without looking whether they agree."""
    ids: torch.Tensor       # int32 [T, top_k]
    weights: torch.Tensor   # fp32 [T, top_k]
    offsets: torch.Tensor   # int32 [E + 1]: slots of expert e are offsets[e] .. offsets[e + 1]
    rows: torch.Tensor      # int32 [T * top_k]: slot -> pair (-1 behind the last)
    slots: torch.Tensor     # int32 [T * top_k]: pair -> slot (-1: nothing chosen)
    num_experts: int

    @property
    def tokens(self) -> int:
        return self.ids.shape[0]

    @property
    def top_k(self) -> int:
        return self.ids.shape[1]


_I32 = torch.int32


def _misfit(t, n: int, dev) -> bool:
    """Whether a kernel would misread t as n contiguous int32 on dev."""
    return not (t is not None and t.dtype is _I32 and t.numel() == n and t.device == dev
                and t.is_contiguous())


def _refuse_list(what: str, name: str, t, n: int, dev):
    if t is not None and t.device != dev:
        raise RuntimeError(f"{what}: x on {dev}, routing.{name} on {t.device}")
    raise ValueError(f"{what}: routing.{name} must be {n} contiguous int32 on {dev}, got "
                     + ("None" if t is None else f"{t.dtype} {tuple(t.shape)} of strides {t.stride()}"))


def _shape_of(what: str, r: Routing):
    if r.ids.dim() != 2:
        raise ValueError(f"{what}: routing.ids must be [tokens, top_k], got {tuple(r.ids.shape)}")
    return r.ids.shape


def _refuse_overlap(what: str, out: torch.Tensor, x: torch.Tensor):
    """Workgroups read rows of x that others' outputs would have taken the place of."""
    a, b = ((t.data_ptr(), t.data_ptr() + t.element_size() * (
        1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (out, x))
    if out.numel() and x.numel() and a[0] < b[1] and b[0] < a[1]:
        raise ValueError(f"{what}: out overlaps the operand in memory")


def _plan_buffers(T: int, k: int, E: int, dev, n_ids: int):
    """(ids, rows, slots, offsets, workspace, its size): the first four, int32, from one
    allocation in this order."""
    n = load().sqmp_route_workspace_bytes(T, E) if T > 256 else 0
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    buf = torch.empty(n_ids + 2 * T * k + E + 1, dtype=torch.int32, device=dev)
    return (*buf.split_with_sizes((n_ids, T * k, T * k, E + 1)), ws, n)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _check_sizes(what: str, T: int, E: int, k: int):
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"{what}: {E} experts, supported are 1 .. {MAX_EXPERTS}")
    if not 1 <= k <= MAX_TOP_K:
        raise ValueError(f"{what}: top_k {k}, supported are 1 .. {MAX_TOP_K}")
    if T * k > MAX_PAIRS:
        raise ValueError(f"{what}: {T} tokens times {k} are more than {MAX_PAIRS} pairs")


@ops.on_tensor_device
def route(logits: torch.Tensor, top_k: int, normalize: bool = True) -> Routing:
    """The top_k largest logits of every token [T, E] (ties: the lowest index; NaN counts as the
    largest, -inf is never chosen) with their softmax weights -- over the chosen ones, or
    over all E with normalize=False -- and the plan of plan_routes.  A token whose logits are all
    -inf (padding) goes to no expert."""
    if not logits.is_cuda:
        ops._require_gpu(logits, "route")
    if logits.dim() != 2:
        raise ValueError(f"route: logits must be [tokens, experts], got {tuple(logits.shape)}")
    T, E = logits.shape
    _check_sizes("route", T, E, top_k)
    if top_k > E:
        raise ValueError(f"route: top_k {top_k} of {E} experts")
    dt = ops._dtype_code(logits.dtype)
    ld, s1 = logits.stride()
    if s1 != 1 or ld < E:
        logits = logits.contiguous()
        ld = E
    dev = logits.device
    weights = torch.empty((T, top_k), dtype=torch.float32, device=dev)
    ids, rows, slots, offsets, wp, n = _plan_buffers(T, top_k, E, dev, T * top_k)
    op = offsets.data_ptr()
    tk = 4 * T * top_k  # bytes of each of the three lists before it
    status = load().sqmp_route(logits.data_ptr(), ld, dt, T, E, top_k, int(normalize),
                               weights.data_ptr(), op - 3 * tk, op, op - 2 * tk, op - tk,
                               _ptr(wp), n, ops._raw_stream(dev.index))
    if status:
        check(status, "route")
    return Routing(ids.view(T, top_k), weights, offsets, rows, slots, E)


@ops.on_tensor_device
def plan_routes(ids: torch.Tensor, weights: torch.Tensor, num_experts: int) -> Routing:
    """The plan for a routing chosen elsewhere: ids [T, top_k] (any integer type; a value outside
    0 .. num_experts - 1 means that nothing was chosen), weights [T, top_k].  The pairs of an expert
    keep the order of the tokens."""
    ops._require_gpu(ids, "plan_routes")
    if ids.dim() != 2 or ids.dtype.is_floating_point or ids.dtype.is_complex or ids.dtype == torch.bool:
        raise ValueError(f"plan_routes: ids must be integers [tokens, top_k], got {ids.dtype} "
                         f"{tuple(ids.shape)}")
    if weights.shape != ids.shape or weights.device != ids.device:
        raise ValueError(f"plan_routes: weights {tuple(weights.shape)} on {weights.device} do not "
                         f"match ids {tuple(ids.shape)} on {ids.device}")
    T, k = ids.shape
    _check_sizes("plan_routes", T, num_experts, k)
    if ids.dtype != torch.int32:
        ids = (ids.long().clamp(-1, num_experts)).to(torch.int32)  # (no id may wrap into range)
    ids = ids.contiguous()
    _, rows, slots, offsets, ws, n = _plan_buffers(T, k, num_experts, ids.device, 0)
    check(load().sqmp_plan_routes(ids.data_ptr(), T, num_experts, k, offsets.data_ptr(),
                                  rows.data_ptr(), slots.data_ptr(), _ptr(ws), n,
                                  ops._raw_stream(ids.device.index)), "plan_routes")
    return Routing(ids, weights.float().contiguous(), offsets, rows, slots, num_experts)


# ------------------------------------------------------------------ packed experts
@dataclass
class PackedExperts:
    """E packed 4-bit weights of one shape (the tile-major operands of sqmp_expert_linear_w4)."""
    codes_t: torch.Tensor            # uint8 [E, ...]
    scale_t: torch.Tensor            # D [E, ...]
    sal_t: Optional[torch.Tensor]    # D [E, ...], None without salient columns
    amap: torch.Tensor               # int32 [Kp], or [E, Kp] where every expert has its own order
    salient: Optional[torch.Tensor]  # int32 [S]
    num_experts: int
    n_out: int                       # columns of the product (gated: of act(gate) * up)
    N: int                           # packed weight rows
    K: int
    Kp: int
    S: int
    S_pad: int
    Gw: int
    ngw: int
    dtype: torch.dtype
    gated: bool
    identity: bool                   # the operand is x itself (columns' order, K % 64 == 0)


def _interleave(t: torch.Tensor) -> torch.Tensor:
    """[E, 2 I, X] (gate rows, then up rows) -> 16 gate and 16 up rows in turn, I padded to 16."""
    E, rows, X = t.shape
    inter, pad = rows // 2, (rows // 2 + 15) // 16 * 16
    halves = t.reshape(E, 2, inter, X)
    if pad != inter:
        halves = torch.nn.functional.pad(halves, (0, 0, 0, pad - inter))
    return halves.view(E, 2, pad // 16, 16, X).transpose(1, 2).reshape(E, 2 * pad, X)


def _packed_rows(pw: ops.PackedWeight, gated: bool):
    """(codes, wscale, wsal, N) of the packed rows, interleaved where gated: after the quantization,
    whose statistics (the mean and spread of a column) see the weight's own rows alone."""
    if not gated:
        return pw.codes, pw.wscale, pw.wsal, pw.N

    def rows(t):
        return _interleave(t[None, :pw.N])[0]
    codes, scale, sal = rows(pw.codes), rows(pw.wscale.t()), rows(pw.wsal)
    N = codes.shape[0]
    more = (0, 0, 0, ops.pad_n(N) - N)
    return (torch.nn.functional.pad(codes, more),
            torch.nn.functional.pad(scale, more).t().contiguous(), sal.contiguous(), N)


def _pack_all(weights, E: int, rows: int, gated: bool) -> PackedExperts:
    """weights: iterator over the E experts' PackedWeight (gated: of [gate; up] rows)."""
    pe, maps = None, []
    for e, pw in enumerate(weights):
        if not ops.gemv_eligible(pw):
            raise ValueError("pack_experts: needs 4-bit codes in groups of a multiple of 8 columns "
                             f"(n_bits {pw.n_bits}, group {pw.Gw})")
        codes, wscale, wsal, N = _packed_rows(pw, gated)
        one = ops.tile_major(codes, wscale, wsal, N, pw.Kp, pw.S_pad, pw.ngw, pw.dtype,
                             None if pe is None else (pe.codes_t[e], pe.scale_t[e],
                                                      all_sal[e]))
        if pe is None:
            stacks = [torch.empty((E,) + t.shape, dtype=t.dtype, device=t.device) for t in one]
            for st, t in zip(stacks, one):
                st[0] = t
            all_sal = stacks[2]
            pe = PackedExperts(stacks[0], stacks[1], all_sal if pw.S_pad else None, pw.amap,
                               pw.salient, E, rows // 2 if gated else rows, N, pw.K, pw.Kp,
                               pw.S, pw.S_pad, pw.Gw, pw.ngw, pw.dtype, gated, False)
        maps.append(pw.amap)
    amap = torch.stack(maps)
    if bool((amap == amap[0]).all()):  # (also on the first use of another stream: a sync)
        amap = amap[0].contiguous()
        pe.identity = pe.S == 0 and pe.K % 64 == 0 and bool(
            torch.equal(amap[:pe.K], torch.arange(pe.K, dtype=torch.int32, device=amap.device)))
    pe.amap = amap
    return pe


def _check_stack(what: str, w: torch.Tensor, gated: bool):
    ops._require_gpu(w, what)
    if w.dim() != 3 or 0 in w.shape:
        raise ValueError(f"{what}: expected [experts, rows, columns], got {tuple(w.shape)}")
    if w.shape[0] > MAX_EXPERTS:
        raise ValueError(f"{what}: {w.shape[0]} experts, at most {MAX_EXPERTS}")
    if gated and w.shape[1] % 2:
        raise ValueError(f"{what}: a gated weight has an even number of rows, got {w.shape[1]}")


@ops.on_tensor_device
def pack_experts(w: torch.Tensor, weight_quant: str = "per_channel", group_size: int = 128,
                 salient: Optional[torch.Tensor] = None, gated: bool = False) -> PackedExperts:
    """Quantize w D [E, N, K] to 4 bits expert by expert (ops.pack_weight).  gated: the rows are
    [gate; up] halves (transformers' gate_up_proj); their statistics (per_tensor, the column
    order of the sorted modes) are taken over both.  salient: one set of exact columns for all."""
    _check_stack("pack_experts", w, gated)
    if weight_quant == "none":
        raise ValueError("pack_experts: needs a quantized weight")
    it = (ops.pack_weight(w[e], weight_quant, 4, group_size, salient) for e in range(w.shape[0]))
    return _pack_all(it, w.shape[0], w.shape[1], gated)


@ops.on_tensor_device
def pack_expert_codes(codes: torch.Tensor, scales: torch.Tensor, group_size: int,
                      gated: bool = False) -> PackedExperts:
    """As ops.pack_codes for codes int8 [E, N, K] and scales D [E, N, ceil(K / group_size)]."""
    _check_stack("pack_expert_codes", codes, gated)
    if scales.dim() != 3 or scales.shape[:2] != codes.shape[:2]:
        raise ValueError(f"pack_expert_codes: scales {tuple(scales.shape)} do not match codes "
                         f"{tuple(codes.shape)}")
    n_rows, scales = codes.shape[1], scales.detach()
    if gated:
        codes, scales = _interleave(codes), _interleave(scales)
    # one weight whose rows are the experts', each padded to the operands' 256
    E, N, K = codes.shape
    pad = (N + 255) // 256 * 256
    if pad != N:
        codes = torch.nn.functional.pad(codes, (0, 0, 0, pad - N))
        scales = torch.nn.functional.pad(scales, (0, 0, 0, pad - N))
    pw = ops.pack_codes(codes.reshape(E * pad, K), scales.reshape(E * pad, -1), group_size)
    if not ops.gemv_eligible(pw):
        raise ValueError("pack_expert_codes: needs groups of a multiple of 8 columns, got "
                         f"{group_size}")
    one = ops.tile_major(pw.codes, pw.wscale, pw.wsal, E * pad, pw.Kp, 0, pw.ngw, pw.dtype)
    return PackedExperts(one[0].view(E, -1), one[1].view(E, -1), None, pw.amap, None, E,
                         n_rows // 2 if gated else n_rows, N, K, pw.Kp, 0, 0, pw.Gw, pw.ngw,
                         pw.dtype, gated, K % 64 == 0)


# ------------------------------------------------------------------ products
def _operand(x: torch.Tensor, pe: PackedExperts, r: Routing, by_slot: bool):
    """(operand, its slot -> pair list or None, its coded columns): x itself where the kernels can read it, a packed
    copy of its rows, or -- where every expert has its own column order -- of every slot's row."""
    rows = None if by_slot else r.rows
    if pe.identity and ops._operand_rows(x, pe.K):
        return x, rows, pe.K
    if x.stride(1) != 1 or x.stride(0) == 0:  # (0: rows of an expanded tensor)
        x = x.contiguous()
    own = pe.amap.dim() == 2
    n = r.rows.shape[0] if own else x.shape[0]
    out = x.new_empty((n, pe.Kp + pe.S_pad))
    status = load().sqmp_pack_rows(x.data_ptr(), max(x.stride(0), 1), ops.DTYPE_CODE[x.dtype], n,
                                   pe.amap.data_ptr(), pe.Kp, _ptr(pe.salient), pe.S, pe.S_pad,
                                   _ptr(rows) if own else None, r.ids.shape[1],
                                   r.offsets.data_ptr() if own else None, pe.num_experts,
                                   pe.Kp if own else 0, out.data_ptr(),
                                   ops._raw_stream(x.device.index))
    if status:
        check(status, "pack_rows")
    return out, None if own else rows, pe.Kp


@ops.on_tensor_device
def expert_linear(x: torch.Tensor, pe: PackedExperts, routing: Routing, act: Optional[str] = None,
                  rows: str = "token", out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """z [tokens * top_k, n_out], rows in expert order: D(W_e x) for every (token, expert) pair, or
    D(act(gate) * up) of a gated weight (act "silu" / "gelu"; fp32 up to the one rounding).

    x: [tokens, K] (rows="token") or [tokens * top_k, K] already in expert order (rows="slot").
    Rows of z behind routing.offsets[-1] (tokens that go nowhere) are left as they were.  `out` may not
    share memory with x."""
    if not x.is_cuda:
        ops._require_gpu(x, "expert_linear")
    code = ACTS.get(act, -1)
    by_slot = rows == "slot"
    T, k = _shape_of("expert_linear", routing)
    S, dev = T * k, x.device
    if (code < 0 or (code > 0) != pe.gated or not (by_slot or rows == "token")
            or routing.num_experts != pe.num_experts or x.dim() != 2
            or x.shape[0] != (S if by_slot else T) or x.shape[1] != pe.K
            or x.dtype is not pe.dtype or dev != pe.codes_t.device):
        _expert_refuse(x, pe, routing, act, rows)
    if _misfit(routing.rows, S, dev):
        _refuse_list("expert_linear", "rows", routing.rows, S, dev)
    if _misfit(routing.offsets, pe.num_experts + 1, dev):
        _refuse_list("expert_linear", "offsets", routing.offsets, pe.num_experts + 1, dev)
    given = out is not None
    if not given:
        out = x.new_empty((S, pe.n_out))
    elif (tuple(out.shape) != (S, pe.n_out) or out.dtype != pe.dtype or out.device != dev
          or not out.is_contiguous()):
        raise ValueError(f"expert_linear: out must be contiguous {pe.dtype} [{S}, {pe.n_out}] on {dev}")
    if given:
        _refuse_overlap("expert_linear", out, x)
    if S == 0:
        return out
    a, pairs, cols = _operand(x, pe, routing, by_slot)
    lib, dt = load(), ops.DTYPE_CODE[pe.dtype]
    n = ops.workspace_bytes("expert", dt, pe.num_experts, S, pe.N, pe.Kp)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    status = lib.sqmp_expert_linear_w4(
        a.data_ptr(), a.stride(0) if a.shape[0] > 1 else pe.Kp + pe.S_pad, cols, _ptr(pairs),
        k, routing.offsets.data_ptr(), pe.num_experts, pe.codes_t.data_ptr(),
        pe.scale_t.data_ptr(), _ptr(pe.sal_t), out.data_ptr(), dt, S, a.shape[0], pe.N, pe.n_out,
        pe.Kp, pe.S_pad, pe.Gw, pe.ngw, code, _ptr(ws), n, ops._raw_stream(dev.index))
    if status:
        check(status, "expert_linear")
    return ops.written(out) if given else out


def _expert_refuse(x, pe, routing, act, rows):
    if act not in ACTS:
        raise ValueError(f"expert_linear: act must be one of {sorted(map(str, ACTS))}, got {act!r}")
    if (act is not None) != pe.gated:
        raise ValueError("expert_linear: an activation goes with a gated weight, and a gated weight "
                         f"with an activation (act={act!r}, gated={pe.gated})")
    if rows not in ("token", "slot"):
        raise ValueError(f"expert_linear: rows must be 'token' or 'slot', got {rows!r}")
    if routing.num_experts != pe.num_experts:
        raise ValueError(f"expert_linear: routing over {routing.num_experts} experts, weight of "
                         f"{pe.num_experts}")
    want = (routing.tokens * (routing.top_k if rows == "slot" else 1), pe.K)
    if tuple(x.shape) != want:
        raise ValueError(f"expert_linear: x must be {list(want)}, got {list(x.shape)}")
    if x.dtype != pe.dtype:
        raise RuntimeError(f"expected input dtype {pe.dtype}, got {x.dtype}")
    raise RuntimeError(f"expert_linear: x on {x.device}, weight on {pe.codes_t.device}")


@ops.on_tensor_device
def combine(z: torch.Tensor, routing: Routing, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [tokens, H]: y[t] = D(sum_j weights[t, j] * z[slot of pair (t, j)]), fp32 sums in the
    order of j; a token that goes nowhere gets zeros.  `out` may not share memory with z."""
    if not z.is_cuda:
        ops._require_gpu(z, "combine")
    T, k = _shape_of("combine", routing)
    if z.dim() != 2 or z.shape[0] != T * k or z.shape[1] == 0:
        raise ValueError(f"combine: z must be [{T * k}, H], got {tuple(z.shape)}")
    if z.shape[1] > MAX_PAIRS:
        raise ValueError(f"combine: {z.shape[1]} columns, at most {MAX_PAIRS}")
    dt = ops.DTYPE_CODE.get(z.dtype)
    if dt is None:
        ops._dtype_code(z.dtype)
    dev = z.device
    if _misfit(routing.slots, T * k, dev):
        _refuse_list("combine", "slots", routing.slots, T * k, dev)
    w = routing.weights
    if w.shape != routing.ids.shape:
        raise ValueError(f"combine: routing.weights must be {[T, k]}, got {list(w.shape)}")
    if w.device != dev:
        raise RuntimeError(f"combine: z on {dev}, routing.weights on {w.device}")
    if w.dtype is not torch.float32 or not w.is_contiguous():  # (a caller's, as in plan_routes)
        w = w.float().contiguous()
    if not z.is_contiguous():
        z = z.contiguous()
    H = z.shape[1]
    given = out is not None
    if not given:
        out = z.new_empty((T, H))
    elif (tuple(out.shape) != (T, H) or out.dtype != z.dtype or out.device != dev
          or not out.is_contiguous()):
        raise ValueError(f"combine: out must be contiguous {z.dtype} [{T}, {H}] on {dev}")
    if given:
        _refuse_overlap("combine", out, z)
    if T == 0:
        return out
    status = load().sqmp_combine(z.data_ptr(), dt, T, k, H, routing.slots.data_ptr(),
                                 w.data_ptr(), out.data_ptr(),
                                 ops._raw_stream(dev.index))
    if status:
        check(status, "combine")
    return ops.written(out) if given else out


# ------------------------------------------------------------------ the module
_TENSORS = ("codes_t", "scale_t", "sal_t", "amap", "salient")
_INTS = ("num_experts", "n_out", "N", "K", "Kp", "S", "S_pad", "Gw", "ngw", "gated", "identity")
# activation quantizers that look at one row at a time: they do not depend on which rows an expert
# gets (the sorted and per_tensor ones take statistics over an expert's whole batch)
ROW_ACTS = ("per_token", "per_group_unsorted")


def _act_name(fn) -> str:
    """The name of a gated MLP's activation module."""
    name = type(fn).__name__
    if isinstance(fn, nn.SiLU) or name == "SiLUActivation":
        return "silu"
    if (isinstance(fn, nn.GELU) and fn.approximate == "none") or name == "GELUActivation":
        return "gelu"
    raise ValueError(f"W4A4Experts: activation {name} (supported: silu, gelu)")


class W4A4Experts(nn.Module):
    """Drop-in for transformers' fused experts (gate_up_proj [E, 2 I, H], down_proj [E, H, I];
    forward(hidden_states, top_k_index, top_k_weights)) with 4-bit weights and row-wise 4-bit
    activations: what fake_quant.py:564-668 does to the experts' separate w1 / w3 / w2, as two
    products grouped by expert.  act(gate) * up is formed in fp32 and rounded once (the reference
    rounds gate, up and act(gate) to the model's type first); the experts' outputs are weighted and
    summed in fp32."""

    EXTRA_FORMAT = "sqmp-w4a4-experts/1"

    def __init__(self, act: str = "silu", act_quant: Optional[str] = "per_token",
                 quant_bits: int = 4, group_size: int = 128):
        super().__init__()
        if act not in ("silu", "gelu"):
            raise ValueError(f"W4A4Experts: activation {act!r} (supported: silu, gelu)")
        if act_quant is not None and act_quant not in ROW_ACTS:
            raise ValueError(f"Invalid act_quant: {act_quant} (experts quantize row by row: "
                             f"{', '.join(ROW_ACTS)} or None)")
        if quant_bits != 4:
            raise ValueError(f"quant_bits={quant_bits}: packed experts support 4 bits")
        self.act, self.act_quant, self.quant_bits, self.group_size = act, act_quant, quant_bits, group_size
        self.weight_quant = "None"
        self._meta = None
        for part in ("gate_up", "down"):
            for n in _TENSORS:
                self.register_buffer(f"{part}_{n}", None)

    # -------------------------------------------------------------- packing
    @staticmethod
    def check(module, weight_quant="per_channel", act_quant="per_token", quant_bits=4, group_size=128):
        """The module that would take over `module`, without its weights; ValueError where none can."""
        for n in ("gate_up_proj", "down_proj", "act_fn"):
            if not hasattr(module, n):
                raise ValueError(f"W4A4Experts: {type(module).__name__} has no fused {n}")
        new = W4A4Experts(_act_name(module.act_fn), act_quant, quant_bits, group_size)
        if weight_quant == "none" or weight_quant not in ops.WEIGHT_MODES:
            raise ValueError(f"W4A4Experts: invalid weight_quant: {weight_quant}")
        for w in (module.gate_up_proj, module.down_proj):
            if w.shape[0] > MAX_EXPERTS:
                raise ValueError(f"W4A4Experts: {w.shape[0]} experts, at most {MAX_EXPERTS}")
            if ops.geometry(w.shape[2], 0, ops.WEIGHT_MODES[weight_quant], group_size)[1] % 8:
                raise ValueError("W4A4Experts: needs groups of a multiple of 8 columns, got "
                                 f"{group_size}")
        return new

    @staticmethod
    def from_float(module, weight_quant="per_channel", act_quant="per_token", importance=None,
                   salient_prop=0, quant_bits=4, group_size=128):
        """module: the fused experts.  importance [H] picks the salient columns of gate_up_proj
        (one set for all experts, as W4A4Linear picks them)."""
        new = W4A4Experts.check(module, weight_quant, act_quant, quant_bits, group_size)
        if not torch.cuda.is_available():
            raise RuntimeError("W4A4Experts packing needs a ROCm GPU (no CPU implementation)")
        gate_up, down = module.gate_up_proj.data, module.down_proj.data
        dev = gate_up.device
        salient = None
        if importance is not None and salient_prop > 0:
            order = torch.argsort(importance, descending=True, stable=True)
            salient = order[:max(1, int(salient_prop * len(order)))]
        gpu = dev if dev.type == "cuda" else torch.device("cuda")
        new._install("gate_up", pack_experts(gate_up.to(gpu), weight_quant, group_size, salient, gated=True))
        new._install("down", pack_experts(down.to(gpu), weight_quant, group_size))
        new.weight_quant = weight_quant
        return new if dev == gpu else new.to(dev)

    def _install(self, part: str, pe: PackedExperts):
        for n in _TENSORS:
            setattr(self, f"{part}_{n}", getattr(pe, n))
        meta = dict(self._meta or {}, dtype=pe.dtype)
        meta.update({f"{part}_{n}": getattr(pe, n) for n in _INTS})
        self._meta = meta
        self.__dict__.pop("_packed", None)

    def packed(self):
        """(gate_up, down) as PackedExperts, and the column maps of the input's quantizer."""
        b = tuple(getattr(self, f"{part}_{n}") for part in ("gate_up", "down") for n in _TENSORS)
        c = self.__dict__.get("_packed")
        if c is not None and all(x is y for x, y in zip(c[0], b)):
            return c[1]
        if self._meta is None:
            raise RuntimeError("W4A4Experts has no packed weight")
        pes = []
        for part in ("gate_up", "down"):
            kw = {n: getattr(self, f"{part}_{n}") for n in _TENSORS}
            kw.update({n: self._meta[f"{part}_{n}"] for n in _INTS})
            pes.append(PackedExperts(dtype=self._meta["dtype"], **kw))
        dev = pes[0].codes_t.device
        with torch.cuda.device(dev):
            maps = [ops.build_maps(pe.K, pe.salient, dev)[2:] for pe in pes]
            if not torch.cuda.is_current_stream_capturing():
                # kept: built on one stream, read later from any (a capture's maps belong to its
                # replays and are built again)
                torch.cuda.synchronize(dev)
                self.__dict__["_packed"] = (b, (pes[0], pes[1], maps))
        return pes[0], pes[1], maps

    # -------------------------------------------------------------- forward
    def _quant(self, t2: torch.Tensor, pe: PackedExperts, maps) -> torch.Tensor:
        if self.act_quant is not None:
            ops.fake_quant_inplace(t2, self.act_quant, self.quant_bits, self.group_size, maps[0],
                                   maps[1], pe.S)
        return t2

    @torch.no_grad()
    def forward(self, hidden_states, top_k_index, top_k_weights):
        ops._require_gpu(hidden_states, "W4A4Experts.forward")
        if hidden_states.device.index != ops._current_device():
            with torch.cuda.device(hidden_states.device):
                return self.forward(hidden_states, top_k_index, top_k_weights)
        gate_up, down, maps = self.packed()
        x = hidden_states.reshape(-1, hidden_states.shape[-1])
        if x.shape[1] != gate_up.K:
            raise ValueError(f"W4A4Experts: hidden size {x.shape[1]}, packed for {gate_up.K}")
        if x.dtype != gate_up.dtype:
            raise RuntimeError(f"expected input dtype {gate_up.dtype}, got {x.dtype}")
        if x.shape[0] == 0:
            return torch.empty_like(hidden_states)
        r = plan_routes(top_k_index, top_k_weights, gate_up.num_experts)
        if r.tokens != x.shape[0]:
            raise ValueError(f"W4A4Experts: {x.shape[0]} tokens, {r.tokens} routed")
        if self.act_quant is not None:
            x = x.clone(memory_format=torch.contiguous_format)  # (the caller's stays as it was)
        h = expert_linear(self._quant(x, gate_up, maps[0]), gate_up, r, act=self.act)
        z = expert_linear(self._quant(h, down, maps[1]), down, r, rows="slot")
        return combine(z, r).view(hidden_states.shape)

    # -------------------------------------------------------------- casts and persistence
    def _apply(self, fn, recurse=True):
        if self._meta is not None and self.gate_up_scale_t is not None:
            dt = fn(torch.empty(0, dtype=self._meta["dtype"], device=self.gate_up_scale_t.device)).dtype
            if dt != self._meta["dtype"]:
                raise RuntimeError(f"W4A4Experts: packed in {self._meta['dtype']}; a cast to {dt} changes "
                                   "the weights' values -- quantize the model in the target dtype")
        return super()._apply(fn, recurse)

    def get_extra_state(self):
        m = self._meta
        return {"format": self.EXTRA_FORMAT, "act": self.act, "act_quant": self.act_quant,
                "quant_bits": self.quant_bits, "group_size": self.group_size,
                "weight_quant": self.weight_quant,
                "meta": None if m is None else {k: str(v).replace("torch.", "") if k == "dtype" else int(v)
                                                for k, v in m.items()}}

    def set_extra_state(self, state):
        if not isinstance(state, dict) or state.get("format") != self.EXTRA_FORMAT:
            raise RuntimeError(f"W4A4Experts: unsupported extra state {type(state)}")
        for n in ("act", "act_quant", "quant_bits", "group_size", "weight_quant"):
            setattr(self, n, state[n])
        m = state["meta"]
        if m is not None:
            m = dict(m, dtype=getattr(torch, m["dtype"]))
            for part in ("gate_up", "down"):
                for n in ("gated", "identity"):
                    m[f"{part}_{n}"] = bool(m[f"{part}_{n}"])
        self._meta = m
        self.__dict__.pop("_packed", None)

    def _load_from_state_dict(self, sd, prefix, *args):
        if prefix + "_extra_state" in sd:  # size the buffers (None in a fresh module)
            for part in ("gate_up", "down"):
                for n in _TENSORS:
                    t = sd.get(f"{prefix}{part}_{n}")
                    setattr(self, f"{part}_{n}", None if t is None else torch.empty_like(t))
        super()._load_from_state_dict(sd, prefix, *args)

    def __repr__(self):
        m = self._meta or {}
        return (f"W4A4Experts({m.get('gate_up_num_experts')} experts, {m.get('gate_up_K')} -> "
                f"{m.get('gate_up_n_out')}, act={self.act}, weight_quant={self.weight_quant}, "
                f"act_quant={self.act_quant}, salient={m.get('gate_up_S')})")


__all__ = ["Routing", "route", "plan_routes", "PackedExperts", "pack_experts", "pack_expert_codes",
           "expert_linear", "combine", "W4A4Experts"]
