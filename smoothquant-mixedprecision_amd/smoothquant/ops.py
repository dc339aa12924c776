"""Torch-facing wrappers over the HIP C ABI (PyTorch supplies device memory and streams).

Every function here launches libsqmp_w4a4 kernels on the caller's current stream and
raises if a tensor is not on a ROCm device: the W4A4 operator has no CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import os
import weakref
from dataclasses import dataclass, field
from typing import Optional

import torch

from . import _lib
from ._lib import check, load

DTYPE_CODE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
ACT_MODES = {"per_token": _lib.ACT_PER_TOKEN, "per_tensor": _lib.ACT_PER_TENSOR,
             "per_group": _lib.ACT_PER_GROUP, "per_group_unsorted": _lib.ACT_PER_GROUP_UNSORTED,
             "per_group_mean3std": _lib.ACT_PER_GROUP_MEAN3STD}
WEIGHT_MODES = {"per_channel": _lib.W_PER_CHANNEL, "per_tensor": _lib.W_PER_TENSOR,
                "per_group": _lib.W_PER_GROUP, "per_group_unsorted": _lib.W_PER_GROUP_UNSORTED,
                "per_group_mean3std": _lib.W_PER_GROUP_MEAN3STD, "none": _lib.W_NONE}


def _p(t: Optional[torch.Tensor]):
    """Device pointer of t for the C-ABI (every kernel operand lives in HBM: a host tensor
    here would be dereferenced by the GPU, so it is refused)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise RuntimeError(f"kernel operand on {t.device}: every operand must be on the GPU")
    return ctypes.c_void_p(t.data_ptr())


def _stream(t: torch.Tensor):
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


# the current stream's handle as an int (torch.cuda.current_stream builds a Stream object: 1.8 us
# against 0.1 us, a fifth of a few-row call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
# A device's default stream has the null handle, which names no device: the few-row and expert
# calls, the modules' forward and packing make their tensors' device current first where it is not
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def on_device(device: torch.device):
    """A context in which `device` (a tensor's) is the current one."""
    if device.type != "cuda" or device.index == _current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def on_tensor_device(fn):
    """fn(tensor, ...) with the tensor's device current."""
    first = fn.__code__.co_varnames[0]

    @functools.wraps(fn)
    def call(*args, **kw):
        t = args[0] if args else kw.get(first)
        if isinstance(t, torch.Tensor) and t.is_cuda and t.device.index != _current_device():
            with torch.cuda.device(t.device):
                return fn(*args, **kw)
        return fn(*args, **kw)
    return call


def _keep(pw, name: str, value):
    """value, kept as pw.<name> for later calls -- not inside a HIP-graph capture, where what was
    built is written at the graph's replays only."""
    if not torch.cuda.is_current_stream_capturing():
        setattr(pw, name, value)
    return value


def written(t: torch.Tensor) -> torch.Tensor:
    """t, after a kernel wrote it through its address: its version counter rises as for a write of
    torch's own, so that what is kept for its former contents (statistics, operands and outputs of
    layers on the same tensor) is not used for the new ones."""
    torch.autograd.graph.increment_version(t)
    return t


def _require_gpu(t: torch.Tensor, what: str):
    if t.device.type != "cuda":
        raise RuntimeError(
            f"{what}: tensors must live on a ROCm GPU (got {t.device}); the W4A4 operator is "
            "implemented only as HIP kernels for gfx950")


def _dtype_code(dt: torch.dtype) -> int:
    if dt not in DTYPE_CODE:
        raise ValueError(f"unsupported dtype {dt}; expected float32, float16 or bfloat16")
    return DTYPE_CODE[dt]


def pad_n(N: int) -> int:
    """Np = roundup(N, 256): rows of the packed codes and stride of the scale rows."""
    return (N + 255) // 256 * 256


def geometry(K: int, S: int, wmode: int, group_size: int):
    """(Kp, Gw, ngw, S_pad) of a packed weight (host only)."""
    out = [ctypes.c_int() for _ in range(4)]
    check(load().sqmp_weight_geometry(K, S, wmode, group_size, *[ctypes.byref(o) for o in out]),
          "weight geometry")
    return tuple(o.value for o in out)


@dataclass
class PackedWeight:
    """Device buffers of one packed W4A4 weight (layout: include/sqmp_w4a4.h)."""
    codes: torch.Tensor          # uint8 [Np, Kp/2] bpack (4-bit), int8-as-uint8 [Np, Kp] (8-bit), D [Np, Kp] (none)
    wscale: torch.Tensor         # D [ngw, Np]
    wsal: torch.Tensor           # D [N, S_pad]
    perm: torch.Tensor           # int32 [Kp]
    amap: torch.Tensor           # int32 [Kp]
    amap_fq: torch.Tensor        # int32 [K]
    nonsal: torch.Tensor         # int32 [max(K-S,1)]
    salient: Optional[torch.Tensor]  # int32 [S] or None
    N: int
    K: int
    S: int
    S_pad: int
    Kp: int
    Gw: int
    ngw: int
    n_bits: int                  # 4 / 8, or 0 for a dense D operand
    wmode: int
    dtype: torch.dtype
    dense: Optional[torch.Tensor] = field(default=None)  # packed-order D operand for fine groups
    posmap: Optional[torch.Tensor] = field(default=None)  # int32 [K]: packed position of column k
    sal_key: Optional[tuple] = field(default=None)        # identity of the salient set (host)
    w8: Optional[torch.Tensor] = field(default=None)     # uint8 [Np, Kp] e4m3 codes (f8 GEMM)
    ws32: Optional[torch.Tensor] = field(default=None)   # fp32 [ngw, Np] scales (f8 GEMM)
    # (codes_t, scale_t, sal_t, J) of gemm_fq7; like gemv's below derived from the codes and not
    # handed to the copy that dataclasses.replace makes, whose codes may be others
    fq7: Optional[tuple] = field(default=None, init=False)
    h2: Optional[tuple] = field(default=None)            # (f16 [2, Np, L], int32 [Np]) (gemm_h2)
    h2d: Optional[torch.Tensor] = field(default=None)    # f16 tile-major planes (gemm_h2d)
    sib_maps: Optional[tuple] = field(default=None)      # sibling position map (sqmp_permute_act)
    ident: Optional[bool] = field(default=None)          # packed order == column order (identity_layout)
    gemv: Optional[tuple] = field(default=None, init=False)       # (codes_t, scale_t, sal_t) of gemv
    gemv_args: Optional[tuple] = field(default=None, init=False)  # what gemv passes for this weight

    def __getstate__(self):
        """Copies and pickles (another device, another process) gather gemv's arguments anew."""
        return dict(self.__dict__, gemv_args=None)

    @property
    def gemm_operand(self):
        """(B operand, n_bits) for sqmp_gemm_fq."""
        if self.dense is not None:
            return self.dense, 0
        return self.codes, self.n_bits


def build_maps(K: int, salient: Optional[torch.Tensor], device, Kp: Optional[int] = None):
    """Identity-order index maps (perm, amap, amap_fq, nonsal) for K columns."""
    S = 0 if salient is None else int(salient.numel())
    Kp = K if Kp is None else Kp
    i32 = dict(dtype=torch.int32, device=device)
    perm = torch.empty(Kp, **i32)
    amap = torch.empty(Kp, **i32)
    amap_fq = torch.empty(K, **i32)
    nonsal = torch.empty(max(K - S, 1), **i32)
    ref = amap_fq
    with on_device(ref.device):
        check(load().sqmp_build_maps(K, _p(salient), S, _p(perm), _p(amap), _p(amap_fq), _p(nonsal),
                                     Kp, _stream(ref)), "build maps")
    return perm, amap, amap_fq, nonsal


@on_tensor_device
def pack_weight(w: torch.Tensor, weight_quant: str, n_bits: int, group_size: int,
                salient: Optional[torch.Tensor]) -> PackedWeight:
    """Quantize + pack W [N, K] (fake_quant.py:324-371 without the module bookkeeping)."""
    _require_gpu(w, "pack_weight")
    if weight_quant not in WEIGHT_MODES:
        raise ValueError(f"Invalid weight_quant: {weight_quant}")
    wmode = WEIGHT_MODES[weight_quant]
    w = w.contiguous()
    N, K = w.shape
    dt = _dtype_code(w.dtype)
    sal = None
    if salient is not None and salient.numel() > 0:
        sal = salient.to(device=w.device, dtype=torch.int32).contiguous()
    S = 0 if sal is None else sal.numel()
    Kp, Gw, ngw, S_pad = geometry(K, S, wmode, group_size)
    Np = pad_n(N)  # weight rows padded to one fast-GEMM N tile (include/sqmp_w4a4.h)
    if wmode == _lib.W_NONE:
        n_bits_eff = 0
        codes = torch.zeros((Np, Kp), dtype=w.dtype, device=w.device)
    else:
        if n_bits not in (4, 8):
            raise ValueError(f"quant_bits={n_bits}: packed weights support 4 or 8 bits")
        n_bits_eff = n_bits
        codes = torch.zeros((Np, Kp * n_bits // 8), dtype=torch.uint8, device=w.device)
    wscale = torch.zeros((ngw, Np), dtype=w.dtype, device=w.device)  # [ngw][Np]
    wsal = torch.empty((N, max(S_pad, 0)), dtype=w.dtype, device=w.device)
    i32 = dict(dtype=torch.int32, device=w.device)
    perm, amap = torch.empty(Kp, **i32), torch.empty(Kp, **i32)
    amap_fq, nonsal = torch.empty(K, **i32), torch.empty(max(K - S, 1), **i32)
    lib = load()
    ws_bytes = lib.sqmp_pack_workspace_bytes(N, K)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=w.device)
    check(lib.sqmp_pack_weight(_p(w), dt, N, K, wmode, n_bits, group_size, _p(sal), S,
                               _p(codes), _p(wscale), _p(wsal) if S_pad else None, _p(perm),
                               _p(amap), _p(amap_fq), _p(nonsal), _p(ws), ws_bytes, _stream(w)),
          "pack_weight")
    pw = PackedWeight(codes, wscale, wsal, perm, amap, amap_fq, nonsal, sal, N, K, S, S_pad, Kp,
                      Gw, ngw, n_bits_eff, wmode, w.dtype)
    pw.posmap = build_posmap(perm, K)
    pw.sal_key = salient_key(K, salient)
    identity_layout(pw)
    epc = 4 if w.dtype == torch.float32 else 8
    if n_bits_eff and Gw % epc != 0:
        # groups finer than one 16-B chunk: keep a dense packed-order operand for the GEMM
        pw.dense = dequant_weight_packed(pw)
    return pw


def identity_layout(pw: PackedWeight) -> bool:
    """Whether the GEMM's activation operand [M, Kp + S_pad] is x_hat in the input's own column
    order: no salient column, no padding position, the identity packed order (per_channel /
    per_tensor / unsorted weights without salient channels, the reference's ppl_eval flow).
    Then the in-place act quantizer's result (fake_quant.py:56-75 on the caller's x) IS the
    operand.  Decided once per packed weight, at pack time or at the first forward outside a
    HIP-graph capture (the check reads the order back); False while capturing."""
    if pw.ident is None:
        if pw.S != 0 or pw.S_pad != 0 or pw.Kp != pw.K:
            pw.ident = False
        elif torch.cuda.is_current_stream_capturing():
            return False
        else:
            pw.ident = bool(torch.equal(pw.perm[:pw.K].long(),
                                        torch.arange(pw.K, device=pw.perm.device)))
    return pw.ident


def build_posmap(perm: torch.Tensor, K: int) -> torch.Tensor:
    """Inverse of the packed order: posmap[k] = p with perm[p] == k (int32 [K])."""
    pos = torch.arange(perm.numel(), dtype=torch.int32, device=perm.device)
    valid = perm >= 0
    out = torch.empty(K, dtype=torch.int32, device=perm.device)
    out[perm[valid].long()] = pos[valid]
    return out


def salient_key(K: int, salient: Optional[torch.Tensor]) -> tuple:
    """Host-side identity of a salient set (equal sets -> equal keys)."""
    if salient is None or salient.numel() == 0:
        return (K, 0, 0)
    s = salient.detach().to("cpu", torch.int64)
    return (K, int(s.numel()), hash(s.numpy().tobytes()))


def dequant_weight_packed(pw: PackedWeight) -> torch.Tensor:
    out = torch.empty((pw.N, pw.Kp), dtype=pw.dtype, device=pw.codes.device)
    with on_device(pw.codes.device):
        check(load().sqmp_dequant_weight_packed(_p(pw.codes), _p(pw.wscale), _dtype_code(pw.dtype),
                                                pw.N, pw.Kp, pw.Gw, pw.ngw, pw.n_bits, _p(out),
                                                _stream(out)), "dequant_weight_packed")
    return out


def dequant_weight(pw: PackedWeight) -> torch.Tensor:
    """The reference's `weight` buffer: W_hat [N, K] in D (salient columns exact)."""
    _require_gpu(pw.codes, "dequant_weight")
    w_hat = torch.zeros((pw.N, pw.K), dtype=pw.dtype, device=pw.codes.device)
    with on_device(pw.codes.device):
        check(load().sqmp_dequant_weight(_p(pw.codes), _p(pw.wscale), _p(pw.wsal) if pw.S_pad else None,
                                         _p(pw.amap), _p(pw.salient), _dtype_code(pw.dtype), pw.N,
                                         pw.K, pw.S, pw.n_bits, pw.Kp, pw.Gw, pw.ngw, pw.S_pad,
                                         _p(w_hat), _stream(w_hat)), "dequant_weight")
    return w_hat


def _pad_rows(M: int) -> int:
    """Activation operands are allocated with rows padded to the GEMM's 256-row tile."""
    return max(256, (M + 255) // 256 * 256)


def padded_operand(t2: torch.Tensor) -> torch.Tensor:
    """An M-row view of a copy of t [M, L] in an allocation of _pad_rows(M) rows (the row
    padding the GEMMs' LDS-DMA tiles read past M)."""
    a = torch.empty((_pad_rows(t2.shape[0]), t2.shape[1]), dtype=t2.dtype, device=t2.device)
    a[:t2.shape[0]].copy_(t2)
    return a[:t2.shape[0]]


def _act_workspace(M: int, K: int, Kp: int, device):
    n = load().sqmp_act_workspace_bytes(M, K, Kp)
    return torch.empty(n, dtype=torch.uint8, device=device), n


# Persistent activation workspaces in the clean-workspace protocol of sqmp_quant_act_v2
# (allocated zeroed; every call leaves its statistics regions zero), plus the identity of
# the batch statistics each currently holds (for SQMP_QA_REUSE_STATS).  The region layout
# depends on (K, Kp), so one workspace per (device, stream, K, Kp): a region one layout
# leaves non-zero is never a must-be-zero region of another.  A HIP-graph capture has
# workspaces of its own, cleared by every replay: graphs are replayed in any order and on any
# stream, behind this bookkeeping, and share neither memory nor statistics with each other or with
# eager calls (the clearing costs a replay 2-3 us per layout).
_WS = {}
_SORTED = ("per_group", "per_group_mean3std")


_WSB = {}


def _ws_bytes(M: int, K: int, Kp: int) -> int:
    """sqmp_act_workspace_bytes, memoized per shape (saves a ctypes call per forward)."""
    n = _WSB.get((M, K, Kp))
    if n is None:
        n = _WSB[(M, K, Kp)] = load().sqmp_act_workspace_bytes(M, K, Kp)
    return n


def capture_id(stream_ptr: int) -> int:
    """Which HIP-graph capture the stream is in (0: none)."""
    return load().sqmp_capture_id(stream_ptr) if stream_ptr else 0


def _act_ws(device, stream_ptr: int, K: int, Kp: int, nbytes: int, tag: str = "in"):
    # tag "out": the in-place output quantizer has workspaces of its own, so quantizing a
    # layer's output (OPT q/k/v) leaves the input statistics for its sibling layers intact
    capture = capture_id(stream_ptr)
    key = (device.index, stream_ptr, K, Kp, tag, capture != 0)
    e = _WS.get(key)
    if e is None or e["buf"].numel() < nbytes or e["capture"] != capture:
        e = {"buf": torch.zeros(nbytes, dtype=torch.uint8, device=device), "stats": None,
             "capture": capture}
        _WS[key] = e
    return e


def _discard_ws(e):
    """A failed call may have left the workspace dirty: the next one starts with another."""
    e["capture"] = None


# Sibling operand reuse (sqmp_permute_act): a layer that quantizes the same input as the
# previous call, with the same salient set, act mode, bits and group size (q/k/v, gate/up),
# gets the previous operand with its positions moved into its own packed order instead of a
# table build + quantizer pass.  Operands up to SIB_MAX_BYTES are kept for this.
SIB_REUSE = os.environ.get("SQMP_SIB_REUSE", "1") == "1"
SIB_MAX_BYTES = 64 << 20


def _sibling_map(src: PackedWeight, dst: PackedWeight) -> torch.Tensor:
    """int32 [Kp]: the packed position in `src` of the column at each packed position of
    `dst` (-1 at dst's salient / padding positions), cached on dst for this exact `src`
    object and the current contents of both orders (a PackedWeight is rebuilt whenever a
    module's buffers change; the perm / amap versions catch in-place rewrites)."""
    if src.posmap is None:
        src.posmap = build_posmap(src.perm, src.K)
    ver = (src.perm._version, src.posmap._version, dst.amap._version)
    c = dst.sib_maps
    if c is not None and c[0]() is src and c[1] == ver:
        return c[2]
    col = dst.amap.long()
    m = torch.where(col >= 0, src.posmap.long()[col.clamp(min=0)], -1).to(torch.int32)
    return _keep(dst, "sib_maps", (weakref.ref(src), ver, m))[2]  # one source per layer (its leader)


def _sibling_ok(src: PackedWeight, dst: PackedWeight) -> bool:
    return (src is not dst and src.K == dst.K and src.S == dst.S and src.Kp == dst.Kp
            and src.S_pad == dst.S_pad and src.sal_key == dst.sal_key and src.dtype == dst.dtype
            and dst.dtype in (torch.float16, torch.bfloat16) and (dst.Kp + dst.S_pad) <= 8192)


def quant_act_fp(x2: torch.Tensor, pw: PackedWeight, act_quant: str, n_bits: int,
                 group_size: int, stats_of: Optional[torch.Tensor] = None, h2: bool = False):
    """x [M, K] -> A [M, Kp + S_pad] in D: x_hat in packed order + exact salient tail.

    The returned tensor is an M-row view of an allocation padded to a multiple of 256 rows
    (the GEMM stages whole 256-row tiles by LDS-DMA; rows >= M are never stored).

    stats_of: the tensor whose identity names this batch (the module's input x).  Layers
    that quantize the same x with the same salient set and sort (q/k/v, gate/up) reuse the
    first call's column statistics and rank instead of recomputing them.

    h2 (fp32, h2_planes_ok): the same values as sqmp_gemm_h2d's operand instead, written by
    the quantizer itself (SQMP_OUT_H2): (f16 planes [2, roundup(M, 128), L], int32 row
    exponents, M) -- bit-identical to sqmp_split2_f16 of the fp32 A."""
    _require_gpu(x2, "quant_act")
    M, K = x2.shape
    L = pw.Kp + pw.S_pad
    if h2:
        ldr = (M + 127) // 128 * 128
        planes = torch.empty((2, ldr, L), dtype=torch.float16, device=x2.device)
        aexp = torch.empty(max(ldr, 1), dtype=torch.int32, device=x2.device)
        a = planes
    else:
        a = torch.empty((_pad_rows(M), L), dtype=x2.dtype, device=x2.device)[:M]
    lib = load()
    nb = _ws_bytes(M, K, pw.Kp)
    stream = torch.cuda.current_stream(x2.device).cuda_stream
    e = _act_ws(x2.device, stream, K, pw.Kp, nb)
    flags = _lib.QA_CLEAN_WS
    skey = None
    if act_quant in _SORTED:
        src = x2 if stats_of is None else stats_of
        skey = (src.data_ptr(), tuple(src.shape), src.dtype, src._version, pw.sal_key,
                act_quant, M, K)
        la = e.get("last_a")
        if (not h2 and SIB_REUSE and la is not None and la[0]() is src
                and la[1] == skey + (n_bits, group_size)
                and la[2]() is not None and _sibling_ok(la[2](), pw)):
            # a sibling of the layer that produced la[3] on this same input
            moves = _sibling_map(la[2](), pw)
            check(lib.sqmp_permute_act(_p(la[3]), _p(a), _p(moves), _dtype_code(x2.dtype), M, pw.Kp,
                                       pw.S_pad, ctypes.c_void_p(stream)), "permute_act")
            return a
        st = e["stats"]
        # only a DIFFERENT layer on the same input reuses them: calling one layer again
        # (e.g. a benchmark loop) always recomputes its statistics
        if (st is not None and st[0]() is src and st[1] == skey
                and st[2] != pw.codes.data_ptr()):
            flags |= _lib.QA_REUSE_STATS
    if pw.posmap is None:
        pw.posmap = build_posmap(pw.perm, K)
    status = lib.sqmp_quant_act_v2(_p(x2), _dtype_code(x2.dtype), M, K, ACT_MODES[act_quant],
                                   n_bits, group_size, _p(pw.amap), pw.Kp, _p(pw.nonsal),
                                   _p(pw.salient), pw.S, pw.S_pad, _p(pw.posmap), flags,
                                   _lib.OUT_H2 if h2 else _lib.OUT_FP, _p(a),
                                   _p(aexp) if h2 else None, None, _p(e["buf"]),
                                   e["buf"].numel(), ctypes.c_void_p(stream))
    if status != _lib.SQMP_OK:
        _discard_ws(e)
        check(status, "quant_act")
    if skey is not None:
        e["stats"] = (weakref.ref(stats_of if stats_of is not None else x2), skey,
                      pw.codes.data_ptr())
        e["last_a"] = None
        if not h2 and SIB_REUSE and a.numel() * a.element_size() <= SIB_MAX_BYTES:
            # held while the input lives: freeing the input drops the operand with it
            e["last_a"] = (weakref.ref(stats_of if stats_of is not None else x2, _drop_last_a(e)),
                           skey + (n_bits, group_size), weakref.ref(pw), a)
    return (planes, aexp, M) if h2 else a


def _drop_last_a(e):
    """weakref callback: the input a kept sibling operand belongs to was freed."""
    def cb(ref):
        la = e.get("last_a")
        if la is not None and la[0] is ref:
            e["last_a"] = None
    return cb


def quant_act_fp_group(x2: torch.Tensor, pws, act_quant: str, n_bits: int,
                       group_size: int):
    """x [M, K] -> [A_0, ..., A_{n-1}]: quant_act_fp's operand for each packed weight of
    `pws` (sibling layers: same K, Kp, S_pad and salient set), from ONE quantizer pass
    (sqmp_quant_act_group); every A_o is bit-identical to quant_act_fp(x2, pws[o], ...)."""
    _require_gpu(x2, "quant_act_group")
    M, K = x2.shape
    p0 = pws[0]
    outs = [torch.empty((_pad_rows(M), p0.Kp + p0.S_pad), dtype=x2.dtype, device=x2.device)[:M]
            for _ in pws]
    for pw in pws:
        if pw.posmap is None:
            pw.posmap = build_posmap(pw.perm, K)
    n = len(pws)
    vp = ctypes.c_void_p
    amaps = (vp * n)(*[t.data_ptr() for t in (pw.amap for pw in pws)])
    posmaps = (vp * n)(*[pw.posmap.data_ptr() for pw in pws])
    optr = (vp * n)(*[t.data_ptr() for t in outs])
    lib = load()
    nb = _ws_bytes(M, K, p0.Kp)
    stream = torch.cuda.current_stream(x2.device).cuda_stream
    e = _act_ws(x2.device, stream, K, p0.Kp, nb)
    status = lib.sqmp_quant_act_group(_p(x2), _dtype_code(x2.dtype), M, K, ACT_MODES[act_quant],
                                      n_bits, group_size, n, amaps, posmaps, p0.Kp,
                                      _p(p0.nonsal), _p(p0.salient), p0.S, p0.S_pad,
                                      _lib.QA_CLEAN_WS, optr, _p(e["buf"]), e["buf"].numel(),
                                      vp(stream))
    if status != _lib.SQMP_OK:
        _discard_ws(e)
        check(status, "quant_act_group")
    # the workspace's sorted column list now describes x2 (a later sibling call on x2 may
    # reuse it); no operand is kept for sqmp_permute_act
    e["stats"] = (weakref.ref(x2), (x2.data_ptr(), tuple(x2.shape), x2.dtype, x2._version,
                                    p0.sal_key, act_quant, M, K), p0.codes.data_ptr())
    e["last_a"] = None
    return outs


def gemm_fq7_group(As, pws, biases):
    """[y_0, ..., y_{n-1}] with y_o = gemm_fq7(As[o], pws[o], biases[o]) in one launch
    (sqmp_gemm_fq7_group): bit for bit, unless only one of the two takes the K split inside the
    workgroup (fq7_plan, OPT bit 16) -- then within fp32 rounding of the partial sums."""
    M = As[0].shape[0]
    p0 = pws[0]
    n = len(pws)
    probs = (_lib.Fq7Problem * n)()
    ys, held = [], []  # (operands that a capture builds live in this call alone)
    for o, (a, pw, b) in enumerate(zip(As, pws, biases)):
        held.append(fq7_operands(pw))
        bt, st, salt, J = held[-1]
        y = torch.empty((M, pw.N), dtype=pw.dtype, device=a.device)
        ys.append(y)
        _require_gpu(a, "gemm_fq7_group")
        probs[o] = _lib.Fq7Problem(a.data_ptr(), bt.data_ptr(), st.data_ptr(), salt.data_ptr(),
                                   None if b is None else b.data_ptr(), y.data_ptr(), None,
                                   pw.N)
    check(load().sqmp_gemm_fq7_group(probs, n, _dtype_code(p0.dtype), M, p0.Kp, p0.S_pad, p0.Gw,
                                     p0.ngw, FQ7_J, _stream(As[0])), "gemm_fq7_group")
    return ys


def fq7_plan(pws, M: int, group: bool):
    """(row-tile height, OPT bits) of the packed-order launch sqmp_gemm_fq7 would take for
    pws[0] alone (group False) or sqmp_gemm_fq7_group for all of pws: OPT bit 16 (the K split
    inside the workgroup) adds the fp32 partial sums in another order."""
    p0 = pws[0]
    n = len(pws) if group else 1
    Ns = (ctypes.c_int * n)(*[pw.N for pw in pws[:n]])
    tm, opt = ctypes.c_int(), ctypes.c_int()
    check(load().sqmp_fq7_plan(_dtype_code(p0.dtype), M, Ns, n if group else 0, p0.Kp, p0.Gw,
                               FQ7_J, ctypes.byref(tm), ctypes.byref(opt)), "fq7_plan")
    return tm.value, opt.value


def group_eligible(pws, act_quant: str, act_bits: int, group_size: int, M: int) -> bool:
    """Whether quant_act_fp_group + gemm_fq7_group compute these sibling layers: sorted
    per_group activations of <= 8 bits in power-of-two groups of 16 .. 1024 on the
    packed-order path (below FQT_MIN_ROWS rows), 4-bit fq7 weights in whole 64-blocks per
    group, 4 (Kp + S_pad + 8) bytes of quantizer LDS per member (+ 4 S_pad) within 150 KiB, one K
    (<= 16384, % 8 == 0) / Kp / S_pad / group geometry / salient set / dtype
    (fp16 / bf16) for all, 2 or 3 layers."""
    # (mirrors what sqmp_quant_act_group / sqmp_gemm_fq7_group accept, so that a refusal
    # never reaches the library: a non-empty batch, 2..8-bit codes, J = 2 tiles)
    if not 2 <= len(pws) <= 3 or act_quant not in _SORTED or not 2 <= act_bits <= 8:
        return False
    if M <= 0 or FQ7_J != 2:
        return False
    if not 16 <= group_size <= 1024 or group_size & (group_size - 1):
        return False
    if pws[0].K > 16384 or pws[0].K % 8:
        return False
    if FQT_MODE == "1" or (FQT_MODE == "auto" and M >= FQT_MIN_ROWS):
        return False
    p0 = pws[0]
    if not FQ7_AUTO or p0.dtype not in (torch.float16, torch.bfloat16) or p0.K - p0.S <= 0:
        return False
    # the quantizer holds one LDS region of Kp + S_pad + 8 words per member + the salient list / masks
    if not lc_lds_ok(p0.Kp, p0.S_pad, len(pws)):
        return False
    return all(fq7_eligible(pw) and pw.Gw % 64 == 0 and pw.K == p0.K and pw.Kp == p0.Kp
               and pw.S_pad == p0.S_pad and pw.S == p0.S and pw.Gw == p0.Gw
               and pw.ngw == p0.ngw and pw.sal_key == p0.sal_key and pw.dtype == p0.dtype
               for pw in pws)


# Activation-order path (SQMP_OUT_C4 + sqmp_perm_weight_c4 + sqmp_gemm_fqt) for sorted
# per_group activations: the GEMM runs over the K - S non-salient positions in activation
# order instead of the Kp packed positions (which carry S zero salient positions), and the
# quantizer writes 4-bit codes instead of D values.  It rebuilds the permuted weight per
# forward (N x (Kq + S_pad) D values), so it pays from FQT_MIN_ROWS rows on.
FQT_MODE = os.environ.get("SQMP_FQT", "auto")   # "auto" | "1" (whenever eligible) | "0"
# from 16384 rows: with fq7 as the packed-order GEMM, the packed order wins at 8192 rows (Llama
# layer forward 3267 vs 3587 us) and the activation order at 16384 (config 2: 0.536 vs 0.556 ms)
FQT_MIN_ROWS = int(os.environ.get("SQMP_FQT_MIN_ROWS", "16384"))
# the activation-order GEMM on fq7's structure (sqmp_gemm_fqt7: tile-major activation
# operands written by the quantizer) when Kq % 128 == 0, else on fq6's (sqmp_gemm_fqt)
FQT7 = os.environ.get("SQMP_FQT7", "1") == "1"
# its register operand's row tiles per wave: 2 (256 weight rows x 256 tokens per tile) or 4
# (128 x 512: half the permuted-weight LDS traffic per MFMA, twice the act-code decode)
FQT7_J = int(os.environ.get("SQMP_FQT7_J", "2"))


def _fqt_j() -> int:
    """Tile-major operand layout of the activation-order path (FQT7_J: 2 or 4)."""
    return FQT7_J if FQT7_J in (2, 4) else 2


def lc_lds_ok(P: int, S_pad: int, nout: int = 1) -> bool:
    """The lane-contiguous quantizer's LDS budget (quant_lc_supported / lc_lds_words in
    sqmp_actquant_lc.hip): min(nout, 2) regions of P + S_pad + 8 words (a third sibling
    output reuses the second region), the salient list and two mask words per 64-position
    chunk, within 150 KiB; P + S_pad < 65536 (16-bit table positions).  Every Python-side
    eligibility check that leads to that kernel applies it, so that a layer the library would
    refuse (EUNSUPPORTED) takes another path instead of raising."""
    nr = min(nout, 2)
    return (4 * ((P + S_pad + 8) * nr + S_pad + 2 * ((P + 63) // 64)) <= 150 * 1024
            and P + S_pad < 65536)


def fqt_eligible(pw: PackedWeight, act_quant: str, act_bits: int, group_size: int,
                 M: int, force: bool = False) -> bool:
    """Whether the activation-order path computes this layer (force: kernel="fqt", no row
    threshold)."""
    if not force and (FQT_MODE == "0" or (FQT_MODE == "auto" and M < FQT_MIN_ROWS)):
        return False
    # the C4 quantizer's limits (quant_lc_supported in sqmp_actquant_lc.hip): power-of-two
    # groups of 64 .. 64 * LC_RPL = 1024 ranks (a group never straddles a wave's ranks)
    return (act_quant in _SORTED or act_quant == "per_group_unsorted") and act_bits <= 4 \
        and pw.n_bits == 4 and pw.dense is None and pw.dtype != torch.float32 \
        and 64 <= group_size <= 1024 and group_size & (group_size - 1) == 0 \
        and pw.N % 8 == 0 and pw.K % 8 == 0 and pw.K <= 16384 and pw.K - pw.S > 0 \
        and lc_lds_ok(pw.Kp, pw.S_pad)


def quant_act_c4(x2: torch.Tensor, pw: PackedWeight, act_quant: str, n_bits: int,
                 group_size: int, stats_of: Optional[torch.Tensor] = None):
    """x [M, K] -> the activation-order operands of gemm_fqt: (int4 codes [M, Kq/2] bytes,
    D group scales [Kq/G, Mp], exact salient x [M, S_pad], permuted weight [Np, Kq + S_pad])
    with Kq = roundup(K - S, 64).  With FQT7 and Kq % 128 == 0 the first three are in
    sqmp_gemm_fqt7's tile-major layouts (SQMP_QA_TILED / _TILED4 for FQT7_J = 2 / 4): codes
    [R, Kq/2], scales [R/(16 J), Kq/G, 16 J] (3-d marks the layout), xs [R, S_pad][:M],
    R = roundup(M, 128 J).
    Statistics reuse as quant_act_fp."""
    _require_gpu(x2, "quant_act")
    M, K = x2.shape
    Mp = _pad_rows(M)
    Kn = K - pw.S
    Kq = (Kn + 63) // 64 * 64
    ngq = (Kn + group_size - 1) // group_size
    dev = x2.device
    tiled = FQT7 and Kq % 128 == 0
    tj = _fqt_j()
    if tiled:
        R = max(128 * tj, (M + 128 * tj - 1) // (128 * tj) * (128 * tj))
        codes = torch.empty((R, Kq // 2), dtype=torch.uint8, device=dev)
        scales = torch.empty((R // (16 * tj), ngq, 16 * tj), dtype=x2.dtype, device=dev)
        xs = torch.empty((R, max(pw.S_pad, 64)), dtype=x2.dtype, device=dev)[:M]
    else:
        codes = torch.empty((Mp, Kq // 2), dtype=torch.uint8, device=dev)[:M]
        scales = torch.empty((ngq, Mp), dtype=x2.dtype, device=dev)
        xs = torch.empty((Mp, max(pw.S_pad, 8)), dtype=x2.dtype, device=dev)[:M]
    lib = load()
    nb = _ws_bytes(M, K, pw.Kp)
    stream = torch.cuda.current_stream(dev).cuda_stream
    e = _act_ws(dev, stream, K, pw.Kp, nb)
    flags = _lib.QA_CLEAN_WS | ((_lib.QA_TILED4 if tj == 4 else _lib.QA_TILED) if tiled else 0)
    src = x2 if stats_of is None else stats_of
    skey = (src.data_ptr(), tuple(src.shape), src.dtype, src._version, pw.sal_key, act_quant,
            M, K)
    st = e["stats"]
    if (act_quant in _SORTED and st is not None and st[0]() is src and st[1] == skey
            and st[2] != pw.codes.data_ptr()):
        flags |= _lib.QA_REUSE_STATS
    if pw.posmap is None:
        pw.posmap = build_posmap(pw.perm, K)
    wp = torch.empty((pad_n(pw.N), Kq + pw.S_pad), dtype=pw.dtype, device=dev)
    # one call: quantizer + weight permutation in the same launch
    status = lib.sqmp_quant_act_c4(_p(x2), _dtype_code(x2.dtype), M, K, ACT_MODES[act_quant],
                                   n_bits, group_size, _p(pw.amap), pw.Kp, _p(pw.nonsal),
                                   _p(pw.salient), pw.S, pw.S_pad, _p(pw.posmap), flags,
                                   _p(codes), _p(scales), _p(xs) if pw.S_pad else None,
                                   _p(pw.codes), _p(pw.wscale), _p(pw.wsal) if pw.S_pad else None,
                                   pw.N, pw.Gw, pw.ngw, _p(wp), _p(e["buf"]), e["buf"].numel(),
                                   ctypes.c_void_p(stream))
    if status != _lib.SQMP_OK:
        _discard_ws(e)
        check(status, "quant_act_c4")
    if act_quant in _SORTED:
        e["stats"] = (weakref.ref(src), skey, pw.codes.data_ptr())
    return codes, scales, xs, wp


def gemm_fqt(codes: torch.Tensor, scales: torch.Tensor, xs: torch.Tensor, wp: torch.Tensor,
             pw: PackedWeight, bias: Optional[torch.Tensor], group_size: int,
             colmax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = D(x_hat . W_hat^T + bias) on the activation-order operands of quant_act_c4.
    colmax (tile-major operands only): as gemm_fq's fused output-quant statistics."""
    M = xs.shape[0]
    y = torch.empty((M, pw.N), dtype=pw.dtype, device=codes.device)
    Kq = codes.shape[1] * 2
    if scales.dim() == 3:   # tile-major (SQMP_QA_TILED: 32-row blocks, TILED4: 64-row)
        check(load().sqmp_gemm_fqt7j(_p(codes), _p(scales), _p(xs), _p(wp), _p(bias), _p(y),
                                     _dtype_code(pw.dtype), M, pw.N, Kq, pw.S_pad, group_size,
                                     scales.shape[1], scales.shape[2] // 16, _p(colmax),
                                     _stream(codes)), "gemm_fqt7")
        return y
    if colmax is not None:
        raise ValueError("gemm_fqt: fused column statistics need the tile-major operands")
    check(load().sqmp_gemm_fqt(_p(codes), _p(scales), _p(xs) if pw.S_pad else None, _p(wp),
                               _p(bias), _p(y), _dtype_code(pw.dtype), M, pw.N, Kq, pw.S_pad,
                               group_size, scales.shape[0], _stream(codes)), "gemm_fqt")
    return y


def out_quant_workspace(M: int, C: int, device):
    """The persistent workspace fake_quant_inplace uses for an [M, C] tensor on the current
    stream (its first C words: the column-maximum region sqmp_gemm_fq_colmax fills)."""
    nb = _ws_bytes(M, C, C)
    stream = torch.cuda.current_stream(device).cuda_stream
    return _act_ws(device, stream, C, C, nb, "out")


def fake_quant_inplace(t2: torch.Tensor, act_quant: str, n_bits: int, group_size: int,
                       amap_fq: torch.Tensor, nonsal: torch.Tensor, S: int,
                       stats_given: bool = False):
    """Fake-quantize t [M, C] in place; columns marked -2 in amap_fq pass through.
    stats_given: the workspace's column maxima were produced by the GEMM that wrote t
    (sqmp_gemm_fq_colmax; act modes per_group / per_tensor)."""
    _require_gpu(t2, "fake_quant")
    M, C = t2.shape
    lib = load()
    nb = lib.sqmp_act_workspace_bytes(M, C, C)
    stream = torch.cuda.current_stream(t2.device).cuda_stream
    e = _act_ws(t2.device, stream, C, C, nb, "out")
    flags = _lib.QA_CLEAN_WS | (_lib.QA_STATS_GIVEN if stats_given else 0)
    # the list table of the unsorted modes depends only on (C, the non-salient list, the
    # salient set): with no salient column the list is 0 .. C-1 (build_maps / pack_weight), so
    # every such call on this workspace builds the same table -- consecutive in-place
    # quantizers (the ppl_eval flow's inputs and q/k/v outputs) skip its launch
    # (SQMP_QA_TABLE_READY).  Not inside a HIP-graph capture.
    tab = (("list", C) if (S == 0 and M > 0 and act_quant in ("per_token", "per_group_unsorted"))
           else None)
    if tab is not None and not e["capture"] and e.get("tab") == tab:
        flags |= _lib.QA_TABLE_READY
    status = lib.sqmp_quant_act_v2(_p(t2), _dtype_code(t2.dtype), M, C, ACT_MODES[act_quant],
                                   n_bits, group_size, _p(amap_fq), C, _p(nonsal), None, S, 0,
                                   None, flags, _lib.OUT_INPLACE, None, None, None,
                                   _p(e["buf"]), e["buf"].numel(), ctypes.c_void_p(stream))
    if status != _lib.SQMP_OK:
        _discard_ws(e)
        check(status, "fake_quant")
    e["tab"] = tab  # (any other mode rebuilt or overwrote the table region)
    e["stats"] = None  # the sorted-column list now describes t2, not a layer input
    # the kernel wrote t2 through a raw pointer: bump its version counter so statistics
    # another workspace recorded for this (now quantized) tensor are not reused
    torch.autograd.graph.increment_version(t2)
    return t2


# Whether gemm_fq runs the register-operand kernel (sqmp_gemm_fq7) where fq7_eligible: on by
# default (same-box GEMM-only A/B, tools/gemm_ab.py: +8 to +10 % at the 2048-token Llama shapes,
# +2.7 % at config 2 in packed order); SQMP_FQ7=0 selects fq6.
FQ7_AUTO = os.environ.get("SQMP_FQ7", "1") == "1"
# weight rows per wave / 16: 4 -> 128 x 512 tiles, 2 -> 256 x 256 tiles
FQ7_J = int(os.environ.get("SQMP_FQ7_J", "2"))


def fq7_eligible(pw: PackedWeight) -> bool:
    """4-bit codes in whole-64-block or 32-wide groups, fp16/bf16, whole 16-B output chunks
    (sqmp_gemm_fq7)."""
    return (pw.n_bits == 4 and pw.dense is None and pw.dtype != torch.float32
            and (pw.Gw % 64 == 0 or pw.Gw == 32) and pw.N % 8 == 0)


def fq7_operands(pw: PackedWeight):
    """(codes_t, scale_t, sal_t, J) of gemm_fq7: tile-major copies of the packed weight, built
    once per packed weight."""
    if pw.fq7 is None or pw.fq7[3] != FQ7_J:
        sizes = [ctypes.c_size_t() for _ in range(3)]
        check(load().sqmp_fq7_sizes(pw.N, pw.Kp, pw.S_pad, pw.ngw, FQ7_J,
                                    *[ctypes.byref(v) for v in sizes]), "fq7_sizes")
        dev = pw.codes.device
        bt = torch.empty(sizes[0].value, dtype=torch.uint8, device=dev)
        st = torch.empty(sizes[1].value, dtype=pw.dtype, device=dev)
        salt = torch.empty(sizes[2].value, dtype=pw.dtype, device=dev)
        check(load().sqmp_pack_fq7(_p(pw.codes), _p(pw.wscale), _p(pw.wsal) if pw.S_pad else None,
                                   _dtype_code(pw.dtype), pw.N, pw.Kp, pw.S_pad, pw.ngw, FQ7_J,
                                   _p(bt), _p(st), _p(salt), _stream(pw.codes)), "pack_fq7")
        return _keep(pw, "fq7", (bt, st, salt, FQ7_J))
    return pw.fq7


def gemm_fq7(a: torch.Tensor, pw: PackedWeight, bias: Optional[torch.Tensor],
             colmax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gemm_fq on the register-operand kernel (same operands and numerics)."""
    M = a.shape[0]
    y = torch.empty((M, pw.N), dtype=pw.dtype, device=a.device)
    bt, st, salt, J = fq7_operands(pw)
    check(load().sqmp_gemm_fq7(_p(a), _p(bt), _p(st), _p(salt), _p(bias), _p(y),
                               _dtype_code(pw.dtype), M, pw.N, pw.Kp, pw.S_pad, pw.Gw, pw.ngw, J,
                               _p(colmax) if colmax is not None else None, _stream(a)),
          "gemm_fq7")
    return y


# The faithful GEMM of fp32 layers: "h2" (default) -- row-scaled two-piece fp16 splits on the
# f16 MFMA (sqmp_gemm_h2, 3 MFMAs per product); "f32" -- the f32 MFMA (1/16 of the bf16 rate).
F32_GEMM = os.environ.get("SQMP_F32_GEMM", "h2")


def _w_full(pw: PackedWeight) -> torch.Tensor:
    """fp32 [N, Kp + S_pad]: the packed-order W_hat + exact salient slice (the GEMM's B)."""
    w = pw.codes[:pw.N] if pw.n_bits == 0 and pw.dense is None else (
        pw.dense if pw.dense is not None else dequant_weight_packed(pw))
    full = torch.cat([w, pw.wsal], dim=1) if pw.S_pad else w
    return full.contiguous()


def h2_operand(pw: PackedWeight):
    """(f16 planes [2, Np, L], int32 row exponents [Np]) of the row-scaled packed-order
    W_hat + salient slice (sqmp_split2_f16), built once per packed fp32 weight."""
    if pw.h2 is None:
        full = _w_full(pw)
        Np, L = pad_n(pw.N), pw.Kp + pw.S_pad
        planes = torch.empty((2, Np, L), dtype=torch.float16, device=full.device)
        bexp = torch.empty(Np, dtype=torch.int32, device=full.device)
        check(load().sqmp_split2_f16(_p(full), pw.N, L, Np, _p(planes), _p(bexp), _stream(full)),
              "split2_f16")
        return _keep(pw, "h2", (planes, bexp))
    return pw.h2


# the fp32 GEMM on the LDS-DMA ring (sqmp_gemm_h2d: pre-split activation planes, weight planes
# in registers; bit-identical to sqmp_gemm_h2) wherever L % 64 == 0 and N % 4 == 0;
# SQMP_H2D=0 keeps sqmp_gemm_h2 (A/B)
H2D = os.environ.get("SQMP_H2D", "1") != "0"


def h2d_operand(pw: PackedWeight) -> torch.Tensor:
    """The weight planes of h2_operand in sqmp_gemm_h2d's tile-major register layout
    (sqmp_pack_h2d), built once per packed fp32 weight."""
    if pw.h2d is None:
        planes, _ = h2_operand(pw)
        wt = torch.empty_like(planes)
        check(load().sqmp_pack_h2d(_p(planes), planes.shape[1], planes.shape[2], _p(wt),
                                   _stream(planes)), "pack_h2d")
        return _keep(pw, "h2d", wt)
    return pw.h2d


def _h2d_rows_ok(M: int, L: int, N: int = 0) -> bool:
    """sqmp_gemm_h2d addresses both activation planes, and both weight planes (roundup(N, 256)
    rows), with 32-bit buffer offsets."""
    return (4 * ((M + 127) // 128 * 128) * L < (1 << 32)
            and 4 * ((N + 255) // 256 * 256) * L < (1 << 32))


_LC_OFF = False  # SQMP_DISABLE_LC: the library's knob, mirrored here (refreshed by reload_knobs)


def _read_lc_off():
    global _LC_OFF
    _LC_OFF = os.environ.get("SQMP_DISABLE_LC") is not None


_read_lc_off()
_lib.on_reload(_read_lc_off)


def h2_planes_ok(pw: PackedWeight, act_quant: str, M: int = 0, group_size: int = 0) -> bool:
    """Whether an fp32 layer's forward runs quantizer -> planes -> sqmp_gemm_h2d
    (quant_act_fp(h2=True) + gemm_h2_planes) instead of the fp32 operand + split: every
    condition under which the SQMP_OUT_H2 quantizer (sqmp_actquant.hip, the fp32 wave kernels)
    and sqmp_gemm_h2d accept the call -- a non-empty batch, the lane-contiguous pipeline on,
    the per-wave row buffer (4 K bytes + 12 bytes per act group) within 160 KiB, 32-bit
    plane offsets."""
    L = pw.Kp + pw.S_pad
    Kn = pw.K - pw.S
    ngroups = (Kn + group_size - 1) // group_size if act_quant.startswith("per_group") and group_size > 0 else 1
    wb = (4 * pw.K + 15) // 16 * 16 + (12 * ngroups + 15) // 16 * 16
    return (pw.dtype == torch.float32 and H2D and F32_GEMM == "h2" and L % 64 == 0
            and pw.N % 4 == 0 and pw.K % 8 == 0 and Kn > 0 and M > 0 and not _LC_OFF
            and wb <= 160 * 1024 and act_quant != "per_tensor" and _h2d_rows_ok(M, L, pw.N))


def gemm_h2_planes(a2, pw: PackedWeight, bias: Optional[torch.Tensor],
                   colmax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = A . W_hat^T + bias on sqmp_gemm_h2d from quant_act_fp(h2=True)'s planes."""
    planes, aexp, M = a2
    _, bexp = h2_operand(pw)
    wt = h2d_operand(pw)
    ldr, L = planes.shape[1], planes.shape[2]
    if L != pw.Kp + pw.S_pad:
        raise ValueError("gemm_h2_planes: operand width does not match the packed weight")
    y = torch.empty((M, pw.N), dtype=torch.float32, device=planes.device)
    check(load().sqmp_gemm_h2d(_p(planes), ldr, _p(aexp), _p(wt), _p(bexp), _p(bias), _p(y), M,
                               pw.N, L, _p(colmax) if colmax is not None else None,
                               _stream(planes)), "gemm_h2d")
    return y


def gemm_h2(a: torch.Tensor, pw: PackedWeight, bias: Optional[torch.Tensor],
            colmax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gemm_fq for fp32 layers on the f16 MFMA (include/sqmp_w4a4.h sqmp_gemm_h2d /
    sqmp_gemm_h2)."""
    M = a.shape[0]
    L = pw.Kp + pw.S_pad
    if a.dtype != torch.float32 or a.shape[1] != L or a.stride(0) != L:
        raise ValueError("gemm_h2: A must be fp32 [M, Kp + S_pad] with row stride Kp + S_pad")
    planes, bexp = h2_operand(pw)
    lib = load()
    if H2D and L % 64 == 0 and pw.N % 4 == 0 and M > 0 and _h2d_rows_ok(M, L, pw.N):
        wt = h2d_operand(pw)
        ldr = (M + 127) // 128 * 128
        a2 = torch.empty((2, ldr, L), dtype=torch.float16, device=a.device)
        aexp = torch.empty(ldr, dtype=torch.int32, device=a.device)
        check(lib.sqmp_split2_f16(_p(a), M, L, ldr, _p(a2), _p(aexp), _stream(a)), "split2_f16")
        y = torch.empty((M, pw.N), dtype=torch.float32, device=a.device)
        check(lib.sqmp_gemm_h2d(_p(a2), ldr, _p(aexp), _p(wt), _p(bexp), _p(bias), _p(y), M,
                                pw.N, L, _p(colmax) if colmax is not None else None,
                                _stream(a)), "gemm_h2d")
        return y
    aexp = torch.empty(max(M, 1), dtype=torch.int32, device=a.device)
    check(lib.sqmp_row_exp(_p(a), M, L, _p(aexp), _stream(a)), "row_exp")
    y = torch.empty((M, pw.N), dtype=torch.float32, device=a.device)
    check(lib.sqmp_gemm_h2(_p(a), _p(aexp), _p(planes), _p(bexp), _p(bias), _p(y), M, pw.N, L,
                           _p(colmax) if colmax is not None else None, _stream(a)), "gemm_h2")
    return y


def gemm_fq(a: torch.Tensor, pw: PackedWeight, bias: Optional[torch.Tensor],
            colmax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = D(A . W_hat^T + bias).  colmax: a zeroed uint32 buffer of >= N words that the
    epilogue max-reduces bits(|y|) per column into (fused output-quant statistics)."""
    if FQ7_AUTO and fq7_eligible(pw):
        return gemm_fq7(a, pw, bias, colmax)
    if pw.dtype == torch.float32 and F32_GEMM == "h2":
        return gemm_h2(a, pw, bias, colmax)
    M = a.shape[0]
    y = torch.empty((M, pw.N), dtype=pw.dtype, device=a.device)
    b_op, nb = pw.gemm_operand
    args = (_p(a), _p(b_op), _p(pw.wscale), _p(pw.wsal) if pw.S_pad else None, _p(bias), _p(y),
            _dtype_code(pw.dtype), M, pw.N, pw.Kp, pw.S_pad, pw.Gw, pw.ngw, nb)
    if colmax is None:
        check(load().sqmp_gemm_fq(*args, _stream(a)), "gemm_fq")
    else:
        check(load().sqmp_gemm_fq_colmax(*args, _p(colmax), _stream(a)), "gemm_fq")
    return y


def _ws32(pw: PackedWeight) -> torch.Tensor:
    """fp32 [ngw, Np] weight scales of the f8 GEMM, built once per packed weight."""
    if pw.ws32 is None:
        ws32 = torch.empty((pw.ngw, pad_n(pw.N)), dtype=torch.float32, device=pw.codes.device)
        check(load().sqmp_pack_f8(_p(pw.codes), _p(pw.wscale), _dtype_code(pw.dtype), pw.N,
                                  pw.Kp, pw.ngw, None, _p(ws32), _stream(pw.codes)), "pack_f8")
        return _keep(pw, "ws32", ws32)
    return pw.ws32


def f8_operands(pw: PackedWeight):
    """(w8, ws32) of the f8 GEMM, built once per packed weight."""
    ws32 = _ws32(pw)
    if pw.w8 is None:
        w8 = torch.empty((pad_n(pw.N), pw.Kp), dtype=torch.uint8, device=pw.codes.device)
        check(load().sqmp_pack_f8(_p(pw.codes), _p(pw.wscale), _dtype_code(pw.dtype), pw.N,
                                  pw.Kp, pw.ngw, _p(w8), _p(ws32), _stream(pw.codes)),
              "pack_f8")
        return _keep(pw, "w8", w8), ws32
    return pw.w8, ws32


def quant_act_f8(x2: torch.Tensor, pw: PackedWeight, act_quant: str, n_bits: int,
                 write_x: bool = False):
    """x [M, K] -> (e4m3 codes [M, Kp] in packed order, fp32 row scales [M], exact salient
    x [M, S_pad]) for gemm_f8 (per_token / per_tensor, n_bits <= 4)."""
    _require_gpu(x2, "quant_act")
    M, K = x2.shape
    Mp = _pad_rows(M)
    width = pw.Kp
    a8 = torch.empty((Mp, width), dtype=torch.uint8, device=x2.device)[:M]
    sa = torch.empty((M,), dtype=torch.float32, device=x2.device)
    xs = torch.empty((Mp, max(pw.S_pad, 8)), dtype=x2.dtype, device=x2.device)[:M]
    lib = load()
    nb = _ws_bytes(M, K, pw.Kp)
    stream = torch.cuda.current_stream(x2.device).cuda_stream
    e = _act_ws(x2.device, stream, K, pw.Kp, nb)
    if pw.posmap is None:
        pw.posmap = build_posmap(pw.perm, K)
    status = lib.sqmp_quant_act_v2(_p(x2), _dtype_code(x2.dtype), M, K, ACT_MODES[act_quant],
                                   n_bits, 0, _p(pw.amap), pw.Kp, _p(pw.nonsal), _p(pw.salient),
                                   pw.S, pw.S_pad, _p(pw.posmap),
                                   _lib.QA_CLEAN_WS | (_lib.QA_WRITE_X if write_x else 0), _lib.OUT_F8,
                                   _p(a8), _p(sa), _p(xs), _p(e["buf"]), e["buf"].numel(),
                                   ctypes.c_void_p(stream))
    if status != _lib.SQMP_OK:
        _discard_ws(e)
        check(status, "quant_act")
    if write_x:
        torch.autograd.graph.increment_version(x2)  # (x was rewritten through a raw pointer)
    return a8, sa, xs


def f8_write_x_ok(x2: torch.Tensor, pw: PackedWeight, act_quant: str, n_bits: int) -> bool:
    """Whether quant_act_f8(..., write_x=True) takes this call (SQMP_QA_WRITE_X): per_token
    4-bit codes, the identity packed order, 16-B aligned contiguous f16 / bf16 rows, K % 8 == 0."""
    return (act_quant == "per_token" and n_bits <= 4 and pw.K % 8 == 0 and not _LC_OFF
            and x2.dtype in (torch.float16, torch.bfloat16) and f8_input_ok(x2)
            and identity_layout(pw))


def f8_colmax_ok(pw: PackedWeight) -> bool:
    """Whether gemm_f8 can fuse the output-quant column statistics: the 16x16x128 kernel
    (Gw % 128 == 0) and not its SQMP_F8_V1=1 A/B variant (the 32x32x64 kernel has no fused
    statistics; read per call like the library does)."""
    return pw.Gw % 128 == 0 and os.environ.get("SQMP_F8_V1") != "1"


def gemm_f8(a8: torch.Tensor, sa: torch.Tensor, xs: torch.Tensor, pw: PackedWeight,
            bias: Optional[torch.Tensor], colmax: Optional[torch.Tensor] = None) -> torch.Tensor:
    """colmax (Gw % 128 == 0): as gemm_fq's fused output-quant statistics."""
    M = a8.shape[0]
    w8, ws32 = f8_operands(pw)
    y = torch.empty((M, pw.N), dtype=pw.dtype, device=a8.device)
    args = (_p(a8), _p(sa), _p(xs) if pw.S_pad else None, _p(w8), _p(ws32),
            _p(pw.wsal) if pw.S_pad else None, _p(bias), _p(y), _dtype_code(pw.dtype), M, pw.N,
            pw.Kp, pw.S_pad, pw.Gw, pw.ngw)
    if colmax is None:
        check(load().sqmp_gemm_f8(*args, _stream(a8)), "gemm_f8")
    else:
        check(load().sqmp_gemm_f8_colmax(*args, _p(colmax), _stream(a8)), "gemm_f8")
    return y


def f8_eligible(pw: PackedWeight, act_quant: str, act_bits: int) -> bool:
    """Whether the block-scaled FP8 MFMA path computes this layer: one act scale per row,
    4-bit codes on both sides (exact in e4m3), weight groups of whole 64-blocks, and the
    lane-contiguous quantizer's shape and LDS limits (K % 8 == 0, K <= 16384, lc_lds_ok;
    quant_lc_supported in sqmp_actquant_lc.hip).  The input pointer's 16-B alignment is
    checked per call (f8_input_ok)."""
    return (act_quant in ("per_token", "per_tensor") and pw.dtype != torch.float32
            and pw.n_bits == 4 and pw.dense is None and pw.Gw % 64 == 0 and act_bits <= 4
            and pw.K <= 16384 and pw.K % 8 == 0 and lc_lds_ok(pw.Kp, pw.S_pad))


def f8_input_ok(x2: torch.Tensor) -> bool:
    """The e4m3 quantizer reads x with 16-B loads: x must be contiguous and 16-B aligned."""
    return x2.is_contiguous() and x2.data_ptr() % 16 == 0


# Whether kernel="auto" takes the FP8 path for eligible layers (f8_eligible): on gfx950
# it is 1.4x the fq GEMM at config 2.
F8_AUTO = True


def f8_auto(pw: PackedWeight, act_quant: str, act_bits: int) -> bool:
    """Whether kernel="auto" runs this layer on the FP8 GEMM: fp16 layers only.  The FP8 path
    factors the scales out and so skips the D rounding of x_hat = D(code * s) and W_hat; in
    fp16 that is 2^-12 per product (y within 3e-3 of the reference).  In bf16 the rounding it
    skips is 2^-9 per product -- the size of bf16's own output rounding -- so y differs from
    the reference's bf16 F.linear in most low bits (2.4e-3 relative on the ppl_eval-flow
    Llama layer) and a 4-bit per-token model amplifies that into 50 % logit differences
    (tests/test_gpu_configs.py, llama7b_l_bf16_pplflow).  bf16 layers run the faithful fq
    GEMM on the bit-exact operands instead; kernel="f8" still forces the FP8 path."""
    return F8_AUTO and pw.dtype == torch.float16 and f8_eligible(pw, act_quant, act_bits)


# ----------------------------------------------------------------------------------------
# few rows: the decoding form of the faithful product
# ----------------------------------------------------------------------------------------
GEMV_MAX_ROWS = 64  # SQMP_GEMV_MAX_ROWS


def bpack_codes(codes: torch.Tensor) -> torch.Tensor:
    """int codes [R, Kp] in -8 .. 7 (Kp % 64 == 0) -> uint8 [R, Kp / 2] in the packed layout of
    include/sqmp_w4a4.h: dword (h * 4 + u) of a 64-position block holds positions
    16 u + 8 h + e, even e in the low half-word, odd e in the high one, nibble = code + 8."""
    R, Kp = codes.shape
    n = (codes.to(torch.int8) + 8).view(R, Kp // 64, 4, 2, 8)
    w = torch.zeros((R, Kp // 64, 2, 4), dtype=torch.int32, device=codes.device)
    for e in range(8):
        sh = (16 if e & 1 else 0) + 4 * (e >> 1)
        w |= (n[..., e].transpose(2, 3).to(torch.int32) & 15) << sh
    return w.view(R, Kp // 8).view(torch.uint8)


@on_tensor_device
def pack_codes(codes: torch.Tensor, scales: torch.Tensor, group_size: int) -> PackedWeight:
    """A PackedWeight from 4-bit codes that exist already (a checkpoint quantized elsewhere):
    codes int8 [N, K] in -8 .. 7, scales D [N, ceil(K / group_size)], W = D(code * scale) with
    the groups over consecutive columns; no salient columns, the columns' own order."""
    _require_gpu(codes, "pack_codes")
    if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.int8:
        raise ValueError("pack_codes: codes must be int8 [N, K], scales [N, groups]")
    N, K = codes.shape
    if N == 0 or K == 0 or group_size <= 0:
        raise ValueError(f"pack_codes: empty weight [{N}, {K}] or group size {group_size}")
    if scales.device != codes.device:
        raise RuntimeError(f"pack_codes: codes on {codes.device}, scales on {scales.device}")
    _dtype_code(scales.dtype)
    if scales.shape != (N, (K + group_size - 1) // group_size):
        raise ValueError(f"pack_codes: scales {tuple(scales.shape)} do not match codes "
                         f"{tuple(codes.shape)} in groups of {group_size}")
    dev, dt = codes.device, scales.dtype
    scales = scales.detach()  # (the weight is a constant)
    wmode = _lib.W_PER_CHANNEL if scales.shape[1] == 1 else _lib.W_PER_GROUP_UNSORTED
    Kp, Gw, ngw, S_pad = geometry(K, 0, wmode, group_size)
    Np = pad_n(N)
    full = torch.zeros((Np, Kp), dtype=torch.int8, device=dev)
    full[:N, :K] = codes
    wscale = torch.zeros((ngw, Np), dtype=dt, device=dev)
    wscale[:scales.shape[1], :N] = scales.t()
    perm, amap, amap_fq, nonsal = build_maps(K, None, dev, Kp)
    pw = PackedWeight(bpack_codes(full), wscale, torch.empty((N, 0), dtype=dt, device=dev), perm,
                      amap, amap_fq, nonsal, None, N, K, 0, S_pad, Kp, Gw, ngw, 4, wmode, dt)
    pw.posmap = torch.arange(K, dtype=torch.int32, device=dev)
    pw.sal_key = salient_key(K, None)
    pw.ident = Kp == K
    if Gw % (4 if dt == torch.float32 else 8):
        pw.dense = dequant_weight_packed(pw)
    return pw


@on_tensor_device
def tile_major(codes: torch.Tensor, wscale: torch.Tensor, wsal: torch.Tensor, N: int, Kp: int,
               S_pad: int, ngw: int, dtype: torch.dtype, out=None):
    """sqmp_pack_fq7 (J = 2) of a packed 4-bit weight: (codes_t, scale_t, sal_t), into `out`
    where given."""
    sizes = [ctypes.c_size_t() for _ in range(3)]
    check(load().sqmp_fq7_sizes(N, Kp, S_pad, ngw, 2, *[ctypes.byref(v) for v in sizes]),
          "fq7_sizes")
    if out is None:
        dev = codes.device
        out = (torch.empty(sizes[0].value, dtype=torch.uint8, device=dev),
               torch.empty(sizes[1].value, dtype=dtype, device=dev),
               torch.empty(sizes[2].value, dtype=dtype, device=dev))
    if tuple(t.numel() for t in out) != tuple(v.value for v in sizes):
        raise ValueError("tile_major: operands of another size")
    check(load().sqmp_pack_fq7(_p(codes), _p(wscale), _p(wsal) if S_pad else None,
                               _dtype_code(dtype), N, Kp, S_pad, ngw, 2, *[_p(t) for t in out],
                               _stream(codes)), "pack_fq7")
    for t in out:
        written(t)
    return out


_SPLIT_WS = {}
_lib.on_reload(_SPLIT_WS.clear)  # (the tile height is a knob)


def workspace_bytes(kind: str, *sizes: int) -> int:
    """sqmp_<kind>_workspace_bytes(*sizes), memoized (saves a ctypes call per product)."""
    n = _SPLIT_WS.get((kind, sizes))
    if n is None:
        n = _SPLIT_WS[(kind, sizes)] = getattr(load(), f"sqmp_{kind}_workspace_bytes")(*sizes)
        if len(_SPLIT_WS) > 65536:
            _SPLIT_WS.clear()
    return n


def gemv_eligible(pw: PackedWeight) -> bool:
    """Whether gemv computes this weight: 4-bit codes in groups of whole 8 positions."""
    return pw.n_bits == 4 and pw.dense is None and pw.Gw % 8 == 0


def gemv_operands(pw: PackedWeight):
    """(codes_t, scale_t, sal_t) of gemv: fq7_operands' copies where those are J = 2 (fp16 /
    bf16), else its own; built once per packed weight.  Inside a HIP-graph capture nothing is
    kept (the copy would be written at replay only): call gemv once before capturing."""
    if pw.gemv is not None:
        return pw.gemv
    adopt = pw.fq7 is not None and pw.fq7[3] == 2
    ops_t = pw.fq7[:3] if adopt else tile_major(pw.codes, pw.wscale, pw.wsal, pw.N, pw.Kp, pw.S_pad,
                                                pw.ngw, pw.dtype)
    if torch.cuda.is_current_stream_capturing():
        return ops_t
    torch.cuda.synchronize(pw.codes.device)  # (built on one stream, read later from any)
    pw.gemv = ops_t
    if pw.fq7 is None and FQ7_J == 2 and pw.dtype != torch.float32:
        pw.fq7 = ops_t + (2,)
    return ops_t


def _operand_rows(x2: torch.Tensor, width: int):
    """Whether the kernels read x2's rows in place: unit column stride, 16-B aligned rows."""
    per = 16 // x2.element_size()
    return (x2.stride(1) == 1 and x2.data_ptr() % 16 == 0
            and (x2.shape[0] == 1 or (x2.stride(0) >= width and x2.stride(0) % per == 0)))


@on_tensor_device
def pack_rows(x2: torch.Tensor, amap: torch.Tensor, Kp: int, salient: Optional[torch.Tensor],
              S: int, S_pad: int) -> torch.Tensor:
    """x [M, K] -> [M, Kp + S_pad]: the unquantized activation operand (columns gathered by amap,
    then the salient columns).  amap int32 [Kp] and salient int32 [S] name columns of x (amap < 0: a
    zero); they are not looked at here."""
    if not x2.is_cuda:
        _require_gpu(x2, "pack_rows")
    if x2.dim() != 2 or Kp <= 0 or not 0 <= S <= S_pad:
        raise ValueError(f"pack_rows: x {tuple(x2.shape)}, Kp {Kp}, {S} of {S_pad} salient columns")
    for name, t, n in (("amap", amap, Kp), ("salient", salient, S)):
        if n and (t is None or t.dtype != torch.int32 or t.numel() < n or not t.is_contiguous()
                  or t.device != x2.device):
            raise ValueError(f"pack_rows: {name} must be {n} contiguous int32 on {x2.device}")
    return _pack_rows(x2, amap, Kp, salient, S, S_pad)


def _pack_rows(x2, amap, Kp, salient, S, S_pad) -> torch.Tensor:
    """pack_rows with the maps of a packed weight."""
    if x2.stride(1) != 1 or x2.stride(0) == 0:  # (0: rows of an expanded tensor)
        x2 = x2.contiguous()
    M = x2.shape[0]
    out = x2.new_empty((M, Kp + S_pad))
    status = load().sqmp_pack_rows(x2.data_ptr(), max(x2.stride(0), 1), _dtype_code(x2.dtype), M,
                                   amap.data_ptr(), Kp,
                                   None if salient is None else salient.data_ptr(), S, S_pad, None,
                                   1, None, 0, 0, out.data_ptr(), _raw_stream(x2.device.index))
    if status:
        check(status, "pack_rows")
    return out


@on_tensor_device
def gemv(x: torch.Tensor, pw: PackedWeight, bias: Optional[torch.Tensor] = None,
         packed: bool = False) -> torch.Tensor:
    """y [M, N] = D(x . W_hat^T + bias) for M <= GEMV_MAX_ROWS rows (the decoding form of
    gemm_fq: the same operands, fp32 sums in another fixed order).

    x: [M, K] in the columns' order -- a 4-bit weight with D activations -- or, with `packed`,
    the [M, Kp + S_pad] operand of quant_act_fp.  Any strides; rows that are not 16-B aligned,
    and those of weights packed in an order of their own, are gathered by the kernel where they
    are few, else copied first (sqmp_pack_rows)."""
    if not x.is_cuda:
        _require_gpu(x, "gemv")
    dtype, device, code, L, K, per, ident, (codes_t, scale_t, sal_t), N, tail = (
        pw.gemv_args or _gemv_args(pw))
    if x.dim() != 2 or x.dtype is not dtype or x.device != device:
        _gemv_refuse(x, dtype, device)
    M, C = x.shape
    if C != (L if packed else K):
        raise ValueError(f"gemv: x has {C} columns, the weight {L if packed else K}")
    if M > GEMV_MAX_ROWS:
        raise ValueError(f"gemv: {M} rows, at most {GEMV_MAX_ROWS}")
    bp = None
    if bias is not None:
        if bias.dtype is not dtype or bias.device != device or bias.numel() != N:
            raise RuntimeError(f"gemv: bias {bias.dtype} [{bias.numel()}] on {bias.device} does "
                               f"not match {dtype} [{N}] on {device}")
        if bias.dim() != 1 or not bias.is_contiguous():
            bias = bias.reshape(-1).contiguous()
        bp = bias.data_ptr()
    y = x.new_empty((M, N))
    if M == 0:
        return y
    lib = load()
    ld, s1 = x.stride()
    xp = x.data_ptr()
    amap = sal = None
    cols = pw.Kp if packed else ident or pw.Kp
    if (packed or ident) and s1 == 1 and xp % 16 == 0 and (M == 1 or (ld >= C and ld % per == 0)):
        if M == 1:
            ld = L
    elif packed:
        x = x.clone(memory_format=torch.contiguous_format)
        xp, ld = x.data_ptr(), L
    elif s1 == 1 and ld > 0 and lib.sqmp_gemv_gathers(code, M, pw.Kp, pw.S_pad):
        cols = pw.Kp
        amap, sal = pw.amap.data_ptr(), None if pw.salient is None else pw.salient.data_ptr()
    else:
        x = _pack_rows(x, pw.amap, pw.Kp, pw.salient, pw.S, pw.S_pad)
        xp, ld, cols = x.data_ptr(), L, pw.Kp
    wp, wn = None, 0
    if M > 32:
        wn = workspace_bytes("gemv", code, M, N, pw.Kp)
        if wn:
            ws = torch.empty(wn, dtype=torch.uint8, device=device)
            wp = ws.data_ptr()
    status = lib.sqmp_gemv_w4(xp, ld, cols, amap, sal, pw.S, codes_t.data_ptr(), scale_t.data_ptr(),
                              sal_t.data_ptr() if pw.S_pad else None, bp, y.data_ptr(), code, M, N,
                              *tail, wp, wn, _raw_stream(device.index))
    if status:
        check(status, "gemv")
    return y


def _gemv_refuse(x: torch.Tensor, dtype: torch.dtype, device: torch.device):
    if x.dim() != 2:
        raise ValueError(f"gemv: x must have 2 dimensions, got {tuple(x.shape)}")
    if x.dtype is not dtype:
        raise RuntimeError(f"expected input dtype {dtype}, got {x.dtype}")
    raise RuntimeError(f"gemv: x on {x.device}, the weight on {device}")


def own_columns(pw: PackedWeight):
    """K where x's rows are the operand as they are -- the identity order, no salient columns, whole
    64-position stages --, 0 where not, None where a capture forbids to look."""
    if pw.S or pw.S_pad or pw.K % 64:
        return 0
    if pw.ident:
        return pw.K
    if torch.cuda.is_current_stream_capturing():
        return None
    arange = torch.arange(pw.K, dtype=torch.int32, device=pw.amap.device)
    return pw.K if torch.equal(pw.amap[:pw.K], arange) else 0


def _gemv_args(pw: PackedWeight):
    """gemv's arguments that depend on the weight alone (its operands as tensors: a call takes their
    addresses); kept on it once its operands and order are known for good (not inside a capture)."""
    if not gemv_eligible(pw):
        raise ValueError(f"gemv: needs 4-bit codes in groups of a multiple of 8 columns (n_bits "
                         f"{pw.n_bits}, group {pw.Gw})")
    t = gemv_operands(pw)
    ident = own_columns(pw)
    dev = pw.codes.device
    a = (pw.dtype, dev, _dtype_code(pw.dtype), pw.Kp + pw.S_pad, pw.K,
         4 if pw.dtype == torch.float32 else 8, ident, t, pw.N, (pw.Kp, pw.S_pad, pw.Gw, pw.ngw))
    if pw.gemv is t and ident is not None:
        pw.gemv_args = a
    return a
