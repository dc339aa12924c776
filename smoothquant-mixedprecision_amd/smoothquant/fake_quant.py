"""Drop-in `smoothquant.fake_quant` for MI355X: W4A4Linear + the model-surgery entry points.

Same import path, names, constructor/forward signatures, attributes and error types as
/root/reference/smoothquant/fake_quant.py, but the operator is real: weights are packed
once to int4 (or int8) codes + per-group scales + an exact salient slice, and forward
runs the HIP kernels of libsqmp_w4a4 (activation quantization + MFMA GEMM with the
salient FP side-GEMM in the same workgroup).  There is no CPU path: a W4A4Linear whose
tensors are not on a ROCm device raises.

Reference map (file:line in fake_quant.py):
  quantizer primitives       9-207   -> quantize_* below (GPU, same in-place semantics)
  W4A4Linear.__init__      210-270   -> W4A4Linear.__init__
  W4A4Linear.forward       279-322   -> W4A4Linear.forward
  W4A4Linear.from_float    324-371   -> W4A4Linear.from_float
  quantize_opt/llama_like/mixtral/falcon/model  377-799 -> same names
"""
from __future__ import annotations

import inspect
import weakref
from functools import partial
from typing import Optional

import torch
from torch import nn

from . import ops
from .ops import PackedWeight

_ACT = ("per_token", "per_tensor", "per_group")
_WEIGHT = ("per_channel", "per_tensor", "per_group")
# Sort-strategy extensions (not accepted by the reference, which only
# wires max-sorted groups): "_unsorted" = the reference's unwired unsorted quantizers
# (fake_quant.py:29-53, :77-101); "_mean3std" = columns sorted by mean|x| + 3 std|x| (the
# README.md:36 "statistical sorting", absent from the reference's code; parity unpinned).
_ACT_EXT = _ACT + ("per_group_unsorted", "per_group_mean3std")
_WEIGHT_EXT = _WEIGHT + ("per_group_unsorted", "per_group_mean3std")


# ----------------------------------------------------------------------------------------
# quantizer primitives (fake_quant.py:9-207) -- GPU implementations, reference semantics
# ----------------------------------------------------------------------------------------
def _fq_act(t: torch.Tensor, mode: str, n_bits: int, group_size: int = 128) -> torch.Tensor:
    t2 = t.view(-1, t.shape[-1])
    C = t2.shape[1]
    _, _, amap_fq, nonsal = ops.build_maps(C, None, t2.device)
    return ops.fake_quant_inplace(t2, mode, n_bits, group_size, amap_fq, nonsal, 0)


@torch.no_grad()
def quantize_activation_per_token_absmax(t, n_bits):
    """fake_quant.py:56-64: in place on `t`, returns the 2-D view."""
    return _fq_act(t, "per_token", n_bits)


@torch.no_grad()
def quantize_activation_per_tensor_absmax(t, n_bits):
    """fake_quant.py:67-75: in place on `t`, returns the 2-D view."""
    return _fq_act(t, "per_tensor", n_bits)


@torch.no_grad()
def quantize_activation_per_group_absmax(t, n_bits, group_size=128):
    """fake_quant.py:77-101 (unsorted groups): returns a new tensor of t's shape."""
    out = t.contiguous().clone()
    _fq_act(out, "per_group_unsorted", n_bits, group_size)
    return out.view(t.shape)


@torch.no_grad()
def quantize_activation_per_group_absmax_sort(t, n_bits, group_size=128):
    """fake_quant.py:104-154 (sorted groups): returns a new tensor of t's shape."""
    out = t.contiguous().clone()
    _fq_act(out, "per_group", n_bits, group_size)
    return out.view(t.shape)


@torch.no_grad()
def quantize_activation_per_group_mean3std_sort(t, n_bits, group_size=128):
    """As :104-154 with the columns sorted by mean|x| + 3 std|x| over the batch instead of
    the column absmax (README.md:36; not in the reference's code -- parity unpinned)."""
    out = t.contiguous().clone()
    _fq_act(out, "per_group_mean3std", n_bits, group_size)
    return out.view(t.shape)


def _fq_weight(w: torch.Tensor, mode: str, n_bits: int, group_size: int) -> torch.Tensor:
    return ops.dequant_weight(ops.pack_weight(w, mode, n_bits, group_size, None))


@torch.no_grad()
def quantize_weight_per_channel_absmax(w, n_bits):
    """fake_quant.py:9-16: in place on `w`, returns `w`."""
    w.copy_(_fq_weight(w, "per_channel", n_bits, 128))
    return w


@torch.no_grad()
def quantize_weight_per_tensor_absmax(w, n_bits):
    """fake_quant.py:19-26: in place on `w`, returns `w`."""
    w.copy_(_fq_weight(w, "per_tensor", n_bits, 128))
    return w


@torch.no_grad()
def quantize_weight_per_group_absmax(w, n_bits, group_size=128):
    """fake_quant.py:29-53 (unsorted groups): returns a new tensor."""
    return _fq_weight(w, "per_group_unsorted", n_bits, group_size)


@torch.no_grad()
def quantize_weight_per_group_absmax_sort(w, n_bits, group_size=128):
    """fake_quant.py:156-207 (sorted groups): returns a new tensor."""
    return _fq_weight(w, "per_group", n_bits, group_size)


@torch.no_grad()
def quantize_weight_per_group_mean3std_sort(w, n_bits, group_size=128):
    """As :156-207 with the columns sorted by mean|W| + 3 std|W| (parity unpinned)."""
    return _fq_weight(w, "per_group_mean3std", n_bits, group_size)


_ACT_FNS = {"per_token": quantize_activation_per_token_absmax,
            "per_tensor": quantize_activation_per_tensor_absmax,
            "per_group": quantize_activation_per_group_absmax_sort,
            "per_group_unsorted": quantize_activation_per_group_absmax,
            "per_group_mean3std": quantize_activation_per_group_mean3std_sort}
_FN_MODE = {fn: mode for mode, fn in _ACT_FNS.items()}
_GROUPED = ("per_group", "per_group_unsorted", "per_group_mean3std")


def _bind_act(mode: str, n_bits: int, group_size: int):
    """The act_quant partial of fake_quant.py:246-256 for `mode`."""
    kw = {"group_size": group_size} if mode in _GROUPED else {}
    return partial(_ACT_FNS[mode], n_bits=n_bits, **kw)


_RQ_MEMO = {}


def resolve_quantizer(fn):
    """Memoized _resolve_quantizer (the signature binding costs ~10 us per call; a partial's
    func / args / keywords are read-only, so the result is fixed per callable object)."""
    e = _RQ_MEMO.get(id(fn))
    if e is not None and e[0] is fn:
        return e[1]
    r = _resolve_quantizer(fn)
    if len(_RQ_MEMO) > 8192:
        _RQ_MEMO.clear()
    _RQ_MEMO[id(fn)] = (fn, r)
    return r


def _resolve_quantizer(fn):
    """(mode, n_bits, group_size) of an act/output quantizer callable, or None for the
    identity.  Accepts what the reference binds (fake_quant.py:246-263) and what its users
    rebind (e.g. W4A8: ``q.act_quant = partial(quantize_activation_per_group_absmax_sort,
    n_bits=8, group_size=G)``): a functools.partial over one of this module's activation
    quantizers.  Any other callable raises -- the HIP operator cannot run arbitrary Python
    quantizers, and silently ignoring one would change the numerics."""
    if fn is None or getattr(fn, "_sqmp_identity", False):
        return None
    base, args, kw = fn, (), {}
    if isinstance(fn, partial):
        base, args, kw = fn.func, fn.args, dict(fn.keywords or {})
    mode = _FN_MODE.get(base)
    if mode is None:
        raise NotImplementedError(
            f"W4A4Linear: unsupported quantizer callable {fn!r}; bind one of "
            f"{sorted(f.__name__ for f in _FN_MODE)} with functools.partial")
    bound = inspect.signature(base).bind_partial(None, *args, **kw)
    bound.apply_defaults()
    n_bits = bound.arguments.get("n_bits")
    if n_bits is None:
        raise TypeError(f"{base.__name__}: missing n_bits")
    return mode, int(n_bits), int(bound.arguments.get("group_size", 128))


def _identity(x):
    return x


def _spec_list(spec):
    return None if spec is None else [spec[0], int(spec[1]), int(spec[2])]


_identity._sqmp_identity = True
# output-quant statistics fused into the GEMM epilogue (SQMP_OQ_FUSE=0: separate
# statistics pass; A/B timing only -- the numerics are identical)
_OQ_FUSE = __import__("os").environ.get("SQMP_OQ_FUSE", "1") != "0"

_PACKED_BUFFERS = ("w_codes", "w_scale", "w_salient", "w_perm", "w_amap", "w_amap_fq",
                   "w_nonsal", "salient_i32", "w_dense", "out_amap_fq", "out_nonsal")
# buffers a PackedWeight holds (W4A4Linear.packed's reuse check)
_PW_KEY = ("w_codes", "w_scale", "w_salient", "w_perm", "w_amap", "w_amap_fq", "w_nonsal",
           "salient_i32", "w_dense", "w_posmap")


# ----------------------------------------------------------------------------------------
# W4A4Linear (fake_quant.py:209-374)
# ----------------------------------------------------------------------------------------
# the forward kernels a module's `kernel` attribute selects (W4A4Linear docstring)
KERNELS = ("auto", "fq", "f8", "fqt", "gemv")


class W4A4Linear(nn.Module):
    """Mixed-precision W4A4 linear: salient input channels in D, the rest int4/int8.

    Forward kernels (chosen per layer, see `kernel`; "auto" = "f8" where ops.f8_auto (fp16),
    "fqt" for large sorted per_group batches, else "fq"):
      "f8"  per_token / per_tensor 4-bit activations: e4m3 act codes x e4m3 weight codes on
            the block-scaled FP8 MFMA (exact integer block sums), per-group fp32 folds.
      "fq"  every act mode: dequantized activations x in-kernel-decoded weights on the D
            MFMA (bit-exact operands; the reference's numerics up to accumulation order).
      "fqt" per_group activations (auto from ops.FQT_MIN_ROWS rows, ops.fqt_eligible): "fq"
            in ACTIVATION order -- 4-bit act codes decoded in the GEMM, the weight W_hat
            permuted per forward, no salient zero positions in the K loop; the same
            operands bit for bit, so "fq"'s numerics.
      "gemv" decoding: up to ops.GEMV_MAX_ROWS rows on the few-row kernel ("fq"'s operands, fp32
            sums in another order), more rows and the weights it does not take as "auto"
            (use_gemv switches a model's layers).
    """

    def __init__(self, in_features, out_features, bias=True, act_quant="per_token",
                 quantize_output=False, importance=None, salient_prop=0, quant_bits=4,
                 group_size=128):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.group_size = group_size
        self.quant_bits = quant_bits
        if act_quant not in _ACT_EXT:
            raise ValueError(f"Invalid act_quant: {act_quant}")     # fake_quant.py:256
        self.act_quant_name = act_quant
        self.act_quant = _bind_act(act_quant, quant_bits, group_size)
        if quantize_output:
            self.output_quant_name = self.act_quant_name
            self.output_quant = self.act_quant
        else:
            self.output_quant_name = "None"
            self.output_quant = _identity
        self.salient_indices = None
        if importance is not None and salient_prop > 0:             # :265-270
            sorted_idx = torch.argsort(importance, descending=True, stable=True)
            num_salient = max(1, int(salient_prop * len(sorted_idx)))
            self.salient_indices = sorted_idx[:num_salient]
        self.weight_quant_name = "None"
        self.kernel = "auto"
        self._meta = None
        for name in _PACKED_BUFFERS:
            self.register_buffer(name, None)
        # column -> packed position (inverse of w_perm), derived: not part of checkpoints
        self.register_buffer("w_posmap", None, persistent=False)
        self._sal_key = None
        if bias:
            self.register_buffer("bias", torch.zeros((1, out_features), dtype=torch.float16))
        else:
            self.register_buffer("bias", None)
        # The reference starts from an unquantized random fp16 weight (:227-235); a directly
        # constructed module draws it on the GPU and packs it as a dense operand on first use.
        self._random_init = True

    # ------------------------------------------------------------------ packing
    def _install(self, pw: PackedWeight, weight_quant: str):
        self.w_codes = pw.codes
        self.w_scale = pw.wscale
        self.w_salient = pw.wsal
        self.w_perm = pw.perm
        self.w_amap = pw.amap
        self.w_amap_fq = pw.amap_fq
        self.w_nonsal = pw.nonsal
        self.salient_i32 = pw.salient
        self.w_dense = pw.dense
        self.w_posmap = pw.posmap
        self._sal_key = pw.sal_key
        self._meta = dict(N=pw.N, K=pw.K, S=pw.S, S_pad=pw.S_pad, Kp=pw.Kp, Gw=pw.Gw,
                          ngw=pw.ngw, n_bits=pw.n_bits, wmode=pw.wmode, dtype=pw.dtype)
        self.weight_quant_name = weight_quant
        self._random_init = False
        if self.output_quant_name != "None" and self.salient_indices is None:
            _, _, self.out_amap_fq, self.out_nonsal = ops.build_maps(pw.N, None, pw.codes.device)

    def _pack_from(self, w: torch.Tensor, weight_quant: str, want_w_hat: bool = False):
        """Pack w on the GPU (a CPU-resident w is packed on cuda and the module moved back
        to w's device).  want_w_hat: also return W_hat (the reference's dequantized weight)
        on w's device, computed on the GPU before any move back."""
        dev = w.device
        wg = w.detach()
        if dev.type != "cuda":
            if not torch.cuda.is_available():
                raise RuntimeError("W4A4Linear packing needs a ROCm GPU (no CPU implementation)")
            wg = wg.to("cuda")
        sal = self.salient_indices
        pw = ops.pack_weight(wg, weight_quant if weight_quant in _WEIGHT_EXT else "none",
                             self.quant_bits, self.group_size, sal)
        self._install(pw, weight_quant)
        w_hat = ops.dequant_weight(pw).to(dev) if want_w_hat else None
        if dev.type != "cuda":
            self.to(dev)
        return w_hat

    def packed(self) -> PackedWeight:
        # One PackedWeight per buffer set: reused while every buffer is the same object and
        # the codes / scales were not written in place (their derived f8 operands, built
        # once per PackedWeight, stay valid) -- a forward then costs no host rebuild.
        # (dict lookups, not Module.__getattr__: this runs once per forward)
        d, b = self.__dict__, self._buffers
        c = d.get("_pw_cache")
        if (c is not None and c[3] is d.get("_meta") and c[4] is d.get("_sal_key")
                and c[2] == (b["w_codes"]._version, b["w_scale"]._version)
                and all(b[n] is t for n, t in zip(_PW_KEY, c[0]))):
            return c[1]
        if self._meta is None:
            if not self._random_init:
                raise RuntimeError("W4A4Linear has no packed weight")
            if not torch.cuda.is_available():
                raise RuntimeError("W4A4Linear needs a ROCm GPU (no CPU implementation)")
            w = torch.randn(self.out_features, self.in_features, dtype=torch.float16,
                            device="cuda")
            self._pack_from(w, "None")
        m = self._meta
        if self.w_posmap is None or self.w_posmap.device != self.w_perm.device:
            self.w_posmap = ops.build_posmap(self.w_perm, m["K"])  # e.g. after a checkpoint load
        if self._sal_key is None:
            self._sal_key = ops.salient_key(m["K"], self.salient_i32)
        pw = PackedWeight(self.w_codes, self.w_scale, self.w_salient, self.w_perm, self.w_amap,
                          self.w_amap_fq, self.w_nonsal, self.salient_i32, m["N"], m["K"],
                          m["S"], m["S_pad"], m["Kp"], m["Gw"], m["ngw"], m["n_bits"],
                          m["wmode"], m["dtype"], self.w_dense, self.w_posmap, self._sal_key)
        b = self._buffers
        self.__dict__["_pw_cache"] = (tuple(b[n] for n in _PW_KEY), pw,
                                      (b["w_codes"]._version, b["w_scale"]._version),
                                      m, self._sal_key)
        return pw

    # ------------------------------------------------------------------ persistence
    # Packed format (the reference persists only the dequantized weight
    # and drops salient_indices).  state_dict() holds the packed buffers (w_codes, w_scale,
    # w_salient, maps) plus `_extra_state`: plain ints / strings / an int64 tensor, so a
    # checkpoint loads with torch.load(weights_only=True) and needs no recalibration.
    EXTRA_FORMAT = "sqmp-w4a4-packed/1"

    def get_extra_state(self):
        m = self._meta
        return {
            "format": self.EXTRA_FORMAT,
            "in_features": self.in_features, "out_features": self.out_features,
            "quant_bits": self.quant_bits, "group_size": self.group_size,
            "act_quant": self.act_quant_name, "output_quant": self.output_quant_name,
            # the bound quantizers themselves (they may have been rebound, e.g. W4A8)
            "act_spec": _spec_list(resolve_quantizer(self.act_quant)),
            "output_spec": _spec_list(resolve_quantizer(self.output_quant)),
            "weight_quant": self.weight_quant_name, "kernel": self.kernel,
            "salient_indices": (None if self.salient_indices is None
                                else self.salient_indices.detach().to("cpu", torch.int64)),
            "meta": None if m is None else {k: (str(v).replace("torch.", "") if k == "dtype" else int(v))
                                            for k, v in m.items()},
        }

    def set_extra_state(self, state):
        if not isinstance(state, dict) or state.get("format") != self.EXTRA_FORMAT:
            raise RuntimeError(f"W4A4Linear: unsupported extra state {type(state)}")
        if (state["in_features"], state["out_features"]) != (self.in_features, self.out_features):
            raise RuntimeError("W4A4Linear: checkpoint shape does not match the module")
        self.quant_bits = state["quant_bits"]
        self.group_size = state["group_size"]
        act = state["act_quant"]
        self.act_quant_name = act
        spec = state.get("act_spec")
        self.act_quant = (_bind_act(spec[0], spec[1], spec[2]) if spec
                          else _bind_act(act, self.quant_bits, self.group_size))
        if state["output_quant"] != "None":
            ospec = state.get("output_spec")
            self.output_quant_name = state["output_quant"]
            self.output_quant = (_bind_act(ospec[0], ospec[1], ospec[2]) if ospec
                                 else self.act_quant)
        else:
            self.output_quant_name, self.output_quant = "None", _identity
        self.weight_quant_name = state["weight_quant"]
        self.kernel = state.get("kernel", "auto")
        sal = state["salient_indices"]
        self.salient_indices = None if sal is None else sal.clone()
        self.w_posmap, self._sal_key = None, None  # re-derived from the loaded buffers
        meta = state["meta"]
        if meta is not None:
            meta = dict(meta)
            meta["dtype"] = getattr(torch, meta["dtype"])
            self._meta = meta
            self._random_init = False

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys,
                              unexpected_keys, error_msgs):
        sd = state_dict
        if prefix + "_extra_state" in sd:
            # size the packed buffers (None in a fresh module) from the checkpoint; the
            # default loader below then copies every key, strictly
            for name in _PACKED_BUFFERS:
                t = sd.get(prefix + name)
                setattr(self, name, None if t is None else torch.empty_like(t))
            t = sd.get(prefix + "bias")
            if t is not None and self.bias is not None:
                # the bias lives with the packed buffers (the checkpoint's device), never
                # on the fresh module's construction device: the GEMM reads it by pointer
                if isinstance(self.bias, nn.Parameter):
                    # from_float aliased the source Linear's bias Parameter (:369-370):
                    # give the module its own, shaped like the checkpoint's
                    self.bias = nn.Parameter(torch.empty_like(t), requires_grad=False)
                elif (self.bias.shape != t.shape or self.bias.dtype != t.dtype
                      or self.bias.device != t.device):
                    self.bias = torch.empty_like(t)
        elif prefix + "weight" in sd:
            # a reference checkpoint (dequantized `weight` buffer): stored as given
            self.weight = sd[prefix + "weight"]
            sd = {k: v for k, v in sd.items() if k != prefix + "weight"}
        super()._load_from_state_dict(sd, prefix, local_metadata, strict, missing_keys,
                                      unexpected_keys, error_msgs)

    # the reference's `weight` buffer (dequantized W_hat, fake_quant.py:357-365)
    @property
    def weight(self) -> torch.Tensor:
        return ops.dequant_weight(self.packed())

    @weight.setter
    def weight(self, value: torch.Tensor):
        # assigning a weight (reference: `new_module.weight = ...`) stores it unquantized,
        # exactly what the reference's F.linear would then consume
        self._pack_from(value.data if isinstance(value, nn.Parameter) else value, "None")

    def __setattr__(self, name, value):
        if name == "weight":
            object.__setattr__(self, name, value)
            return
        super().__setattr__(name, value)

    def _apply(self, fn, recurse=True):
        # A dtype cast (model.half(), .float(), .to(torch.bfloat16)) turns the reference's
        # dequantized W_hat buffer into cast(W_hat) (fake_quant.py:272-277 / nn.Module).
        # The packed form is kept only when the check in _apply_cast passes, i.e.
        # cast(W_hat) == D'(code * cast(s)) for every weight (D(code*s) may round, so even an
        # up-cast is not guaranteed): the codes stay, the scales and the salient slice are
        # cast.  Otherwise the layer keeps the reference's values as a dense operand and
        # says so (a dense GEMM moves 4x the weight bytes).  The check dequantizes once per
        # dtype cast, not per forward.
        if self._meta is not None and self.w_scale is not None:
            old = self._meta["dtype"]
            probe = fn(torch.empty(0, dtype=old, device=self.w_scale.device))
            if probe.dtype != old:
                return self._apply_cast(fn, recurse, probe.dtype)
        return super()._apply(fn, recurse)

    def _apply_cast(self, fn, recurse, new_dtype):
        w_new = fn(self.weight)
        pw = self.packed()
        keep_packed = pw.n_bits == 0
        if not keep_packed:
            cand = ops.PackedWeight(pw.codes, fn(pw.wscale), fn(pw.wsal), pw.perm, pw.amap,
                                    pw.amap_fq, pw.nonsal, pw.salient, pw.N, pw.K, pw.S,
                                    pw.S_pad, pw.Kp, pw.Gw, pw.ngw, pw.n_bits, pw.wmode,
                                    new_dtype)
            keep_packed = bool(torch.equal(ops.dequant_weight(cand), w_new.to(pw.codes.device)))
        if keep_packed:
            out = super()._apply(fn, recurse)
            self._meta = dict(self._meta, dtype=new_dtype)
            self.__dict__.pop("_pw_cache", None)
            return out
        import warnings
        warnings.warn(
            f"W4A4Linear({self.in_features}, {self.out_features}): casting {pw.dtype} -> "
            f"{new_dtype} changes the dequantized weight values (cast(code*s) != code*cast(s)); "
            "the layer keeps the reference's cast(W_hat) as a DENSE operand -- quantize the "
            "model in the target dtype to keep the int4 packing", RuntimeWarning, stacklevel=3)
        out = super()._apply(fn, recurse)
        name = self.weight_quant_name
        self._pack_from(w_new, "None")
        self.weight_quant_name = name
        return out

    def to(self, *args, **kwargs):
        super().to(*args, **kwargs)
        return self

    # ------------------------------------------------------------------ forward
    def _kernel_for(self, rows: int, pw: PackedWeight) -> str:
        """The kernel of a batch: "gemv" is "auto" where the few-row product does not take it."""
        if self.kernel == "gemv" and not (rows <= ops.GEMV_MAX_ROWS and ops.gemv_eligible(pw)):
            return "auto"
        return self.kernel

    @torch.no_grad()
    def forward(self, x):
        if self.kernel not in KERNELS:
            raise ValueError(f"kernel must be one of {KERNELS}, got {self.kernel!r}")
        if x.is_cuda and x.device.index != ops._current_device():
            with torch.cuda.device(x.device):
                return self.forward(x)
        x_shape = x.shape
        if len(x_shape) == 3:
            x2 = x.reshape(-1, x_shape[-1])
        elif len(x_shape) == 2:
            x2 = x
        else:
            raise ValueError(f"Unsupported input shape: {x_shape}")          # :287
        if x.device.type != "cuda":
            raise RuntimeError("W4A4Linear.forward runs on a ROCm GPU only (HIP kernels); "
                               f"got a tensor on {x.device}")
        if x2.shape[0] == 0:
            # an empty batch: nothing to quantize or multiply (the kernels take no 0-row
            # operands: a 0-element tensor has no device pointer)
            pw = self.packed()
            if x2.dtype != pw.dtype:
                raise RuntimeError(f"expected input dtype {pw.dtype}, got {x2.dtype}")
            return x.new_empty(tuple(x_shape[:-1]) + (self.out_features,))
        grp = self.__dict__.get("_sqmp_group")
        if grp is not None:
            y = grp.forward(self, x, x2)
            if y is not None:
                return y
        pw = self.packed()
        if x2.dtype != pw.dtype:
            raise RuntimeError(f"expected input dtype {pw.dtype}, got {x2.dtype}")
        # the bound quantizers (fake_quant.py:246-263), honouring a rebinding such as W4A8
        amode, bits, ag = resolve_quantizer(self.act_quant)
        ospec = resolve_quantizer(self.output_quant)
        # per_token / per_tensor quantize the caller's activation in place when no channel
        # is salient (:304 -> :56-75); the grouped quantizers return new tensors
        mutate_input = (self.salient_indices is None and amode in ("per_token", "per_tensor")
                        and x2.data_ptr() == x.data_ptr() and x2.is_contiguous())
        xc = x2.contiguous()
        bias = None if self.bias is None else self.bias.reshape(-1)
        if bias is not None and bias.dtype != pw.dtype:
            raise RuntimeError(f"bias dtype {bias.dtype} does not match {pw.dtype}")
        if bias is not None and bias.device != x.device:
            raise RuntimeError(f"bias on {bias.device}, input on {x.device}: move the module "
                               "to the input's device")
        kernel = self._kernel_for(x2.shape[0], pw)
        use_gemv = kernel == "gemv"
        if use_gemv:
            kernel = "fq"  # (the operand)
        use_f8 = kernel == "f8" or (
            kernel == "auto" and ops.f8_auto(pw, amode, bits) and ops.f8_input_ok(xc))
        use_fqt = (not use_f8 and kernel in ("auto", "fqt")
                   and ops.fqt_eligible(pw, amode, bits, ag, x2.shape[0], force=kernel == "fqt")
                   and ops.f8_input_ok(xc))
        # fp32 layers: the quantizer writes sqmp_gemm_h2d's two f16 planes itself
        use_h2 = (not use_f8 and not use_fqt and kernel == "auto"
                  and ops.h2_planes_ok(pw, amode, x2.shape[0], ag))
        # the in-place quantization of the caller's x is the GEMM operand itself when the
        # packed order is the column order (ops.identity_layout): one quantizer pass, not two
        # (the operand rows the GEMM over-reads up to its 256-row tiles exist only when M is a
        # multiple of 256; else the quantized rows are copied into a padded operand)
        inplace_op = (mutate_input and not (use_f8 or use_fqt or use_h2)
                      and ops.identity_layout(pw) and ops.f8_input_ok(xc))
        # on the FP8 path the same pass writes the codes and x_hat over x (SQMP_QA_WRITE_X)
        f8_write_x = use_f8 and mutate_input and ops.f8_write_x_ok(xc, pw, amode, bits)
        if use_f8:
            a8, sa, xs = ops.quant_act_f8(xc, pw, amode, bits, write_x=f8_write_x)
        elif use_fqt:
            c4 = ops.quant_act_c4(xc, pw, amode, bits, ag, stats_of=x)
        elif use_h2:
            a2 = ops.quant_act_fp(xc, pw, amode, bits, ag, stats_of=x, h2=True)
        elif not inplace_op:
            a = ops.quant_act_fp(xc, pw, amode, bits, ag, stats_of=x)
        if mutate_input and not f8_write_x:
            ops.fake_quant_inplace(xc, amode, bits, ag, pw.amap_fq, pw.nonsal, 0)
        if inplace_op:
            a = xc if use_gemv or xc.shape[0] % 256 == 0 else ops.padded_operand(xc)
        if ospec is not None and self.salient_indices is not None and pw.N != pw.K:
            raise IndexError(                                                # :311-314
                f"The shape of the mask [{pw.K}] at index 0 does not match the shape "
                f"of the indexed tensor [{x2.shape[0]}, {pw.N}] at index 1")
        # output quantization fused into the GEMM epilogue (fake_quant.py:308-316): for
        # per_group (sorted) / per_tensor the faithful GEMM also writes the column maxima of
        # y into the output quantizer's workspace, which then skips its statistics pass
        fuse = (ospec is not None and ospec[0] in ("per_group", "per_tensor") and _OQ_FUSE
                and (not use_f8 or ops.f8_colmax_ok(pw))       # the 16x16x128 FP8 kernel
                and not use_gemv
                and (not use_fqt or c4[1].dim() == 3)          # the tile-major fqt7 GEMM
                and (self.salient_indices is None or pw.K - pw.S > 0))
        colmax = ops.out_quant_workspace(x2.shape[0], pw.N, x2.device)["buf"] if fuse else None
        if use_f8:
            y = ops.gemm_f8(a8, sa, xs, pw, bias, colmax=colmax)
        elif use_fqt:
            y = ops.gemm_fqt(*c4, pw, bias, ag, colmax=colmax)
        elif use_h2:
            y = ops.gemm_h2_planes(a2, pw, bias, colmax=colmax)
        elif use_gemv:
            y = ops.gemv(a, pw, bias, packed=True)
        else:
            y = ops.gemm_fq(a, pw, bias, colmax=colmax)
        if ospec is not None:                                                # :308-316
            omode, obits, og = ospec
            if self.salient_indices is not None:
                if pw.K - pw.S > 0:
                    ops.fake_quant_inplace(y, omode, obits, og, pw.amap_fq, pw.nonsal, pw.S,
                                           stats_given=fuse)
            else:
                if self.out_amap_fq is None:
                    _, _, self.out_amap_fq, self.out_nonsal = ops.build_maps(pw.N, None, y.device)
                ops.fake_quant_inplace(y, omode, obits, og, self.out_amap_fq, self.out_nonsal, 0,
                                       stats_given=fuse)
        if len(x_shape) == 3:
            return y.view(x_shape[0], x_shape[1], -1)
        return y

    # ------------------------------------------------------------------ from_float
    @staticmethod
    def from_float(module, weight_quant="per_channel", act_quant="per_token",
                   quantize_output=False, importance=None, salient_prop=0, quant_bits=4,
                   group_size=128):
        assert isinstance(module, torch.nn.Linear)                           # :335
        new_module = W4A4Linear(module.in_features, module.out_features,
                                module.bias is not None, act_quant=act_quant,
                                quantize_output=quantize_output, importance=importance,
                                salient_prop=salient_prop, quant_bits=quant_bits,
                                group_size=group_size)
        if weight_quant not in _WEIGHT_EXT:
            raise ValueError(f"Invalid weight_quant: {weight_quant}")         # :361
        in_place = weight_quant in ("per_channel", "per_tensor")
        w_hat = new_module._pack_from(module.weight.data, weight_quant, want_w_hat=in_place)
        if in_place:
            # the reference quantizes module.weight IN PLACE for these modes and then
            # restores the salient columns through the alias (:349-355, :363-365): the
            # source Linear (and any weight tied to it) ends up holding W_hat.  W_hat is
            # dequantized on the GPU inside _pack_from, so a CPU-resident source works too.
            with torch.no_grad():
                module.weight.data.copy_(w_hat)
        if module.bias is not None:
            new_module.bias = module.bias                                     # :369-370
        return new_module

    def __repr__(self):
        return (f"W4A4Linear({self.in_features}, {self.out_features}, bias={self.bias is not None}, "
                f"weight_quant={self.weight_quant_name}, act_quant={self.act_quant_name}, "
                f"output_quant={self.output_quant_name}, salient_indices={self.salient_indices})")


# ----------------------------------------------------------------------------------------
# sibling layers (q/k/v, gate/up)
# ----------------------------------------------------------------------------------------
class SiblingGroup:
    """W4A4Linear layers that the model calls one after another on the SAME input tensor:
    q/k/v of an attention block and gate/up of a gated MLP (fake_quant.py:479-561 swaps them
    one by one; the reference then repeats the activation quantization of :291-304 for each).

    The first member called computes every member's output: one quantizer pass for all of
    them (ops.quant_act_fp_group: the column statistics, the rank and the quantized values
    once, each member's operand in its own packed order) and one GEMM launch
    (ops.gemm_fq7_group).  The other members' outputs are kept for their own call on the same
    input object (identity, storage, shape and version must match -- an input changed in
    place, or another tensor, is computed as usual) and handed out once.  Each output is
    bit-identical to the member's own forward unless exactly one of the two launches takes the
    K split inside the workgroup (ops.fq7_plan, OPT bit 16: a member alone on a grid of at most
    one 128-row tile per CU) -- then equal within fp32 rounding of the partial sums; layers that
    the grouped kernels do not cover (other act modes, output quantization, the
    activation-order path, ...) compute alone."""

    def __init__(self, members):
        self.members = list(members)
        self._stash = {}  # member index -> (weakref(x), key(x), y)

    def __getstate__(self):  # (pickling a model: outputs kept for one input are not state)
        return {"members": self.members, "_stash": {}}

    @staticmethod
    def _key(x):
        # (the capture: outputs of a graph are written at its replays only)
        return (x.data_ptr(), tuple(x.shape), tuple(x.stride()), x.dtype, x._version,
                ops.capture_id(ops._raw_stream(x.device.index)) if x.is_cuda else 0)

    @staticmethod
    def _sig(m):
        """What a member's output depends on besides its input: the resolved act / output
        quantizers (a caller may rebind them, e.g. the reference's W4A8 idiom), the kernel
        choice and the bias; the packed weight is compared by identity (packed() returns a new
        PackedWeight whenever a buffer was replaced or written in place)."""
        b = m.bias
        return (m.kernel, resolve_quantizer(m.act_quant), resolve_quantizer(m.output_quant),
                None if b is None else (b.data_ptr(), b._version, b.dtype))

    def _plan(self, x2):
        """(packed weights, biases, (mode, bits, group_size)) when the grouped kernels cover
        every member for this input, else None."""
        spec, pws, biases = None, [], []
        for m in self.members:
            if m.kernel not in ("auto", "gemv") or resolve_quantizer(m.output_quant) is not None:
                return None
            sp = resolve_quantizer(m.act_quant)
            if spec is None:
                spec = sp
            elif sp != spec:
                return None
            pw = m.packed()
            if m._kernel_for(x2.shape[0], pw) != "auto":
                return None
            b = None if m.bias is None else m.bias.reshape(-1)
            if x2.dtype != pw.dtype or (b is not None and (b.dtype != pw.dtype
                                                            or b.device != x2.device)):
                return None
            pws.append(pw)
            biases.append(b)
        if spec is None or not ops.f8_input_ok(x2):
            return None
        if not ops.group_eligible(pws, spec[0], spec[1], spec[2], x2.shape[0]):
            return None
        return pws, biases, spec

    def forward(self, member, x, x2):
        """member's output for x, or None (the member then computes alone)."""
        i = self.members.index(member)
        key = self._key(x)
        e = self._stash.pop(i, None)
        # a stashed output only while the input AND everything the member's forward reads are
        # unchanged since the group ran (a rebound quantizer, a new weight: computed again)
        if (e is not None and e[0]() is x and e[1] == key and e[3] == self._sig(member)
                and member.packed() is e[4]):
            return e[2]
        plan = self._plan(x2)
        if plan is None:
            return None
        pws, biases, (mode, bits, gs) = plan
        a = ops.quant_act_fp_group(x2.contiguous(), pws, mode, bits, gs)
        ys = ops.gemm_fq7_group(a, pws, biases)
        if x.dim() == 3:
            ys = [y.view(x.shape[0], x.shape[1], -1) for y in ys]
        ref = weakref.ref(x)
        self._stash = {j: (ref, key, y, self._sig(self.members[j]), pws[j])
                       for j, y in enumerate(ys) if j != i}
        return ys[i]


def link_siblings(*modules):
    """Declare W4A4Linear layers that the model calls one after another on the same input
    (see SiblingGroup); returns the group.  quantize_llama_like / quantize_mixtral link q/k/v
    and gate/up (w1/w3) themselves; other members than W4A4Linear are ignored."""
    mods = [m for m in modules if isinstance(m, W4A4Linear)]
    if len(mods) < 2:
        return None
    g = SiblingGroup(mods)
    for m in mods:
        m.__dict__["_sqmp_group"] = g
    return g


def use_gemv(model: nn.Module, enable: bool = True) -> int:
    """Switch the W4A4Linear layers of `model` whose kernel is "auto" to "gemv" (enable=False:
    every "gemv" layer to "auto", one set by hand too) and return how many changed: a model that
    decodes a few tokens at a time."""
    was, now = ("auto", "gemv") if enable else ("gemv", "auto")
    n = 0
    for m in model.modules():
        if isinstance(m, W4A4Linear) and m.kernel == was:
            m.kernel, n = now, n + 1
    return n


# ----------------------------------------------------------------------------------------
# model surgery (fake_quant.py:377-799)
# ----------------------------------------------------------------------------------------
def _importance(input_feat, key, guarded):
    if guarded:
        return sum(input_feat[key]).float() if input_feat else None
    return sum(input_feat[key]).float()


def _swap(parent, attr, key, input_feat, guarded, quantize_output=False, **kw):
    imp = _importance(input_feat, key, guarded)
    setattr(parent, attr, W4A4Linear.from_float(getattr(parent, attr), importance=imp,
                                                quantize_output=quantize_output, **kw))


def quantize_opt(model, weight_quant="per_tensor", act_quant="per_tensor",
                 quantize_bmm_input=True, input_feat=None, salient_prop=0, quant_bits=4,
                 group_size=128):
    """fake_quant.py:377-461 (no guard on input_feat: a missing key raises KeyError)."""
    from transformers.models.opt.modeling_opt import OPTAttention, OPTDecoderLayer
    kw = dict(weight_quant=weight_quant, act_quant=act_quant, salient_prop=salient_prop,
              quant_bits=quant_bits, group_size=group_size)
    for name, m in list(model.model.named_modules()):
        pre = "model." + name + "."
        if isinstance(m, OPTDecoderLayer):
            _swap(m, "fc1", pre + "fc1", input_feat, False, **kw)
            _swap(m, "fc2", pre + "fc2", input_feat, False, **kw)
        elif isinstance(m, OPTAttention):
            for proj in ("q_proj", "k_proj", "v_proj"):
                _swap(m, proj, pre + proj, input_feat, False, quantize_output=quantize_bmm_input, **kw)
            _swap(m, "out_proj", pre + "out_proj", input_feat, False, **kw)
    return model


def quantize_llama_like(model, weight_quant="per_channel", act_quant="per_token",
                        quantize_bmm_input=False, input_feat=None, salient_prop=0, quant_bits=4,
                        group_size=128):
    """fake_quant.py:464-561 (Llama and Mistral)."""
    from transformers.models.llama.modeling_llama import LlamaAttention, LlamaMLP
    from transformers.models.mistral.modeling_mistral import MistralAttention, MistralMLP
    kw = dict(weight_quant=weight_quant, act_quant=act_quant, salient_prop=salient_prop,
              quant_bits=quant_bits, group_size=group_size)
    for name, m in list(model.model.named_modules()):
        pre = "model." + name + "."
        if isinstance(m, (LlamaMLP, MistralMLP)):
            for proj in ("gate_proj", "up_proj", "down_proj"):
                _swap(m, proj, pre + proj, input_feat, True, **kw)
            link_siblings(m.gate_proj, m.up_proj)      # both called on the MLP input
        elif isinstance(m, (LlamaAttention, MistralAttention)):
            for proj in ("q_proj", "k_proj", "v_proj"):
                _swap(m, proj, pre + proj, input_feat, True, quantize_output=quantize_bmm_input, **kw)
            _swap(m, "o_proj", pre + "o_proj", input_feat, True, **kw)
            link_siblings(m.q_proj, m.k_proj, m.v_proj)  # all three on the hidden states
    return model


def quantize_mixtral(model, weight_quant="per_channel", act_quant="per_token",
                     quantize_bmm_input=False, input_feat=None, salient_prop=0, quant_bits=4,
                     group_size=128, quantize_experts=False):
    """fake_quant.py:564-668.  Experts are swapped where they are nn.Linear modules
    (w1/w2/w3); transformers >= 5 fuses them into 3-D parameters, which stay unquantized unless
    quantize_experts swaps them for experts.W4A4Experts (its row-wise activation modes and 4 bits
    only; salient columns of gate_up by the router's input statistic, the key `gate`)."""
    from transformers.models.mixtral import modeling_mixtral as mm
    kw = dict(weight_quant=weight_quant, act_quant=act_quant, salient_prop=salient_prop,
              quant_bits=quant_bits, group_size=group_size)
    if quantize_experts:
        from .experts import W4A4Experts
        W4A4Experts(act_quant=act_quant, quant_bits=quant_bits)  # (refuses before anything is swapped)
        for m in model.modules():
            if (isinstance(m, mm.MixtralSparseMoeBlock)
                    and hasattr(getattr(m, "experts", None), "gate_up_proj")):
                W4A4Experts.check(m.experts, weight_quant, act_quant, quant_bits, group_size)
    expert_cls = getattr(mm, "MixtralBLockSparseTop2MLP", None) or getattr(mm, "MixtralBlockSparseTop2MLP", None)
    for name, m in list(model.model.named_modules()):
        pre = "model." + name + "."
        if expert_cls is not None and isinstance(m, expert_cls):
            for proj in ("w1", "w2", "w3"):
                _swap(m, proj, pre + proj, input_feat, True, **kw)
            link_siblings(m.w1, m.w3)                  # w2(act(w1(x)) * w3(x))
        elif isinstance(m, mm.MixtralAttention):
            for proj in ("q_proj", "k_proj", "v_proj"):
                _swap(m, proj, pre + proj, input_feat, True, quantize_output=quantize_bmm_input, **kw)
            _swap(m, "o_proj", pre + "o_proj", input_feat, True, **kw)
            link_siblings(m.q_proj, m.k_proj, m.v_proj)
        elif isinstance(m, mm.MixtralSparseMoeBlock) and isinstance(getattr(m, "gate", None), nn.Linear):
            _swap(m, "gate", pre + "gate", input_feat, True, **kw)
        if (quantize_experts and isinstance(m, mm.MixtralSparseMoeBlock)
                and hasattr(getattr(m, "experts", None), "gate_up_proj")):
            imp = _importance(input_feat, pre + "gate", True) if salient_prop else None
            m.experts = W4A4Experts.from_float(m.experts, importance=imp, **kw)
    return model


def quantize_falcon(model, weight_quant="per_channel", act_quant="per_token",
                    quantize_bmm_input=True, input_feat=None, salient_prop=0, quant_bits=4,
                    group_size=128):
    """fake_quant.py:671-731 (iterates model.named_modules(), keys 'model.' + name)."""
    from transformers.models.falcon.modeling_falcon import FalconAttention, FalconMLP
    kw = dict(weight_quant=weight_quant, act_quant=act_quant, salient_prop=salient_prop,
              quant_bits=quant_bits, group_size=group_size)
    for name, m in list(model.named_modules()):
        pre = "model." + name + "."
        if isinstance(m, FalconMLP):
            _swap(m, "dense_h_to_4h", pre + "dense_h_to_4h", input_feat, True, **kw)
            _swap(m, "dense_4h_to_h", pre + "dense_4h_to_h", input_feat, True, **kw)
        elif isinstance(m, FalconAttention):
            _swap(m, "query_key_value", pre + "query_key_value", input_feat, True,
                  quantize_output=quantize_bmm_input, **kw)
            _swap(m, "dense", pre + "dense", input_feat, True, **kw)
    return model


def quantize_model(model, weight_quant="per_channel", act_quant="per_token",
                   quantize_bmm_input=False, input_feat=None, salient_prop=None, quant_bits=4,
                   group_size=128, min_prop=0, max_prop=0, quantize_experts=False):
    """fake_quant.py:734-799: dispatch on the HF model class (quantize_experts: quantize_mixtral)."""
    if input_feat is None:
        input_feat = {}
    from transformers.models.falcon.modeling_falcon import FalconPreTrainedModel
    from transformers.models.llama.modeling_llama import LlamaPreTrainedModel
    from transformers.models.mistral.modeling_mistral import MistralPreTrainedModel
    from transformers.models.mixtral.modeling_mixtral import MixtralPreTrainedModel
    from transformers.models.opt.modeling_opt import OPTPreTrainedModel
    kw = dict(weight_quant=weight_quant, act_quant=act_quant,
              quantize_bmm_input=quantize_bmm_input, input_feat=input_feat,
              salient_prop=salient_prop, quant_bits=quant_bits, group_size=group_size)
    if isinstance(model, OPTPreTrainedModel):
        return quantize_opt(model, **kw)
    if isinstance(model, (LlamaPreTrainedModel, MistralPreTrainedModel)):
        return quantize_llama_like(model, **kw)
    if isinstance(model, MixtralPreTrainedModel):
        return quantize_mixtral(model, quantize_experts=quantize_experts, **kw)
    if isinstance(model, FalconPreTrainedModel):
        return quantize_falcon(model, **kw)
    raise ValueError(f"Unsupported model type: {type(model)}")
