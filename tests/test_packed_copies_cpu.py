"""Copies of packed weights own what they use: nothing in a copied, pickled or replaced PackedWeight
(or in a layer that holds one) is an address in the original's memory."""
import copy
import dataclasses
import io
import pickle

import pytest
import torch

from smoothquant import ops
from smoothquant.fake_quant import W4A4Linear

N, K = 8, 128


def packed(dt=torch.float16):
    i32 = dict(dtype=torch.int32)
    return ops.PackedWeight(torch.zeros(256, K // 2, dtype=torch.uint8), torch.zeros(2, 256, dtype=dt),
                            torch.zeros(N, 0, dtype=dt), torch.arange(K, **i32), torch.arange(K, **i32),
                            torch.arange(K, **i32), torch.arange(K, **i32), None, N, K, 0, 0, K, 64, 2, 4, 2, dt)


def fill(pw):
    """The fields that the first gemv fills."""
    pw.ident = True
    pw.gemv = (torch.zeros(4096, dtype=torch.uint8), torch.zeros(512, dtype=pw.dtype), torch.zeros(0, dtype=pw.dtype))
    ops._gemv_args(pw)
    assert pw.gemv_args is not None
    return pw


def tensors(v):
    if isinstance(v, torch.Tensor):
        yield v
    elif isinstance(v, (tuple, list)):
        for i in v:
            yield from tensors(i)


def addresses(pw):
    return {t.data_ptr() for f in dataclasses.fields(pw) for t in tensors(getattr(pw, f.name)) if t.numel()}


def ints(v):
    if isinstance(v, bool):
        return
    if isinstance(v, int):
        yield int(v)
    elif isinstance(v, (tuple, list)):
        for i in v:
            yield from ints(i)


def check_copy(src, dst, same_tensors=False):
    foreign = addresses(src)
    for f in dataclasses.fields(dst):
        v = getattr(dst, f.name)
        assert not foreign & set(ints(v)), f.name            # no address of the original as a number
        if not same_tensors:
            assert not foreign & {t.data_ptr() for t in tensors(v) if t.numel()}, f.name
    a = dst.gemv_args or ops._gemv_args(dst)
    own = {t.data_ptr() for t in tensors(dst.gemv)}
    assert all(t.data_ptr() in own for t in tensors(a))      # what a product of the copy would read
    assert a[1] == dst.codes.device


@pytest.fixture(autouse=True)
def host_operands(monkeypatch):
    """gemv's operands of a weight on the host (this test looks at who owns them)."""
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops, "tile_major", lambda *a, **k: (
        torch.zeros(4096, dtype=torch.uint8), torch.zeros(512, dtype=torch.float16),
        torch.zeros(0, dtype=torch.float16)))


def test_packed_weight():
    src = fill(packed())
    check_copy(src, copy.deepcopy(src))
    check_copy(src, pickle.loads(pickle.dumps(src)))
    buf = io.BytesIO()
    torch.save(src, buf)
    buf.seek(0)
    check_copy(src, torch.load(buf, weights_only=False))
    check_copy(src, copy.copy(src), same_tensors=True)
    check_copy(src, dataclasses.replace(src), same_tensors=True)
    check_copy(src, dataclasses.replace(src, salient=None), same_tensors=True)
    # another weight in the place of the codes: no operand of the former one
    other = dataclasses.replace(src, codes=torch.ones_like(src.codes))
    assert other.gemv is None and other.gemv_args is None


def test_the_arguments_hold_the_tensors_not_their_addresses():
    """The operands' memory can be exchanged (`.data = ...`, a load with another map): what a call
    passes is read from the tensors then."""
    pw = fill(packed())
    assert not addresses(pw) & set(ints(pw.gemv_args))
    kept = list(tensors(pw.gemv_args))
    assert kept and all(any(t is o for o in pw.gemv) for t in kept)


def test_layer_loaded_from_a_state_dict():
    """A layer whose buffers a state dict filled (their versions are those of copied tensors): its
    cached weight does not carry the original's addresses into a copy."""
    lin = W4A4Linear(K, N, bias=False)
    pw = packed()
    pw.posmap, pw.sal_key = torch.arange(K, dtype=torch.int32), ops.salient_key(K, None)
    lin._install(pw, "per_group_unsorted")
    loaded = W4A4Linear(K, N, bias=False)
    loaded.load_state_dict(lin.state_dict())
    src = fill(loaded.packed())
    for dst in (copy.deepcopy(loaded), pickle.loads(pickle.dumps(loaded))):
        check_copy(src, dst.packed())
    buf = io.BytesIO()
    torch.save(loaded, buf)
    buf.seek(0)
    check_copy(src, torch.load(buf, weights_only=False).packed())


class Library:
    """Every entry succeeds and does nothing; the calls are kept."""
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            if name == "sqmp_fq7_sizes":
                for a, n in zip(args[-3:], (4096, 512, 0)):
                    a._obj.value = n
            return 0
        return entry


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    monkeypatch.setattr(ops, "load", lambda: lib)
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    monkeypatch.setattr(ops, "_p", lambda t: None)
    return lib


def test_operands_first_built_in_a_capture_are_not_kept(library, monkeypatch):
    """The copies that a capture builds are written at its replays only: neither gemm_fq7 nor gemv,
    which share them, may use them outside of it."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    pw = packed()
    first = ops.fq7_operands(pw)
    assert pw.fq7 is None and first[3] == ops.FQ7_J
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    t = ops.gemv_operands(pw)
    assert not {v.data_ptr() for v in t if v.numel()} & {v.data_ptr() for v in first[:3] if v.numel()}
    kept = ops.fq7_operands(pw)
    assert pw.fq7 is kept and kept[0] is t[0]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert ops.fq7_operands(pw) is kept                       # built before: used


@pytest.mark.parametrize("name,build", [
    ("w8", lambda pw: ops.f8_operands(pw)), ("ws32", lambda pw: ops.f8_operands(pw)),
    ("h2", lambda pw: ops.h2_operand(pw)), ("h2d", lambda pw: ops.h2d_operand(pw)),
    ("sib_maps", lambda pw: ops._sibling_map(LEADER, pw))])
def test_nothing_that_a_capture_builds_is_kept(library, monkeypatch, name, build):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    pw = packed(torch.float32 if name.startswith("h2") else torch.float16)
    assert build(pw) is not None and getattr(pw, name) is None
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    build(pw)
    kept = getattr(pw, name)
    assert kept is not None
    build(pw)
    assert getattr(pw, name) is kept


LEADER = packed()


def test_grouped_products_hold_their_operands_until_the_launch(library, monkeypatch):
    """In a capture each weight's copies live in the call alone: all of them until the one launch."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    monkeypatch.setattr(ops, "_require_gpu", lambda *a: None)
    import weakref
    born = []
    build = ops.fq7_operands

    def watched(pw):
        o = build(pw)
        born.append(weakref.ref(o[0]))
        return o
    monkeypatch.setattr(ops, "fq7_operands", watched)
    alive = []

    class Lib(Library):
        def __getattr__(self, name):
            if name == "sqmp_gemm_fq7_group":
                return lambda *a: alive.extend(r() is not None for r in born) or 0
            return super().__getattr__(name)
    lib = Lib()
    monkeypatch.setattr(ops, "load", lambda: lib)
    a = [torch.zeros(4, K, dtype=torch.float16) for _ in range(3)]
    ops.gemm_fq7_group(a, [packed() for _ in range(3)], [None] * 3)
    assert alive == [True] * 3
