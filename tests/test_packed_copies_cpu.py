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
