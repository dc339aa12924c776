"""What needs no GPU of the few-row and expert operators: the C entries' refusals, the modules'
argument checks and the host-side layouts."""
import inspect

import pytest
import torch

from smoothquant import _lib, experts, fake_quant, ops

P = 4096  # a non-null, 16-B aligned pointer that no refused call may follow


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_gemv_refusals(lib):
    def call(x=P, ldx=128, cols=None, amap=None, salient=None, S=0, codes=P, scale=P, sal=None, bias=None, y=P, dtype=1,
             M=1, N=32, Kp=128, S_pad=0, Gw=64, ngw=2):
        return lib.sqmp_gemv_w4(x, ldx, Kp if cols is None else cols, amap, salient, S, codes, scale, sal, bias, y, dtype, M, N, Kp, S_pad, Gw, ngw, None, 0, None)
    assert call(M=0) == 0 and call(M=0, cols=64, ldx=64) == 0   # nothing to do
    for bad in (dict(x=None), dict(codes=None), dict(scale=None), dict(y=None), dict(S_pad=64, ldx=192),
                dict(M=-1), dict(M=65), dict(N=0), dict(Kp=64), dict(Kp=100), dict(S_pad=-64),
                dict(S_pad=32, sal=P), dict(Gw=0), dict(ngw=0), dict(ldx=127), dict(ldx=132),
                dict(x=P + 2), dict(ldx=64), dict(cols=32), dict(cols=192), dict(cols=0), dict(cols=-64),
                dict(cols=64, S_pad=64, sal=P, ldx=192), dict(cols=64, ldx=56), dict(cols=64, amap=P)):
        assert call(**bad) == -1, bad
    assert call(dtype=3) == -2
    assert call(Gw=12) == -2                                # groups of whole 8 positions only
    assert call(dtype=0, ldx=130) == -1
    assert call(S=1, amap=P, S_pad=64, sal=P) == -1 and call(S=65, S_pad=64, sal=P, ldx=192) == -1
    assert call(amap=P, ldx=0) == -1
    # rows gathered by the kernel: few enough for its LDS
    assert lib.sqmp_gemv_gathers(1, 1, 12800, 0) == 1 and lib.sqmp_gemv_gathers(1, 1, 16384, 0) == 0
    assert lib.sqmp_gemv_gathers(1, 17, 128, 0) == 0
    assert lib.sqmp_gemv_gathers(1, 16, 4096, 0) == 0 and call(amap=P, M=16, Kp=4096, ngw=64) == -2


def test_expert_linear_refusals(lib):
    def call(x=P, ldx=128, cols=None, rows=None, top_k=2, offsets=P, E=4, codes=P, scale=P, sal=None, y=P, dtype=1, slots=8,
             x_rows=4, N=32, n_out=32, Kp=128, S_pad=0, Gw=64, ngw=2, act=0):
        return lib.sqmp_expert_linear_w4(x, ldx, Kp if cols is None else cols, rows, top_k, offsets, E, codes, scale, sal, y, dtype, slots,
                                         x_rows, N, n_out, Kp, S_pad, Gw, ngw, act, None, 0, None)
    assert call(slots=0) == 0
    for bad in (dict(x=None), dict(offsets=None), dict(y=None), dict(E=0), dict(E=65536), dict(top_k=0),
                dict(slots=-1), dict(x_rows=-1), dict(act=3), dict(act=-1), dict(n_out=31), dict(act=1),
                dict(act=1, n_out=17), dict(act=1, N=64, n_out=16), dict(act=1, N=40, n_out=20),
                dict(S_pad=64, ldx=192), dict(ldx=120)):
        assert call(**bad) == -1, bad


def test_routing_refusals(lib):
    def route(T=4, E=8, k=2, ldl=8, dtype=1, logits=P, w=P, ids=P, off=P, rows=P, slots=P, ws=None, n=0):
        return lib.sqmp_route(logits, ldl, dtype, T, E, k, 1, w, ids, off, rows, slots, ws, n, None)
    for bad in (dict(T=-1), dict(E=0), dict(k=0), dict(k=9), dict(ldl=7), dict(logits=None), dict(w=None),
                dict(ids=None), dict(off=None), dict(rows=None), dict(slots=None)):
        assert route(**bad) == -1, bad
    for bad in (dict(E=257, ldl=257), dict(k=17, E=20, ldl=20), dict(dtype=7)):
        assert route(**bad) == -2, bad
    assert route(T=257) == -4 and route(T=257, ws=P, n=8) == -4      # workspace
    assert lib.sqmp_route_workspace_bytes(256, 8) == 0
    assert lib.sqmp_route_workspace_bytes(257, 8) == 3 * 8 * 4
    assert lib.sqmp_plan_routes(None, 4, 8, 2, P, P, P, None, 0, None) == -1
    assert lib.sqmp_combine(None, 1, 4, 2, 8, P, P, P, None) == -1
    assert lib.sqmp_combine(None, 1, 0, 2, 8, None, None, None, None) == 0
    assert lib.sqmp_combine(P, 1, 4, 0, 8, P, P, P, None) == -1
    assert lib.sqmp_combine(P, 9, 4, 2, 8, P, P, P, None) == -2
    assert lib.sqmp_pack_rows(P, 8, 1, 4, None, 128, None, 0, 0, None, 1, None, 0, 0, P, None) == -1
    assert lib.sqmp_pack_rows(P, 8, 1, 4, P, 128, None, 3, 0, None, 1, None, 0, 0, P, None) == -1
    assert lib.sqmp_pack_rows(P, 8, 1, 4, P, 128, None, 0, 0, P, 1, None, 0, 0, P, None) == -1


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8, dtype=torch.float16)
    r = experts.Routing(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1), None, None, None, 1)
    for call in (lambda: ops.gemv(x, None), lambda: experts.route(x, 1),
                 lambda: experts.plan_routes(torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, 1), 8),
                 lambda: experts.expert_linear(x, None, r), lambda: experts.combine(x, r),
                 lambda: ops.pack_codes(torch.zeros(2, 8, dtype=torch.int8), x, 8),
                 lambda: experts.pack_experts(torch.zeros(2, 8, 8))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


def test_bpack_layout():
    """Position p of a 64-position block: dword (p / 8 % 2) * 4 + p / 16, even elements in the low
    half-word, nibble = code + 8."""
    codes = torch.randint(-8, 8, (3, 128), generator=torch.Generator().manual_seed(0), dtype=torch.int8)
    words = ops.bpack_codes(codes).view(torch.int32).view(3, 2, 8)
    for p in range(128):
        e = p & 7
        d, sh = ((p >> 3) & 1) * 4 + ((p & 63) >> 4), (16 if e & 1 else 0) + 4 * (e >> 1)
        assert torch.equal(((words[:, p >> 6, d] >> sh) & 15) - 8, codes[:, p].int())


def test_interleaved_halves():
    t = torch.arange(40).view(1, 40, 1)
    rows = experts._interleave(t).view(2, 2, 16)             # 20 + 20 rows, padded to 32 + 32
    assert rows[0, 0].tolist() == list(range(16)) and rows[0, 1].tolist() == list(range(20, 36))
    assert rows[1, 0, :4].tolist() == [16, 17, 18, 19] and rows[1, 1, :4].tolist() == [36, 37, 38, 39]
    assert rows[1, :, 4:].abs().sum() == 0


def test_module_arguments():
    with pytest.raises(ValueError, match="row by row"):
        experts.W4A4Experts(act_quant="per_group")
    with pytest.raises(ValueError, match="row by row"):
        experts.W4A4Experts(act_quant="per_tensor")
    with pytest.raises(ValueError, match="activation"):
        experts.W4A4Experts(act="relu")
    with pytest.raises(ValueError, match="4 bits"):
        experts.W4A4Experts(quant_bits=8)
    with pytest.raises(ValueError, match="fused"):
        experts.W4A4Experts.from_float(torch.nn.Linear(2, 2))
    assert experts._act_name(torch.nn.SiLU()) == "silu" and experts._act_name(torch.nn.GELU()) == "gelu"
    with pytest.raises(ValueError):
        experts._act_name(torch.nn.GELU(approximate="tanh"))
    m = experts.W4A4Experts()
    with pytest.raises(RuntimeError):
        m(torch.zeros(1, 4), torch.zeros(1, 1, dtype=torch.long), torch.zeros(1, 1))
    # what ran before keeps its results: nothing new by default
    for fn in (fake_quant.quantize_mixtral, fake_quant.quantize_model):
        assert inspect.signature(fn).parameters["quantize_experts"].default is False
    assert fake_quant.W4A4Linear(8, 8).kernel == "auto"


def test_module_state_roundtrip(tmp_path):
    m = experts.W4A4Experts("gelu", None, 4, 64)
    for part in ("gate_up", "down"):
        setattr(m, f"{part}_codes_t", torch.randint(0, 255, (2, 64), dtype=torch.uint8))
        setattr(m, f"{part}_scale_t", torch.randn(2, 8).half())
        setattr(m, f"{part}_amap", torch.arange(128, dtype=torch.int32))
    m._meta = {f"{p}_{n}": 1 for p in ("gate_up", "down") for n in experts._INTS} | {"dtype": torch.float16}
    path = str(tmp_path / "e.pt")
    torch.save(m.state_dict(), path)
    sd = torch.load(path, weights_only=True)
    fresh = experts.W4A4Experts()
    fresh.load_state_dict(sd, strict=True)
    assert fresh.act == "gelu" and fresh.act_quant is None and fresh.group_size == 64
    assert fresh._meta["dtype"] is torch.float16 and fresh._meta["gate_up_gated"] is True
    for k, v in m.state_dict().items():
        if not k.endswith("_extra_state"):
            assert torch.equal(fresh.state_dict()[k], v)
    with pytest.raises(RuntimeError, match="cast"):
        fresh.float()


def test_calls_make_their_tensors_device_current(monkeypatch):
    """A device's default stream is the null handle: the calls enter their tensor's device when it is
    not the current one (shown with a stand-in for a tensor on the second device)."""
    class OnDevice1(torch.Tensor):
        is_cuda = True
        device = torch.device("cuda", 1)

    entered = []

    class Ctx:
        def __init__(self, dev):
            entered.append(dev)

        def __enter__(self):
            monkeypatch.setattr(ops, "_current_device", lambda: 1)

        def __exit__(self, *exc):
            monkeypatch.setattr(ops, "_current_device", lambda: 0)
            return False

    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "device", Ctx)
    t = torch.zeros(2, 8).as_subclass(OnDevice1)
    seen = ops.on_tensor_device(lambda x, y: (ops._current_device(), y))(t, 5)
    assert seen == (1, 5) and entered == [torch.device("cuda", 1)] and ops._current_device() == 0
    assert ops.on_tensor_device(lambda x: ops._current_device())(torch.zeros(1)) == 0
    for fn in (ops.pack_codes, ops.tile_major, ops.pack_rows, ops.gemv, experts.route, experts.plan_routes,
               experts.pack_experts, experts.pack_expert_codes, experts.expert_linear, experts.combine):
        assert fn.__wrapped__ is not None
