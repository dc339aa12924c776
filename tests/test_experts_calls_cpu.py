"""The expert calls up to their kernels, without a GPU: host tensors that say they are on one, and a
library that records the calls and does nothing."""
import pytest
import torch

from smoothquant import experts, ops

CUDA0 = torch.device("cuda", 0)


class OnGpu(torch.Tensor):
    """A host tensor that says that it is on the first GPU."""
    is_cuda = True
    device = CUDA0


def gpu(t):
    return t.as_subclass(OnGpu)


class Library:
    """Every entry succeeds; the calls are kept."""
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, args))
            return 0
        return entry


@pytest.fixture
def library(monkeypatch):
    lib = Library()
    for m in (ops, experts):
        monkeypatch.setattr(m, "load", lambda: lib)
    monkeypatch.setattr(ops, "_SPLIT_WS", {})
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    return lib


def routing(T=4, k=2, E=3, dtype=torch.int32):
    i32 = dict(dtype=dtype)
    return experts.Routing(gpu(torch.zeros(T, k, **i32)), gpu(torch.ones(T, k)),
                           gpu(torch.zeros(E + 1, **i32)), gpu(torch.zeros(T * k, **i32)),
                           gpu(torch.zeros(T * k, **i32)), E)


def weight(E=3, N=32, K=128, dtype=torch.float16):
    return experts.PackedExperts(gpu(torch.zeros(E, 256, dtype=torch.uint8)), gpu(torch.zeros(E, 64, dtype=dtype)),
                                 None, gpu(torch.arange(K, dtype=torch.int32)), None, E, N, N, K, K, 0, 0,
                                 64, K // 64, dtype, False, True)


def test_out_is_a_write_that_torch_sees(library):
    """A kernel writes `out` through its address; its version counter, by which results kept for a
    tensor are told from those for its former contents, has to rise as for a write of torch's own."""
    r = routing()
    base = torch.zeros(9, 64, dtype=torch.float16)
    y = gpu(base[1:5])                                       # a view: one counter with its base
    was = base._version
    assert experts.combine(gpu(torch.zeros(8, 64, dtype=torch.float16)), r, out=y) is y
    assert y._version > was and base._version > was
    z = gpu(torch.zeros(8, 32, dtype=torch.float16))
    was = z._version
    assert experts.expert_linear(gpu(torch.zeros(4, 128, dtype=torch.float16)), weight(), r, out=z) is z
    assert z._version > was
    assert [c[0] for c in library.calls if "workspace" not in c[0]] == ["sqmp_combine", "sqmp_expert_linear_w4"]
    was = z._version
    with pytest.raises(ValueError):                          # refused: nothing written
        experts.expert_linear(gpu(torch.zeros(4, 128, dtype=torch.float16)), weight(), r, act="silu", out=z)
    assert z._version == was
    with torch.inference_mode():                             # (tensors without a counter)
        o = gpu(torch.zeros(4, 64, dtype=torch.float16))
        assert experts.combine(gpu(torch.zeros(8, 64, dtype=torch.float16)), r, out=o) is o


def test_packed_operands_written_into_tensors_of_the_caller(library, monkeypatch):
    monkeypatch.setattr(ops, "_stream", lambda t: None)
    out = tuple(gpu(torch.zeros(0, dtype=d)) for d in (torch.uint8, torch.float16, torch.float16))
    was = [t._version for t in out]
    ops.tile_major(gpu(torch.zeros(1, dtype=torch.uint8)), gpu(torch.zeros(1).half()), gpu(torch.zeros(1).half()),
                   32, 128, 0, 2, torch.float16, out)
    assert all(t._version > v for t, v in zip(out, was))


def test_every_capture_has_its_own_workspaces(library, monkeypatch):
    """A graph's workspace is cleared inside the graph (it is allocated in its capture) and belongs to
    it alone: not the eager one of the stream, not that of another capture."""
    capture = [0]
    monkeypatch.setattr(ops, "capture_id", lambda stream: capture[0])
    monkeypatch.setattr(ops, "_WS", {})
    dev = torch.device("cpu")

    def ws():
        return ops._act_ws(dev, 7, 64, 128, 1024)
    eager = ws()
    eager["stats"] = "of an eager call"
    capture[0] = 3
    first = ws()
    assert first is not eager and first["stats"] is None and ws() is first
    capture[0] = 4
    second = ws()
    assert second is not first and second["buf"].data_ptr() != eager["buf"].data_ptr()
    capture[0] = 0
    assert ws() is eager and eager["stats"] == "of an eager call"
    ops._discard_ws(eager)                                    # after a failure
    assert ws() is not eager


def test_outputs_kept_for_siblings_do_not_leave_their_capture(monkeypatch):
    from smoothquant.fake_quant import SiblingGroup
    capture = [0]
    monkeypatch.setattr(ops, "capture_id", lambda stream: capture[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 7)
    x = gpu(torch.zeros(2, 8))
    key = SiblingGroup._key(x)
    assert SiblingGroup._key(x) == key
    capture[0] = 3
    assert SiblingGroup._key(x) != key


def test_capture_id_outside_of_a_capture():
    assert ops.capture_id(0) == 0


# ------------------------------------------------------------------ routings by hand
def _combine(r, T=4, k=2):
    return experts.combine(gpu(torch.zeros(T * k, 64, dtype=torch.float16)), r)


def _linear(r, T=4):
    return experts.expert_linear(gpu(torch.zeros(T, 128, dtype=torch.float16)), weight(), r)


@pytest.mark.parametrize("name,call", [("rows", _linear), ("offsets", _linear), ("slots", _combine)])
@pytest.mark.parametrize("bad", [lambda t: gpu(t.long()), lambda t: gpu(t.float()), lambda t: gpu(t[:-1]),
                                 lambda t: gpu(torch.zeros(2 * len(t), dtype=torch.int32))[::2],
                                 lambda t: gpu(t.view(-1, 1)[:0]), lambda t: torch.zeros(t.shape, dtype=torch.int32),
                                 lambda t: None], ids=["int64", "float", "short", "strided", "empty", "host", "none"])
def test_lists_that_the_kernels_would_misread(library, name, call, bad):
    """The kernels read a routing's lists as contiguous int32 of the routing's size on x's device: any
    other tensor there is refused before a launch."""
    r = routing()
    call(r)
    assert library.calls
    library.calls.clear()
    t = getattr(r, name)
    setattr(r, name, bad(torch.Tensor(t) if t.dtype.is_floating_point else t.as_subclass(torch.Tensor)))
    with pytest.raises((ValueError, RuntimeError), match=name):
        call(r)
    assert not [c for c in library.calls if "workspace" not in c[0]]


def test_weights_of_another_type_or_stride(library):
    """Router weights cast to the model's type, or strided, are converted as plan_routes converts them;
    of another shape or on another device, refused."""
    def passed():
        return [c for c in library.calls if c[0] == "sqmp_combine"][-1][1][6]
    for w in (torch.rand(4, 2).half(), torch.rand(4, 2).bfloat16(), torch.rand(4, 2).double(),
              torch.rand(2, 4).t(), torch.rand(4, 4)[:, ::2], torch.rand(1, 2).expand(4, 2)):
        r = routing()
        r.weights = gpu(w)
        before = r.weights
        _combine(r)
        assert passed() != w.data_ptr()                       # a converted copy
        assert r.weights is before
    r = routing()
    _combine(r)
    assert passed() == r.weights.data_ptr()
    for w in (torch.rand(8), torch.rand(4, 1), torch.rand(2, 4), torch.rand(0, 2)):
        r.weights = gpu(w)
        with pytest.raises(ValueError, match="weights"):
            _combine(r)
    r.weights = torch.rand(4, 2)
    with pytest.raises(RuntimeError, match="weights"):
        _combine(r)
    r = routing()
    r.ids = gpu(torch.zeros(8, dtype=torch.int32))
    for call in (_combine, _linear):
        with pytest.raises(ValueError, match="ids"):
            call(r)


@pytest.mark.parametrize("rows,eligible,grouped", [(65, True, True), (64, True, False), (1, True, False), (3, False, True)])
def test_linked_layers_switched_to_gemv_stay_a_group_on_prompts(monkeypatch, rows, eligible, grouped):
    """"gemv" is "auto" for more rows than the few-row product takes, and for weights that it does not:
    linked layers share their quantizer pass and product there, as with "auto"."""
    from smoothquant import fake_quant
    layers = [fake_quant.W4A4Linear(64, 32, bias=False, act_quant="per_group") for _ in range(2)]
    pw = type("Pw", (), dict(dtype=torch.float16))()
    for m in layers:
        monkeypatch.setattr(m, "packed", lambda: pw)
    monkeypatch.setattr(ops, "gemv_eligible", lambda p: eligible)
    monkeypatch.setattr(ops, "group_eligible", lambda *a: True)
    g = fake_quant.link_siblings(*layers)
    x = torch.zeros(max(rows, 8), 64, dtype=torch.float16)[:rows]
    monkeypatch.setattr(ops, "f8_input_ok", lambda x: True)
    assert g._plan(x) is not None
    assert fake_quant.use_gemv(torch.nn.ModuleList(layers)) == 2
    assert (g._plan(x) is not None) == grouped
    layers[1].kernel = "fq"
    assert g._plan(x) is None


def test_calls_by_keyword(library, monkeypatch):
    """The tensor by whose device a call goes may be given by its name, as any argument."""
    r = routing()
    assert experts.combine(z=gpu(torch.zeros(8, 64).half()), routing=r).shape == (4, 64)
    assert experts.combine(routing=r, z=gpu(torch.zeros(8, 64).half())).shape == (4, 64)
    assert experts.expert_linear(x=gpu(torch.zeros(4, 128).half()), pe=weight(), routing=r).shape == (8, 32)
    for call in (lambda: experts.route(top_k=2, logits=torch.zeros(4, 3)),       # (reached: host tensors)
                 lambda: experts.plan_routes(num_experts=3, weights=torch.zeros(4, 2), ids=torch.zeros(4, 2)),
                 lambda: ops.gemv(x=torch.zeros(1, 8), pw=None),
                 lambda: experts.pack_experts(w=torch.zeros(2, 8, 8))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()
    for name in ("pack_codes", "pack_rows", "tile_major"):
        with pytest.raises(TypeError, match="missing"):
            getattr(ops, name)()
    entered = []
    monkeypatch.setattr(ops, "_current_device", lambda: 1)

    class Ctx:
        def __init__(self, dev):
            entered.append(dev)

        def __enter__(self):
            return self

        def __exit__(self, *exc):
            return False
    monkeypatch.setattr(torch.cuda, "device", Ctx)
    experts.combine(routing=r, z=gpu(torch.zeros(8, 64).half()))
    assert entered == [CUDA0]


# ------------------------------------------------------------------ calls to refuse
def test_out_in_the_memory_of_the_operand(library):
    """A product reads its rows while it writes others': `out` may not share memory with them."""
    r = routing()
    buf = torch.zeros(40, 64, dtype=torch.float16)
    z = gpu(buf[:8])
    for at in (0, 3, 7):
        with pytest.raises(ValueError, match="overlap"):
            experts.combine(z, r, out=gpu(buf[at:at + 4]))
    assert experts.combine(z, r, out=gpu(buf[8:12])) is not None
    assert experts.combine(gpu(buf[4:12]), r, out=gpu(buf[:4])) is not None
    pe = weight(N=128)
    buf = torch.zeros(40, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="overlap"):
        experts.expert_linear(gpu(buf[:8]), pe, r, rows="slot", out=gpu(buf[:8]))
    with pytest.raises(ValueError, match="overlap"):
        experts.expert_linear(gpu(buf[7:11]), pe, r, out=gpu(buf[:8]))
    with pytest.raises(ValueError, match="overlap"):          # rows apart, the last one inside
        experts.expert_linear(gpu(buf[:40:10]), pe, r, out=gpu(buf[30:38]))
    assert experts.expert_linear(gpu(buf[:31:10]), pe, r, out=gpu(buf[31:39])) is not None
    n = len([c for c in library.calls if "workspace" not in c[0]])
    assert n == 3


@pytest.mark.parametrize("T,k", [(2 ** 32 + 5, 1), (2 ** 31, 1), (2 ** 28, 8)])
def test_more_pairs_than_the_lists_can_number(library, T, k):
    """Slots and pairs are 32-bit numbers: more of them are refused, not wrapped."""
    with pytest.raises(ValueError, match="pairs"):
        experts.route(gpu(torch.zeros(1, 8).expand(T, 8)), k)
    with pytest.raises(ValueError, match="pairs"):
        experts.plan_routes(gpu(torch.zeros(1, k, dtype=torch.int32).expand(T, k)),
                            gpu(torch.zeros(1, k).expand(T, k)), 8)
    assert not library.calls


def test_rows_wider_than_the_kernels_count(library):
    r = routing()
    with pytest.raises(ValueError, match="columns"):
        experts.combine(gpu(torch.zeros(1, 1, dtype=torch.float16).expand(8, 2 ** 32 + 8)), r)
    assert not library.calls


@pytest.mark.parametrize("call", ["experts", "linear", "linear_group", "pack"])
def test_modules_run_on_their_inputs_device(monkeypatch, call):
    """A device's default stream is the null handle, which a C entry takes for the current device's: a
    module called with a tensor of another device makes that one current for all of its launches."""
    from smoothquant import fake_quant
    current, seen = [0], []
    monkeypatch.setattr(ops, "_current_device", lambda: current[0])

    class Ctx:
        def __init__(self, dev):
            self.dev = torch.device(dev) if not isinstance(dev, torch.device) else dev

        def __enter__(self):
            self.was, current[0] = current[0], self.dev.index

        def __exit__(self, *exc):
            current[0] = self.was
            return False
    monkeypatch.setattr(torch.cuda, "device", Ctx)

    class OnSecond(OnGpu):
        device = torch.device("cuda", 1)
    x = torch.zeros(2, 64, dtype=torch.float16).as_subclass(OnSecond)

    class Reached(Exception):
        pass

    def reached(*a, **k):
        seen.append(current[0])
        raise Reached
    if call == "experts":
        m = experts.W4A4Experts()
        monkeypatch.setattr(m, "packed", reached)
        run = lambda: m(x, torch.zeros(2, 1, dtype=torch.long), torch.ones(2, 1))
    elif call == "pack":
        monkeypatch.setattr(ops, "geometry", reached)
        run = lambda: ops.pack_weight(x, "per_channel", 4, 64, None)
    else:
        m = fake_quant.W4A4Linear(64, 8, bias=False)
        if call == "linear_group":
            fake_quant.link_siblings(m, fake_quant.W4A4Linear(64, 8, bias=False))
            monkeypatch.setattr(fake_quant.SiblingGroup, "forward", reached)
        monkeypatch.setattr(m, "packed", reached)
        run = lambda: m(x)
    with pytest.raises(Reached):
        run()
    assert seen == [1] and current == [0]


@pytest.mark.parametrize("config,kw,match", [
    (dict(hidden_act="relu"), {}, "activation"),
    (dict(hidden_act="gelu_new"), {}, "activation"),
    ({}, dict(weight_quant="per_group", group_size=12), "multiple of 8"),
    ({}, dict(weight_quant="none"), "weight_quant"),
    (dict(num_local_experts=260), {}, "experts"),
    ({}, dict(act_quant="per_group"), "row by row"),
    ({}, dict(quant_bits=8), "4 bits")])
def test_quantize_mixtral_refuses_before_it_swaps_anything(monkeypatch, config, kw, match):
    """Experts that cannot be packed: the model is left whole, not with its first layers quantized."""
    from transformers import MixtralConfig, MixtralForCausalLM
    from smoothquant import fake_quant
    c = dict(vocab_size=16, hidden_size=32, intermediate_size=24, num_hidden_layers=1, num_attention_heads=2,
             num_key_value_heads=2, num_local_experts=2, num_experts_per_tok=1)
    model = MixtralForCausalLM(MixtralConfig(**dict(c, **config)))
    if not any(hasattr(m, "gate_up_proj") for m in model.modules()):
        pytest.skip("experts are not fused in this version of transformers")
    swapped = []
    monkeypatch.setattr(fake_quant, "_swap", lambda *a, **k: swapped.append(a[1]))
    with pytest.raises(ValueError, match=match):
        fake_quant.quantize_model(model, quantize_experts=True, **kw)
    assert not swapped


def test_pack_rows_refuses_maps_it_would_misread(library):
    """ops.pack_rows: int32 maps of the operand's size, on the rows' device."""
    x = gpu(torch.zeros(3, 64, dtype=torch.float16))
    amap, sal = gpu(torch.arange(128, dtype=torch.int32)), gpu(torch.arange(4, dtype=torch.int32))

    def call(x=x, amap=amap, Kp=128, salient=None, S=0, S_pad=0):
        return ops.pack_rows(x, amap, Kp, salient, S, S_pad)
    assert call().shape == (3, 128) and call(salient=sal, S=4, S_pad=64).shape == (3, 192)
    library.calls.clear()
    for bad in (dict(amap=gpu(torch.arange(128))), dict(amap=gpu(torch.arange(127, dtype=torch.int32))),
                dict(amap=gpu(torch.arange(256, dtype=torch.int32))[::2]), dict(amap=None), dict(Kp=0), dict(x=x[0]),
                dict(salient=sal, S=5, S_pad=64), dict(S=4, S_pad=64), dict(salient=sal, S=4, S_pad=2),
                dict(salient=gpu(torch.arange(4)), S=4, S_pad=64), dict(S=-1), dict(x=x.int())):
        with pytest.raises(ValueError):
            call(**bad)
    for bad in (dict(amap=torch.arange(128, dtype=torch.int32)),
                dict(salient=torch.arange(4, dtype=torch.int32), S=4, S_pad=64)):
        with pytest.raises((ValueError, RuntimeError)):
            call(**bad)
    assert not library.calls
