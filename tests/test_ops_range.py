"""Stream operators without a GPU: sizes beyond 32 bits, kinds of tensors, gradients, alignment."""
import ctypes as ct

import pytest
import torch

from fast_audiovae import _native, build, ops

MANY = 2 ** 31


@pytest.fixture(scope="module", autouse=True)
def library():
    if not build.LIBRARY.exists():
        build.build()


def wide(*shape, dtype=torch.float32):
    """A tensor of any shape that holds one element."""
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape)


@pytest.mark.parametrize("call,words", [
    (lambda: ops.causal_conv(wide(MANY, 8), torch.zeros(8, 4)), "too many rows"),
    (lambda: ops.causal_conv(wide(2, MANY // 2, 8), torch.zeros(8, 4)), "too many rows"),
    (lambda: ops.selective_scan(wide(MANY, 8), wide(MANY, 8), torch.zeros(4, 8), wide(MANY, 1, 4), wide(MANY, 1, 4)),
     "too many rows"),
    (lambda: ops.group_norm(wide(MANY, 8), 4), "too many rows"),
    (lambda: ops.group_norm(wide(1, MANY), 4), "too many rows or channels"),
    (lambda: ops.group_norm(torch.zeros(2, 8), 2 ** 32 + 4), "divides the channels"),
    (lambda: ops.project_int4(wide(MANY, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2), group=32), "too large"),
    (lambda: ops.project_int4(torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2),
                              group=2 ** 32 + 32), "scales must be"),
])
def test_sizes_beyond_32_bits_are_refused(call, words):
    with pytest.raises(ValueError, match=words):
        call()


X, W, Q, S = torch.zeros(6, 64), torch.zeros(64, 4), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2)
MAPS, A, CODES = torch.zeros(6, 1, 4), torch.zeros(4, 64), torch.zeros(6, dtype=torch.int32)
CALLS = [   # a call by its floating point tensors
    (lambda x, w, b, h, out: ops.causal_conv(x, w, b, state=h, codes=CODES, out=out),
     [X, W, torch.zeros(64), torch.zeros(6, 2, 3, 64), X]),
    (lambda x, dt, a, b, c, d, z, bias, h, out: ops.selective_scan(x, dt, a, b, c, d=d, z=z, dt_bias=bias, state=h,
                                                                  codes=CODES, out=out),
     [X, X, A, MAPS, MAPS, torch.zeros(64), X, torch.zeros(64), torch.zeros(6, 2, 4, 64), X]),
    (lambda x, w, b, alpha, r, out: ops.group_norm(x, 4, w, b, activation="snake", alpha=alpha, reciprocal=r, out=out),
     [X] + [torch.zeros(64)] * 4 + [X]),
    (lambda x, s, b, out: ops.project_int4(x, Q, s, b, group=32, out=out), [X, S, torch.zeros(8), torch.zeros(6, 8)]),
]
PLACES = [(call, tensors, i) for call, tensors in CALLS for i in range(len(tensors))]


@pytest.mark.parametrize("call,tensors,place", PLACES)
def test_gradients_of_any_tensor_are_refused(call, tensors, place):
    """Reverse and forward ones, of inputs, states and outputs."""
    def given(t):
        return [t if i == place else other for i, other in enumerate(tensors)]
    leaf = tensors[place].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        call(*given(leaf))
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        call(*given(leaf))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(tensors[place].clone(), torch.ones_like(tensors[place]))
        with pytest.raises(RuntimeError, match="no gradients"):
            call(*given(dual))
        with pytest.raises(RuntimeError, match="no CPU path"):
            call(*tensors)
        with torch.inference_mode(), pytest.raises(RuntimeError, match="no CPU path"):
            call(*(t.clone() for t in tensors))


def test_derivatives_of_functions_are_refused():
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.func.jvp(lambda x: ops.causal_conv(x, W), (X,), (X,))
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.func.grad(lambda x: ops.causal_conv(x, W).sum())(X)


@pytest.fixture
def native_reading(monkeypatch):
    """Tensors go through the native entry points first, which leave those of the CPU to the caller."""
    held = _native.tensor_functions(torch.Tensor)
    assert held
    monkeypatch.setattr(ops, "_held", held)


def without_plain_memory(t):
    yield t.to_sparse()
    yield t.to_mkldnn()
    yield torch.quantize_per_tensor(t, 0.1, 0, torch.qint8)
    yield torch.nested.nested_tensor([t, t], layout=torch.strided)


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("native", [False, True])
def test_tensors_without_plain_memory_are_refused(native, request):
    """Whichever tensor it is, and whichever way it is read, with the reason."""
    if native:
        request.getfixturevalue("native_reading")
    for call, tensors in CALLS:
        for i, t in enumerate(tensors[:-1]):   # outputs are looked at on the device
            for odd in without_plain_memory(t):
                with pytest.raises(ValueError, match="must be|must have"):
                    call(*(odd if j == i else other for j, other in enumerate(tensors)))
    for name in ("offsets", "status"):
        with pytest.raises(ValueError, match=f"{name} must"):
            ops.causal_conv(X, W, **{name: CODES.to_sparse()})
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.causal_conv(X, W)


def negated(t):
    """t as the negative of its memory: the imaginary part of conjugated numbers."""
    return torch.complex(torch.zeros_like(t), -t).conj().imag


@pytest.mark.parametrize("native", [False, True])
def test_negated_views_are_refused(native, request):
    """Their memory holds the opposite sign."""
    if native:
        request.getfixturevalue("native_reading")
    rows, one = torch.arange(6.0), torch.ones(1)
    x = rows[:, None]
    assert torch.equal(negated(rows), rows) and negated(rows).is_neg()
    maps = x.unsqueeze(2)
    for call in (lambda: ops.causal_conv(negated(rows)[:, None], torch.ones(1, 4)),
                 lambda: ops.causal_conv(x, torch.ones(1, 4), negated(one)),
                 lambda: ops.selective_scan(x, x, one[None], negated(rows)[:, None, None], maps),
                 lambda: ops.group_norm(x, 1, negated(one)),
                 lambda: ops.project_int4(torch.zeros(1, 64), Q[:1], negated(one)[None], group=64)):
        with pytest.raises(ValueError, match="must be"):
            call()


FAR = 1 << 24   # no two of the arrays below meet
ARRAYS = {      # fields of the element type, and of 4 bytes
    "fav_causal_conv": ("x y state_pool", "weight bias slot_codes offsets status"),
    "fav_selective_scan": ("x dt z b c y", "a d dt_bias state_pool slot_codes offsets status workspace"),
    "fav_group_norm": ("x y", "weight bias alpha reciprocal offsets status"),
    "fav_project_int4": ("x y", "scales bias"),
}
SIZES = {
    "fav_causal_conv": (_native.ConvArgs, dict(x_stride=8, y_stride=8, channels=8, taps=4, n=2, rows=6, num_slots=2)),
    "fav_selective_scan": (_native.ScanArgs, dict(x_stride=8, dt_stride=8, z_stride=8, b_stride=4, c_stride=4, y_stride=8,
                                                  channels=8, states=4, groups=1, n=2, rows=6, num_slots=2)),
    "fav_group_norm": (_native.NormArgs, dict(x_stride=8, y_stride=8, channels=8, groups=2, n=2, rows=6, eps=1e-5)),
    "fav_project_int4": (_native.Int4Args, dict(x_stride=64, y_stride=8, weight=1 << 20, rows=2, depth=64, out=8, group=32)),
}


@pytest.mark.parametrize("name", list(ARRAYS))
@pytest.mark.parametrize("kind,size", [(0, 4), (1, 2), (2, 2)])
def test_arrays_off_their_elements_are_refused(name, kind, size):
    """Every array of the C ABI, at each address between two elements; such a load would fault."""
    lib = _native.load_library()
    struct, sizes = SIZES[name]
    rows, words = (fields.split() for fields in ARRAYS[name])
    arrays = {field: FAR * (i + 1) for i, field in enumerate(rows + words)}
    for field, width in [(f, size) for f in rows] + [(f, 4) for f in words]:
        for off in range(1, width):
            args = struct(type=kind, **sizes, **{**arrays, field: arrays[field] + off})
            assert getattr(lib, name)(ct.byref(args), None) == 1, (field, off)
            assert b"aligned" in lib.fav_last_error()


def test_codes_into_a_given_tensor():
    slots, out = ops.StreamSlots(4, device="cpu"), torch.zeros(2, dtype=torch.int32)
    assert slots.codes([3, 1], out=out) is out and out.tolist() == [3 << 2 | 2, 1 << 2 | 2]
    for bad in (torch.zeros(3, dtype=torch.int32), torch.zeros(2), torch.zeros(4, dtype=torch.int32)[::2], [0, 0]):
        with pytest.raises(ValueError, match="out must be"):
            slots.codes([3, 1], out=bad)


@pytest.mark.parametrize("name", list(ARRAYS))
def test_outputs_over_any_input_are_refused(name):
    """Each array that a call writes, at the address of each other one."""
    lib = _native.load_library()
    struct, sizes = SIZES[name]
    if name == "fav_selective_scan":   # long enough for a workspace
        sizes = dict(sizes, rows=2000)
        sizes["workspace_bytes"] = lib.fav_selective_scan_workspace_bytes(ct.byref(struct(offsets=FAR, **sizes)))
        assert sizes["workspace_bytes"]
    arrays = {field: FAR * (i + 1) for i, field in enumerate(" ".join(ARRAYS[name]).split())}
    if name == "fav_project_int4":
        arrays["weight"] = sizes["weight"]
        sizes = {k: v for k, v in sizes.items() if k != "weight"}
    for written in ("y", "state_pool", "workspace", "status"):
        for other in arrays:
            if written in arrays and other != written:
                args = struct(**sizes, **{**arrays, written: arrays[other]})
                assert getattr(lib, name)(ct.byref(args), None) == 3, (written, other)


def test_quantising_a_parameter_leaves_its_gradients_behind():
    """Scales that wanted gradients would be refused by every projection."""
    weight = torch.nn.Linear(64, 8).weight
    packed, scales = ops.quantize_int4(weight, 32)
    assert not scales.requires_grad and weight.requires_grad
    assert all(torch.equal(*pair) for pair in zip((packed, scales), ops.quantize_int4(weight.detach(), 32)))


@pytest.mark.parametrize("slots", [0, 2 ** 29 + 1, 2 ** 31, 4.0])
def test_slots_that_codes_cannot_name_are_refused(slots):
    """A code holds a slot's number in 29 bits."""
    with pytest.raises(ValueError, match="slots must be"):
        ops.StreamSlots(slots, device="cpu")
