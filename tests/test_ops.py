"""Stream operators without a GPU: refusals, argument structures, slots, 4-bit codes."""
import ctypes as ct
import re
import subprocess
from pathlib import Path

import pytest
import torch

from fast_audiovae import _native, build, ops

INCLUDE = Path(__file__).resolve().parent.parent / "include"
STRUCTS = {"fav_conv_args": _native.ConvArgs, "fav_scan_args": _native.ScanArgs, "fav_norm_args": _native.NormArgs,
           "fav_int4_args": _native.Int4Args}


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _native.load_library()


def test_argument_structures_match_the_header(tmp_path):
    """Sizes and offsets of every field, from a C compiler."""
    lines = []
    for name, struct in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in struct._fields_]
    source = tmp_path / "layout.c"
    source.write_text('#include <stdio.h>\n#include "fast_audiovae_cuda.h"\nint main(void) {%s return 0; }\n'
                      % "\n".join(lines))
    subprocess.run(["gcc", "-I", str(INCLUDE), str(source), "-o", str(tmp_path / "layout")], check=True)
    said = dict(line.split() for line in
                subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.splitlines())
    for name, struct in STRUCTS.items():
        assert int(said[name]) == ct.sizeof(struct)
        for field, _ in struct._fields_:
            assert int(said[f"{name}.{field}"]) == getattr(struct, field).offset, (name, field)
    text = (INCLUDE / "fast_audiovae_cuda.h").read_text()
    for name, struct in STRUCTS.items():
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        fields = [f.strip(" *") for line in body.split(";") for f in line.replace("const", "").strip().partition(" ")[2].split(",")]
        assert [f for f in fields if f] == [f for f, _ in struct._fields_]


# A call the library would accept, up to the launch; every change below is refused before it.
BASE = {
    "fav_causal_conv": (_native.ConvArgs, dict(x=4096, y=1 << 20, x_stride=8, y_stride=8, weight=4096, type=0,
                                               channels=8, taps=4, n=2, length=3, rows=6)),
    "fav_selective_scan": (_native.ScanArgs, dict(x=4096, dt=4096, b=4096, c=4096, y=1 << 20, x_stride=8, dt_stride=8,
                                                  b_stride=4, c_stride=4, y_stride=8, a=4096, channels=8, states=4,
                                                  groups=1, n=2, length=3, rows=6)),
    "fav_group_norm": (_native.NormArgs, dict(x=4096, y=1 << 20, x_stride=8, y_stride=8, channels=8, groups=2, n=2,
                                              length=3, rows=6, eps=1e-5)),
    "fav_project_int4": (_native.Int4Args, dict(x=4096, y=1 << 20, x_stride=64, y_stride=8, weight=4096, scales=4096,
                                                rows=2, depth=64, out=8, group=32)),
}
REFUSED = [
    ("fav_causal_conv", 1, dict(channels=0)), ("fav_causal_conv", 1, dict(taps=1)), ("fav_causal_conv", 1, dict(taps=9)),
    ("fav_causal_conv", 2, dict(type=3)), ("fav_causal_conv", 2, dict(activation=2)), ("fav_causal_conv", 1, dict(rows=5)),
    ("fav_causal_conv", 1, dict(length=0, rows=0)), ("fav_causal_conv", 1, dict(x=0)), ("fav_causal_conv", 1, dict(weight=0)),
    ("fav_causal_conv", 1, dict(x_stride=7)), ("fav_causal_conv", 1, dict(y_stride=1 << 31)),
    ("fav_causal_conv", 1, dict(state_pool=1 << 22)), ("fav_causal_conv", 1, dict(slot_codes=4096)),
    ("fav_causal_conv", 1, dict(state_pool=1 << 22, slot_codes=4096, num_slots=1)),
    ("fav_causal_conv", 3, dict(y=4096)), ("fav_causal_conv", 3, dict(y=4096 + 4)),
    ("fav_causal_conv", 3, dict(state_pool=4096, slot_codes=4096, num_slots=2)),
    ("fav_causal_conv", 1, dict(n=1 << 20, length=1 << 20, rows=0)), ("fav_causal_conv", 1, dict(n=-1)),
    ("fav_selective_scan", 1, dict(states=0)), ("fav_selective_scan", 1, dict(states=129)),
    ("fav_selective_scan", 1, dict(groups=3)), ("fav_selective_scan", 1, dict(groups=0)),
    ("fav_selective_scan", 1, dict(a=0)), ("fav_selective_scan", 1, dict(dt=0)), ("fav_selective_scan", 3, dict(y=4096)),
    ("fav_selective_scan", 1, dict(groups=2, b_group_stride=1)), ("fav_selective_scan", 1, dict(z=4096, z_stride=4)),
    ("fav_selective_scan", 1, dict(b_stride=0)), ("fav_selective_scan", 2, dict(type=-1)),
    ("fav_selective_scan", 1, dict(n=1, length=1 << 16, rows=1 << 16, y=1 << 30)),   # pieces without a workspace
    ("fav_group_norm", 1, dict(groups=3)), ("fav_group_norm", 1, dict(eps=-1.0)), ("fav_group_norm", 1, dict(eps=float("nan"))),
    ("fav_group_norm", 1, dict(activation=2)), ("fav_group_norm", 2, dict(activation=3)), ("fav_group_norm", 3, dict(y=4096)),
    ("fav_project_int4", 1, dict(depth=48)), ("fav_project_int4", 1, dict(group=16)), ("fav_project_int4", 1, dict(group=48)),
    ("fav_project_int4", 1, dict(out=0)), ("fav_project_int4", 1, dict(weight=4100)), ("fav_project_int4", 1, dict(scales=0)),
    ("fav_project_int4", 1, dict(x_stride=63)), ("fav_project_int4", 3, dict(y=4096)),
]


@pytest.mark.parametrize("name,status,change", REFUSED)
def test_the_c_abi_refuses(lib, name, status, change):
    struct, good = BASE[name]
    assert getattr(lib, name)(ct.byref(struct(**{**good, **change})), None) == status
    assert lib.fav_last_error()


def test_the_c_abi_refuses_null(lib):
    for name in BASE:
        assert getattr(lib, name)(None, None) == 1
    assert lib.fav_selective_scan_workspace_bytes(None) == 0


def test_binding_tensors_needs_an_exchange(lib):
    assert lib.fav_bind_tensors(None, None) == 1
    assert lib.fav_bind_tensors(ct.byref((ct.c_uint32 * 32)(2)), id(None)) == 2   # DLPack 2 is not known


def test_scan_workspace_grows_only_for_few_long_sequences(lib):
    def need(n, length, channels):
        return lib.fav_selective_scan_workspace_bytes(ct.byref(_native.ScanArgs(
            channels=channels, states=16, groups=1, n=n, length=length, rows=n * length)))
    assert need(512, 1, 2048) == 0 and need(64, 750, 2048) == 0 and need(1, 20, 64) == 0
    pieces = need(1, 6000, 1024) / (1024 * 17 * 4)
    assert pieces == int(pieces) and 2 <= pieces <= 6000 / 32 + 1


X, W = torch.zeros(6, 8), torch.zeros(8, 4)
MAPS = torch.zeros(6, 1, 4)
A = torch.zeros(4, 8)
I32 = dict(dtype=torch.int32)
Q, S = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2)
H = torch.zeros(6, 2, 3, 8)


@pytest.mark.parametrize("call,words", [
    (lambda: ops.causal_conv(X.double(), W), "x must be"),
    (lambda: ops.causal_conv([1.0], W), "x must be"),
    (lambda: ops.causal_conv(torch.zeros(8), W), "x must have shape"),
    (lambda: ops.causal_conv(torch.zeros(2, 0, 8), W), "at least one row"),
    (lambda: ops.causal_conv(X.t(), torch.zeros(6, 4)), "adjacent channels"),
    (lambda: ops.causal_conv(torch.zeros(4, 3, 8)[:, :2], W), "one stride"),
    (lambda: ops.causal_conv(X, torch.zeros(8, 9)), "2 to 8 taps"),
    (lambda: ops.causal_conv(X, torch.zeros(7, 4)), "weight must be"),
    (lambda: ops.causal_conv(X, W.half()), "weight must be"),
    (lambda: ops.causal_conv(X, W, torch.zeros(7)), "bias must be"),
    (lambda: ops.causal_conv(X, W, activation="snake"), "activation"),
    (lambda: ops.causal_conv(X, W, offsets=torch.zeros(3, dtype=torch.int64)), "offsets must be"),
    (lambda: ops.causal_conv(X, W, offsets=torch.zeros(0, **I32)), "n \\+ 1"),
    (lambda: ops.causal_conv(X.view(2, 3, 8), W, offsets=torch.zeros(3, **I32)), "Packed sequences"),
    (lambda: ops.causal_conv(X, W, state=H), "go together"),
    (lambda: ops.causal_conv(X, W, codes=torch.zeros(6, **I32)), "go together"),
    (lambda: ops.causal_conv(X, W, state=H, codes=torch.zeros(5, **I32)), "codes must be"),
    (lambda: ops.causal_conv(X, W, state=H[:5], codes=torch.zeros(6, **I32)), "as many slots"),
    (lambda: ops.causal_conv(X, W, state=H.half(), codes=torch.zeros(6, **I32)), "state must be"),
    (lambda: ops.causal_conv(X, W, state=H[:, :, :2], codes=torch.zeros(6, **I32)), "state must be"),
    (lambda: ops.causal_conv(X, W, status=torch.zeros(2, **I32)), "status must be"),
    (lambda: ops.selective_scan(X, X, torch.zeros(129, 8), MAPS, MAPS), "1 to 128 states"),
    (lambda: ops.selective_scan(X, X[:5], A, MAPS, MAPS), "dt must be"),
    (lambda: ops.selective_scan(X, X, A, torch.zeros(6, 3, 4), MAPS), "groups that divide"),
    (lambda: ops.selective_scan(X, X, A, MAPS[:, 0], MAPS), "groups that divide"),
    (lambda: ops.selective_scan(X, X, A, MAPS, torch.zeros(6, 2, 4)), "c must be"),
    (lambda: ops.selective_scan(X, X, A, torch.zeros(6, 1, 5), MAPS), "b must be"),
    (lambda: ops.selective_scan(X, X, A, torch.zeros(6, 1, 8)[:, :, ::2], MAPS), "adjacent states"),
    (lambda: ops.selective_scan(X, X, A, MAPS, MAPS, z=X.half()), "z must be"),
    (lambda: ops.selective_scan(X, X, A, MAPS, MAPS, d=torch.zeros(4)), "d must be"),
    (lambda: ops.group_norm(X, 3), "divides the channels"),
    (lambda: ops.group_norm(X, 0), "divides the channels"),
    (lambda: ops.group_norm(X, 2, eps=-1.0), "eps"),
    (lambda: ops.group_norm(X, 2, activation="relu"), "activation must"),
    (lambda: ops.group_norm(X, 2, activation="snake"), "alpha and reciprocal"),
    (lambda: ops.group_norm(X, 2, alpha=torch.ones(8)), "alpha and reciprocal"),
    (lambda: ops.project_int4(torch.zeros(2, 64), Q, S, group=48), "multiples of 32"),
    (lambda: ops.project_int4(torch.zeros(2, 48), Q, S, group=32), "multiples of 32"),
    (lambda: ops.project_int4(torch.zeros(2, 96), Q, S, group=32), "weight must be"),
    (lambda: ops.project_int4(torch.zeros(2, 64), Q.view(16, 16).t(), S, group=32), "weight must be"),
    (lambda: ops.project_int4(torch.zeros(2, 64), Q, S[:, :1], group=32), "scales must be"),
    (lambda: ops.project_int4(torch.zeros(2, 64), Q, None, group=32), "scales are required"),
    (lambda: ops.project_int4(torch.zeros(2, 2, 64), Q, S, group=32), "x must have shape"),
    (lambda: ops.quantize_int4(torch.full((2, 32), float("inf")), 32), "finite"),
    (lambda: ops.quantize_int4(torch.zeros(2, 40), 32), "multiples of 32"),
])
def test_arguments_are_checked_before_the_device(call, words):
    with pytest.raises(ValueError, match=words):
        call()


@pytest.mark.parametrize("call", [
    lambda: ops.causal_conv(X, W), lambda: ops.selective_scan(X, X, A, MAPS, MAPS), lambda: ops.group_norm(X, 2),
    lambda: ops.project_int4(torch.zeros(2, 64), Q, S, group=32)])
def test_there_is_no_cpu_path(call):
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()


def test_gradients_are_refused():
    x = X.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.causal_conv(x, W)
    with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
        ops.causal_conv(x, W)


def test_slots_advance_only_when_committed():
    slots = ops.StreamSlots(4, device="cpu")
    assert slots.codes([2, 0]).tolist() == [2 << 2 | 2, 0 << 2 | 2]
    assert slots.codes([2]).tolist() == [2 << 2 | 2]
    slots.commit([2])
    assert slots.codes([0, 2]).tolist() == [2, 2 << 2 | 1]
    slots.commit([2])
    assert slots.codes([2]).tolist() == [2 << 2]
    slots.reset([2])
    assert slots.codes([2]).tolist() == [2 << 2 | 2]
    assert slots.codes([]).shape == (0,)
    for bad in ([4], [-1], [1, 1], [[0, 1]], [0.5]):
        with pytest.raises(ValueError):
            slots.codes(bad)


def test_states_have_two_tables():
    assert ops.conv_state(3, 8, 4, device="cpu").shape == (3, 2, 3, 8)
    assert ops.scan_state(3, 8, 16, device="cpu").dtype == torch.float32


@pytest.mark.parametrize("out,depth,group", [(5, 64, 32), (3, 96, 64), (1, 32, 128)])
def test_quantised_codes_are_the_nearest(out, depth, group):
    w = torch.randn(out, depth, generator=torch.Generator().manual_seed(depth))
    w[0, :32] = 0
    packed, scales = ops.quantize_int4(w, group)
    assert packed.shape == (out, depth // 2) and scales.shape == (out, -(-depth // group))
    q = torch.stack([packed & 15, packed >> 4], 2).view(out, depth).double() - 8
    step = scales.double().repeat_interleave(group, 1)[:, :depth]
    assert ((q * step - w.double()).abs() <= step / 2 * (1 + 1e-6)).all() and q.abs().max() <= 7
