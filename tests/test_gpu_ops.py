"""The stream operators against their plain 64-bit forms, on a B200 (``-m gpu``)."""
import ctypes as ct

import pytest
import torch

from fast_audiovae import _native, build, ops
import ops_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
RAGGED = [0, 5, 5, 6, 40, 40, 137, 139, 201]   # lengths 5, 0, 1, 34, 0, 97, 2, 62


@pytest.fixture(scope="module", autouse=True)
def library():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if not build.LIBRARY.exists():
        build.build()
    assert _native.load_library().fav_device_supported()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def wide(t, pad, shift=0):
    """``t`` [rows, ...] as columns of a wider device buffer: a row stride, and an odd start with ``shift``."""
    flat = t.reshape(t.shape[0], -1)
    buffer = torch.full((t.shape[0], flat.shape[1] + pad), 7.0, dtype=t.dtype, device="cuda")
    part = buffer[:, shift:shift + flat.shape[1]]
    part.copy_(flat)
    return part if t.dim() == 2 else part.unflatten(1, t.shape[1:])


def codes_for(g, n, slots):
    """Codes of n distinct slots in any order, some fresh, either table."""
    slot = torch.randperm(slots, generator=g)[:n]
    bits = torch.randint(0, 4, (n,), generator=g)
    return ((slot << 2) | bits).to(torch.int32)


def layout(kind, n, length):
    """(spans, offsets list or None, rows) of a layout."""
    if kind == "ragged":
        return list(zip(RAGGED[:-1], RAGGED[1:])), RAGGED, RAGGED[-1]
    return [(i * length, (i + 1) * length) for i in range(n)], None, n * length


def close(got, want, tol, what=""):
    got = got.cpu().to(torch.float64)
    excess = (got - want).abs() - tol
    assert not torch.isnan(excess).any(), what
    assert excess.max() <= 0, (what, float(excess.max()), float(((got - want).abs() / tol).max()))


def check_states(pool, before, codes, new, tol, what):
    """The written tables hold ``new``; every other table is untouched."""
    after = pool.cpu()
    expect = before.clone()
    for code, value, t in zip(codes.tolist(), new, tol):
        slot, table = code >> 2, 1 - (code & 1)
        close(after[slot, table], value, t, what)
        expect[slot, table] = after[slot, table]
    assert torch.equal(after, expect), what


def shaped(t, kind, n, length):
    return t.unflatten(0, (n, length)) if kind == "equal" else t


# ------------------------------------------------------------- causal_conv
CONV = [  # layout, n, length, channels, taps, dtype, act, pad, shift
    ("step", 1, 1, 64, 4, BF16, "silu", 0, 0),
    ("step", 5, 1, 1024, 2, F16, None, 8, 0),
    ("step", 3, 1, 33, 8, F32, "silu", 3, 1),
    ("equal", 2, 1, 40, 4, BF16, "silu", 0, 0),
    ("equal", 3, 2, 24, 7, BF16, None, 0, 0),
    ("equal", 1, 700, 96, 4, F32, "silu", 4, 0),
    ("equal", 4, 257, 2048, 4, BF16, "silu", 0, 0),
    ("ragged", 8, 0, 64, 4, BF16, "silu", 0, 0),
    ("ragged", 8, 0, 36, 5, F16, None, 4, 4),
    ("ragged", 8, 0, 1, 3, F32, "silu", 0, 0),
    ("ragged", 8, 0, 513, 8, BF16, "silu", 5, 3),
    ("ragged", 8, 0, 2048, 6, F32, None, 0, 0),
]


@pytest.mark.parametrize("kind,n,length,channels,taps,dtype,act,pad,shift", CONV)
@pytest.mark.parametrize("kept", [True, False])
def test_causal_conv(kind, n, length, channels, taps, dtype, act, pad, shift, kept):
    g = gen(taps * 1000 + channels)
    spans, offsets, rows = layout(kind, n, length)
    x = normal(g, rows, channels, dtype=dtype, scale=2)
    weight, bias = normal(g, channels, taps), normal(g, channels) if taps != 5 else None
    pool = normal(g, n + 2, 2, taps - 1, channels, dtype=dtype)
    codes = codes_for(g, n, n + 2)
    old = ref.states_before(pool, codes.tolist()) if kept else [torch.zeros(taps - 1, channels, dtype=ref.WIDE)] * n
    want, tol, new = ref.causal_conv(x, weight, bias, act, spans, old)
    dev, status = pool.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.causal_conv(shaped(wide(x, pad, shift), kind, n, length), weight.cuda(),
                          None if bias is None else bias.cuda(), activation=act,
                          offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda(),
                          state=dev if kept else None, codes=codes.cuda() if kept else None, status=status)
    close(got.reshape(rows, channels), want, tol)
    assert status.item() == 0
    if kept:
        check_states(dev, pool, codes, new, [torch.zeros_like(h) for h in new], "history")


def test_causal_conv_in_pieces_equals_the_whole():
    """Any split into chunks with a carried history gives the same bits."""
    g = gen(3)
    x = normal(g, 1, 50, 72, dtype=BF16).cuda()
    weight, bias = normal(g, 72, 4).cuda(), normal(g, 72).cuda()
    whole = ops.causal_conv(x, weight, bias, activation="silu")
    slots, pool = ops.StreamSlots(3), ops.conv_state(3, 72, 4)
    parts, at = [], 0
    for size in (1, 2, 1, 5, 3, 37, 1):
        parts.append(ops.causal_conv(x[:, at:at + size], weight, bias, activation="silu", state=pool,
                                     codes=slots.codes([2])))
        slots.commit([2])
        at += size
    assert torch.equal(torch.cat(parts, 1), whole)


# ---------------------------------------------------------- selective_scan
SCAN = [  # layout, n, length, channels, states, groups, dtype, gate, pad, shift
    ("step", 1, 1, 64, 16, 1, BF16, True, 0, 0),
    ("step", 7, 1, 96, 16, 2, F32, True, 4, 0),
    ("step", 3, 1, 33, 5, 3, F16, False, 3, 1),
    ("step", 70, 1, 2048, 4, 1, BF16, True, 0, 0),
    ("step", 2, 1, 8, 128, 1, F32, False, 0, 0),
    ("equal", 2, 1, 40, 16, 1, BF16, True, 0, 0),
    ("equal", 1, 33, 64, 16, 1, F32, True, 0, 0),
    ("equal", 3, 100, 130, 16, 1, BF16, True, 2, 0),
    ("equal", 1, 700, 72, 16, 2, F32, False, 0, 0),
    ("equal", 2, 130, 65, 64, 1, F32, True, 3, 1),
    ("equal", 1, 200, 36, 100, 1, F16, True, 0, 0),
    ("equal", 2, 65, 20, 1, 4, F32, False, 0, 0),
    ("equal", 1, 96, 64, 8, 1, BF16, False, 0, 0),
    ("equal", 1, 90, 48, 24, 1, BF16, True, 0, 0),
    ("ragged", 8, 0, 64, 16, 1, BF16, True, 0, 0),
    ("ragged", 8, 0, 150, 16, 3, F32, True, 6, 4),
    ("ragged", 8, 0, 17, 7, 1, F16, False, 0, 0),
    ("ragged", 8, 0, 1600, 16, 1, F32, True, 0, 0),
    ("ragged", 8, 0, 3, 40, 1, BF16, True, 0, 0),
]


def scan_inputs(g, rows, channels, states, groups, dtype, gate):
    return dict(x=normal(g, rows, channels, dtype=dtype), dt=normal(g, rows, channels, dtype=dtype, scale=1.5),
                a=-torch.rand(states, channels, generator=g) * 8,
                b=normal(g, rows, groups, states, dtype=dtype), c=normal(g, rows, groups, states, dtype=dtype),
                d=normal(g, channels), z=normal(g, rows, channels, dtype=dtype, scale=2) if gate else None,
                dt_bias=normal(g, channels) - 2)


@pytest.mark.parametrize("kind,n,length,channels,states,groups,dtype,gate,pad,shift", SCAN)
@pytest.mark.parametrize("kept", [True, False])
def test_selective_scan(kind, n, length, channels, states, groups, dtype, gate, pad, shift, kept):
    g = gen(states * 1000 + channels)
    spans, offsets, rows = layout(kind, n, length)
    inputs = scan_inputs(g, rows, channels, states, groups, dtype, gate)
    if states % 3 == 1:
        inputs["d"] = None
    if states == 24:
        inputs["dt_bias"] = None
    softplus = states != 8
    if not softplus:
        inputs["dt"], inputs["dt_bias"] = inputs["dt"].abs() / 8, None
    pool = normal(g, n + 1, 2, states, channels)
    codes = codes_for(g, n, n + 1)
    old = ref.states_before(pool, codes.tolist()) if kept else [torch.zeros(states, channels, dtype=ref.WIDE)] * n
    want, tol, new, new_tol = ref.selective_scan(**inputs, softplus=softplus, spans=spans, old=old)
    rowwise = ("x", "dt", "b", "c", "z")
    given = {k: None if v is None else shaped(wide(v, pad, shift), kind, n, length) if k in rowwise else v.cuda()
             for k, v in inputs.items()}
    dev, status = pool.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    got = ops.selective_scan(**given, softplus=softplus,
                             offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda(),
                             state=dev if kept else None, codes=codes.cuda() if kept else None, status=status)
    close(got.reshape(rows, channels), want, tol)
    assert status.item() == 0
    if kept:
        check_states(dev, pool, codes, new, new_tol, "state")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_selective_scan_steps_follow_a_prompt(dtype):
    """A prompt, then single rows from its state, is the scan of all rows."""
    g = gen(11)
    n, prompt, steps, channels, states = 3, 40, 6, 80, 16
    rows = prompt + steps
    inputs = scan_inputs(g, n * rows, channels, states, 1, dtype, True)
    spans = [(i * rows, (i + 1) * rows) for i in range(n)]
    zero = [torch.zeros(states, channels, dtype=ref.WIDE)] * n
    want, tol, _, _ = ref.selective_scan(**inputs, softplus=True, spans=spans, old=zero)
    given = {k: v.cuda().unflatten(0, (n, rows)) if k in ("x", "dt", "b", "c", "z") else v.cuda()
             for k, v in inputs.items()}
    slots, pool = ops.StreamSlots(8), ops.scan_state(8, channels, states)
    pool.fill_(float("nan"))   # a fresh stream reads nothing of its slot
    streams = [5, 0, 3]
    def part(t, rows, flat):
        t = t[:, rows]
        return t[:, 0] if flat else t.contiguous()
    parts = []
    for at in [slice(0, prompt)] + [slice(t, t + 1) for t in range(prompt, rows)]:
        flat = at.stop - at.start == 1
        y = ops.selective_scan(**{k: part(v, at, flat) if k in ("x", "dt", "b", "c", "z") else v
                                  for k, v in given.items()}, state=pool, codes=slots.codes(streams))
        slots.commit(streams)
        parts.append(y.unsqueeze(1) if flat else y)
    close(torch.cat(parts, 1).reshape(n * rows, channels), want, tol)


def test_selective_scan_extremes():
    """Large and vanishing steps: no state survives, or none moves; -inf and large gates close and open."""
    n, channels, states = 4, 32, 16
    one = torch.ones(n, channels)
    dt = torch.stack([one[0] * 1e4, one[0] * -1e4, one[0] * -100, one[0] * 80])
    z = one * torch.tensor([1.0, -float("inf"), 100.0, -200.0])[:, None]
    b = c = torch.ones(n, 1, states)
    pool = torch.ones(n, 2, states, channels)
    codes = (torch.arange(n) << 2).to(torch.int32)
    dev = pool.cuda()
    y = ops.selective_scan(one.cuda(), dt.cuda(), -one[:1].expand(states, -1).contiguous().cuda(), b.cuda(), c.cuda(),
                           z=z.cuda(), state=dev, codes=codes.cuda()).cpu()
    state = dev[:, 1].cpu()
    assert torch.equal(state[0], torch.full_like(state[0], 1e4))
    assert torch.equal(state[1], torch.ones_like(state[1]))
    assert torch.allclose(state[3], torch.full_like(state[3], 80.0), rtol=1e-6, atol=0)
    assert torch.equal(y[1], 0 * y[1]) and torch.isfinite(y).all()
    assert torch.allclose(y[2], torch.full_like(y[2], 1600.0), rtol=1e-5)


# -------------------------------------------------------------- group_norm
NORM = [  # layout, n, length, channels, groups, dtype, act, affine, pad, shift
    ("step", 1, 1, 64, 4, BF16, "silu", True, 0, 0),
    ("step", 9, 1, 2048, 16, F32, "snake", True, 0, 0),
    ("step", 5, 1, 2048, 1, BF16, "silu", True, 8, 0),
    ("step", 5, 1, 66, 22, F16, None, False, 3, 1),
    ("step", 3, 1, 4100, 2, F32, "silu", True, 0, 0),
    ("step", 2, 1, 40000, 1, BF16, None, True, 0, 0),
    ("step", 4, 1, 32, 32, F32, "silu", True, 0, 0),
    ("equal", 2, 1, 40, 4, BF16, "silu", True, 0, 0),
    ("equal", 3, 50, 96, 8, F32, "snake", True, 4, 0),
    ("equal", 1, 1000, 64, 2, BF16, "silu", True, 0, 0),
    ("equal", 2, 333, 330, 11, F16, "silu", True, 0, 0),
    ("equal", 1, 3000, 32, 32, F32, None, False, 0, 0),
    ("equal", 2, 700, 512, 1, F32, "silu", True, 0, 0),
    ("equal", 1, 6000, 200, 8, BF16, "snake", True, 0, 0),
    ("ragged", 8, 0, 64, 4, BF16, "silu", True, 0, 0),
    ("ragged", 8, 0, 35, 7, F32, "snake", True, 3, 2),
    ("ragged", 8, 0, 1024, 32, F16, None, True, 0, 0),
    ("ragged", 8, 0, 1, 1, F32, "silu", False, 0, 0),
]


@pytest.mark.parametrize("kind,n,length,channels,groups,dtype,act,affine,pad,shift", NORM)
@pytest.mark.parametrize("offset", [0.0, 50.0])
def test_group_norm(kind, n, length, channels, groups, dtype, act, affine, pad, shift, offset):
    g = gen(channels + groups)
    spans, offsets, rows = layout(kind, n, length)
    # A mean far from zero, where a difference of squares would lose the variance.
    x = (normal(g, rows, channels) * 1.5 + offset).to(dtype)
    weight, bias = (normal(g, channels) + 1, normal(g, channels)) if affine else (None, None)
    alpha = torch.rand(channels, generator=g) + 0.5 if act == "snake" else None
    recip = 1 / (alpha + 1e-9) if act == "snake" else None
    want, tol = ref.group_norm(x, groups, weight, bias, 1e-5, act, alpha, recip, spans)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    up = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = ops.group_norm(shaped(wide(x, pad, shift), kind, n, length), groups, up(weight), up(bias), activation=act,
                         alpha=up(alpha), reciprocal=up(recip), status=status,
                         offsets=None if offsets is None else torch.tensor(offsets, dtype=torch.int32).cuda())
    close(got.reshape(rows, channels), want, tol)
    assert status.item() == 0


def test_group_norm_of_equal_values():
    """No variance: every value is the bias, and a single value is its own mean."""
    x = torch.full((3, 64), 1000.0, device="cuda")
    bias = torch.arange(64.0, device="cuda")
    assert torch.equal(ops.group_norm(x, 4, None, bias), bias.expand(3, -1))
    assert torch.equal(ops.group_norm(x, 64, None, bias), bias.expand(3, -1))
    assert torch.equal(ops.group_norm(x.unsqueeze(0), 4, None, bias)[0], bias.expand(3, -1))


def test_group_norm_keeps_nonfinite_values_apart():
    """A NaN or an infinity spoils its own sequence and group alone."""
    x = normal(gen(5), 12, 64)
    clean = ops.group_norm(x.view(3, 4, 64).cuda(), 4)
    x[5, 20], x[2, 3] = float("nan"), float("inf")
    got = ops.group_norm(x.view(3, 4, 64).cuda(), 4)
    bad = torch.zeros(3, 4, 64, dtype=torch.bool)
    bad[1, :, 16:32] = True
    bad[0, :, 0:16] = True
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])
    assert torch.isnan(got.cpu()[1, :, 16:32]).all() and not torch.isfinite(got.cpu()[0, 2, 3])


# ------------------------------------------------------------ project_int4
INT4 = [  # rows, out, depth, group, dtype, pad, shift
    (1, 64, 64, 32, BF16, 0, 0), (1, 2048, 4096, 64, BF16, 0, 0), (1, 1000, 2048, 128, F32, 0, 0),
    (2, 17, 96, 64, F16, 0, 0), (3, 1, 32, 32, F32, 0, 0), (7, 333, 160, 128, BF16, 3, 1),
    (8, 512, 1024, 32, F16, 8, 0), (9, 130, 608, 96, F32, 4, 0), (16, 256, 2048, 2048, BF16, 0, 0),
    (33, 100, 512, 128, BF16, 0, 0), (48, 640, 1056, 64, F16, 0, 0), (70, 65, 320, 32, F32, 0, 0),
    (1, 8192, 64, 64, BF16, 0, 0), (5, 48, 8192, 128, BF16, 8, 8),
]


@pytest.mark.parametrize("rows,out,depth,group,dtype,pad,shift", INT4)
def test_project_int4(rows, out, depth, group, dtype, pad, shift):
    g = gen(rows + out)
    x = normal(g, rows, depth, dtype=dtype)
    weight = torch.randint(0, 256, (out, depth // 2), generator=g, dtype=torch.uint8)
    scales = torch.rand(out, -(-depth // group), generator=g) * 0.02
    bias = normal(g, out) if out != 17 else None
    want, tol = ref.project_int4(x, weight, scales, bias, group)
    got = ops.project_int4(wide(x, pad, shift), weight.cuda(), scales.cuda(), None if bias is None else bias.cuda(),
                           group=group)
    close(got, want, tol)


def test_project_int4_passes_nonfinite_values():
    """An infinity or a NaN reaches its own row's outputs and no other row."""
    g = gen(9)
    weight = torch.full((20, 32), 0x99, dtype=torch.uint8)   # every weight is 1
    for dtype in (F32, BF16, F16):
        x = normal(g, 4, 64, dtype=dtype)
        x[1, 5], x[3, 40] = float("inf"), float("nan")
        got = ops.project_int4(x.cuda(), weight.cuda(), torch.ones(20, 2, device="cuda"), group=32).cpu()
        assert torch.isfinite(got[[0, 2]]).all()
        assert (got[1] == float("inf")).all() and torch.isnan(got[3]).all()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantised_projection_is_near_the_full_one(group):
    """A code is off by half a step: scale / 2 a weight, over every input."""
    g = gen(21)
    w, x = normal(g, 200, 320), normal(g, 3, 320)
    packed, scales = ops.quantize_int4(w.cuda(), group)
    got = ops.project_int4(x.cuda(), packed, scales, group=group).cpu().to(ref.WIDE)
    step = scales.cpu().to(ref.WIDE).repeat_interleave(group, 1)[:, :320] / 2
    assert ((got - x.to(ref.WIDE) @ w.to(ref.WIDE).t()).abs() <= x.to(ref.WIDE).abs() @ step.t() * 1.0001).all()


# ------------------------------------------------- rows, slots, status, graphs
def every_operator(x, offsets, status, out, codes=None):
    """Runs the three row operators over packed rows; yields (name, out)."""
    channels, n = x.shape[1], offsets.shape[0] - 1
    one = torch.ones(channels, device="cuda")
    maps = torch.ones(x.shape[0], 1, 4, device="cuda")
    states = dict(state=None, codes=None), dict(state=None, codes=None)
    if codes is not None:
        states = (dict(state=torch.zeros(n, 2, 3, channels, device="cuda"), codes=codes),
                  dict(state=torch.zeros(n, 2, 4, channels, device="cuda"), codes=codes))
    yield "conv", ops.causal_conv(x, torch.ones(channels, 4, device="cuda"), offsets=offsets, status=status,
                                  out=out.clone(), **states[0])
    yield "scan", ops.selective_scan(x, x, -one.expand(4, -1).contiguous(), maps, maps, offsets=offsets,
                                     status=status, out=out.clone(), **states[1])
    if codes is None:
        yield "norm", ops.group_norm(x, 4, offsets=offsets, status=status, out=out.clone())


def test_rows_of_no_sequence_are_left_alone():
    x = normal(gen(1), 90, 64).cuda()
    x[:7] = float("nan")
    x[80:] = float("nan")
    out = torch.full_like(x, 123.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for name, y in every_operator(x, torch.tensor([7, 7, 30, 80], dtype=torch.int32).cuda(), status, out):
        assert (y[:7] == 123).all() and (y[80:] == 123).all(), name
        assert torch.isfinite(y[7:80]).all() and not (y[7:80] == 123).any(), name
    assert status.item() == 0


def test_sequences_without_any_row():
    x = torch.empty(0, 64, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    offsets = torch.zeros(3, dtype=torch.int32, device="cuda")
    codes = torch.tensor([1, 4], dtype=torch.int32, device="cuda")
    for name, y in every_operator(x, offsets, status, x, codes):
        assert y.shape == (0, 64)
    for name, y in every_operator(x, offsets, status, x):
        assert y.shape == (0, 64)
    assert status.item() == 0


@pytest.mark.parametrize("offsets", [[0, 50, 30, 90], [-4, 10, 20, 90], [0, 10, 20, 91], [5, 3, 2, 1],
                                     [2 ** 31 - 1, -2 ** 31, 0, 90]])
def test_bad_offsets_are_reported(offsets):
    x = normal(gen(1), 90, 64).cuda()
    codes = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    for with_codes in (None, codes):
        for i in range(3):
            status = torch.zeros(1, dtype=torch.int32, device="cuda")
            runs = every_operator(x, torch.tensor(offsets, dtype=torch.int32).cuda(), status, torch.zeros_like(x),
                                  with_codes)
            for name, _ in runs:
                assert status.item() == 0x201, name
                status.zero_()


@pytest.mark.parametrize("slot", [-1, 3, 2 ** 28])
def test_bad_slots_are_reported_and_skipped(slot):
    x = normal(gen(1), 90, 64).cuda()
    codes = torch.tensor([0, slot << 2, 8], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full_like(x, 123.0)
    for name, y in every_operator(x, torch.tensor([0, 20, 60, 90], dtype=torch.int32).cuda(), status, out, codes):
        assert status.item() == 0x202, name
        assert (y[20:60] == 123).all() and not (y[:20] == 123).any() and not (y[60:] == 123).any(), name
        status.zero_()
    y = torch.full((3, 64), 123.0, device="cuda")
    one = torch.ones(4, 64, device="cuda")
    ops.selective_scan(x[:3], x[:3], -one, x[:3, :4].unsqueeze(1), x[:3, :4].unsqueeze(1), status=status, out=y,
                       state=torch.zeros(3, 2, 4, 64, device="cuda"), codes=codes)
    assert status.item() == 0x202 and (y[1] == 123).all() and not (y[[0, 2]] == 123).any()


def test_overlapping_outputs_are_refused():
    x = torch.zeros(8, 128, device="cuda")
    w = torch.ones(64, 4, device="cuda")
    with pytest.raises(_native.NativeError) as error:
        ops.causal_conv(x[:, :64], w, out=x[:, 32:96])
    assert error.value.status == 3
    ops.causal_conv(x[:, :64], w, out=x[:, 64:])          # other columns of the same rows
    with pytest.raises(_native.NativeError):
        ops.group_norm(x, 4, out=x)


def test_long_strides_pass_32_bits():
    """Rows that lie over 2^31 elements apart."""
    x = torch.empty((2 << 30) + 64, dtype=BF16, device="cuda").as_strided((3, 64), (1 << 30, 1))
    for i in range(3):
        x[i] = float(i + 1)
    w = torch.tensor([[0.5, 1.0]], device="cuda").expand(64, -1).contiguous()
    y = ops.causal_conv(x, w, offsets=torch.tensor([0, 3], dtype=torch.int32, device="cuda"))
    assert y[:, 0].tolist() == [1.0, 2.5, 4.0]
    y = ops.group_norm(x, 64, None, torch.arange(64.0, device="cuda"))
    assert torch.equal(y[2].float(), torch.arange(64.0, device="cuda"))


class Block:
    """A recurrent block as a latent model has it: project, convolve, scan, normalise, project back."""

    def __init__(self, width, inner, states, dtype, slots):
        g = gen(77)
        self.inner, self.states, self.dtype = inner, states, dtype
        def packed(out, depth):
            return ops.quantize_int4(normal(g, out, depth, scale=depth ** -0.5), 32)
        self.cpu = dict(into=packed(2 * inner, width), maps=packed(inner + 2 * states, inner), back=packed(width, inner),
                        conv=normal(g, inner, 4, scale=0.5), conv_bias=normal(g, inner, scale=0.1),
                        a=-torch.arange(1.0, states + 1)[:, None].expand(-1, inner).contiguous(),
                        d=normal(g, inner), dt_bias=normal(g, inner) - 2, w=normal(g, inner) * 0.1 + 1,
                        b=normal(g, inner) * 0.1)
        self.dev = {k: tuple(t.cuda() for t in v) if isinstance(v, tuple) else v.cuda() for k, v in self.cpu.items()}
        self.slots = ops.StreamSlots(slots)
        self.history = ops.conv_state(slots, inner, 4, dtype=dtype)
        self.state = ops.scan_state(slots, inner, states)

    def __call__(self, x, codes, offsets=None):
        p, inner, states = self.dev, self.inner, self.states
        project = lambda t, key: ops.project_int4(t, *p[key], group=32)  # noqa: E731
        xz = project(x, "into")
        u = ops.causal_conv(xz[:, :inner], p["conv"], p["conv_bias"], activation="silu", offsets=offsets,
                            state=self.history, codes=codes)
        maps = project(u, "maps")
        b, c = maps[:, inner:inner + states].unsqueeze(1), maps[:, inner + states:].unsqueeze(1)
        y = ops.selective_scan(u, maps[:, :inner], p["a"], b, c, d=p["d"], z=xz[:, inner:], dt_bias=p["dt_bias"],
                               offsets=offsets, state=self.state, codes=codes)
        y = ops.group_norm(y, 4, p["w"], p["b"])
        return x + project(y, "back")

    def plain(self, x):
        """One whole sequence in float64."""
        p, inner, states = self.cpu, self.inner, self.states
        project = lambda t, key: ref.project_int4(t, *p[key], None, 32)[0]  # noqa: E731
        x = x.to(ref.WIDE)
        spans = [(0, x.shape[0])]
        xz = project(x, "into")
        u, _, _ = ref.causal_conv(xz[:, :inner], p["conv"], p["conv_bias"], "silu", spans,
                                  [torch.zeros(3, inner, dtype=ref.WIDE)])
        maps = project(u, "maps")
        b, c = maps[:, inner:inner + states].unsqueeze(1), maps[:, inner + states:].unsqueeze(1)
        y, _, _, _ = ref.selective_scan(u, maps[:, :inner], p["a"], b, c, p["d"], xz[:, inner:], p["dt_bias"], True,
                                        spans, [torch.zeros(states, inner, dtype=ref.WIDE)])
        y, _ = ref.group_norm(y, 4, p["w"], p["b"], 1e-5, None, None, None, [(i, i + 1) for i in range(len(x))])
        return x + project(y, "back")


def block_prompt_and_steps(block, x, streams, prompts, graph):
    """Ragged prompts of ``streams``, then single steps to the end of x [n, rows, width]."""
    packed = torch.cat([x[i, :p] for i, p in enumerate(prompts)]).cuda()
    offsets = torch.tensor([0] + prompts).cumsum(0).to(torch.int32).cuda()
    y = block(packed, block.slots.codes(streams), offsets).cpu()
    block.slots.commit(streams)
    outs = [list(part) for part in y.split(prompts)]
    step = [torch.stack([x[i, p + t] for i, p in enumerate(prompts)]).cuda()
            for t in range(x.shape[1] - max(prompts))]
    feed, codes = step[0].clone(), block.slots.codes(streams)
    if graph:   # one captured step, replayed with new rows and codes in its own inputs
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured, stream=side):
            result = block(feed, codes)
        torch.cuda.current_stream().wait_stream(side)
    for rows in step:
        if graph:
            feed.copy_(rows)
            codes.copy_(block.slots.codes(streams))
            captured.replay()
            y = result
        else:
            y = block(rows, block.slots.codes(streams))
            y = block(rows, block.slots.codes(streams))   # a step that was not committed has changed nothing
        block.slots.commit(streams)
        for i, row in enumerate(y.cpu()):
            outs[i].append(row)
    return [torch.stack(rows) for rows in outs]


@pytest.mark.parametrize("graph", [False, True])
def test_recurrent_block(graph):
    """Prompts and steps of a block against its float64 form over whole sequences.

    The block runs in fp32. A relative error of 2e-5 against the largest value
    allows each of its five operators some 60 roundings of its own, carried
    through gains of at most 1.
    """
    block = Block(64, 128, 16, F32, 5)
    x = normal(gen(2), 3, 24, 64)
    prompts = [9, 1, 16]
    got = block_prompt_and_steps(block, x, [4, 0, 2], prompts, graph)
    for i, rows in enumerate(got):
        want = block.plain(x[i, :len(rows)])
        assert (rows.to(ref.WIDE) - want).abs().max() <= 2e-5 * want.abs().max(), i


def test_two_streams_at_once():
    """Calls on two CUDA streams with their own tensors do not disturb one another."""
    g = gen(4)
    inputs = [{k: v.cuda().unflatten(0, (1, 3000)) if k in ("x", "dt", "b", "c", "z") else v.cuda()
               for k, v in scan_inputs(g, 3000, 128, 16, 1, F32, True).items()} for _ in range(2)]
    alone = [ops.selective_scan(**i) for i in inputs]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    both = [[], []]
    for _ in range(4):
        for i in range(2):
            with torch.cuda.stream(side[i]):
                both[i].append(ops.selective_scan(**inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for y in both[i]:
            assert torch.equal(y, alone[i])


def test_both_ways_of_reading_tensors_agree(monkeypatch):
    """Plain tensors read natively, and tensors of another class read from Python: the same bits."""
    class Other(torch.Tensor):
        pass

    g = gen(8)
    x, q = normal(g, 6, 64, dtype=BF16).cuda(), torch.randint(0, 256, (48, 32), generator=g, dtype=torch.uint8).cuda()
    w, b = normal(g, 64, 4).cuda(), normal(g, 64).cuda()
    maps, a = normal(g, 6, 2, 8, dtype=BF16).cuda(), -torch.rand(8, 64, generator=g).cuda()
    codes, offsets = codes_for(g, 6, 6).cuda(), torch.tensor([0, 1, 1, 6], dtype=torch.int32, device="cuda")
    # Long enough to be cut into pieces, with a map whose rows lie further apart.
    long = [normal(g, 1, 2000, 64).cuda(), normal(g, 1, 2000, 64).cuda(), a,
            normal(g, 1, 2000, 3, 8).cuda()[:, :, :2], normal(g, 1, 2000, 2, 8).cuda()]
    def run(kind):
        history, state = torch.ones(6, 2, 3, 64, dtype=BF16, device="cuda"), torch.ones(6, 2, 8, 64, device="cuda")
        first = x.as_subclass(Other) if kind == "subclass" else x
        return [ops.causal_conv(first, w, b, activation="silu", state=history, codes=codes), history,
                ops.causal_conv(first.view(2, 3, 64), w),
                ops.selective_scan(first, x, a, maps, maps, d=b, z=x, dt_bias=b, state=state, codes=codes), state,
                ops.group_norm(first, 8, b, b, activation="snake", alpha=b, reciprocal=b),
                ops.group_norm(first.view(3, 2, 64), 8, b), ops.group_norm(first, 8, offsets=offsets),
                ops.causal_conv(first, w, offsets=offsets),
                ops.selective_scan(first.view(2, 3, 64), x.view(2, 3, 64), a, maps.view(2, 3, 2, 8), maps.view(2, 3, 2, 8)),
                ops.selective_scan(first, x, a, maps, maps, offsets=offsets),
                ops.selective_scan(*(t.as_subclass(Other) if kind == "subclass" and t is long[0] else t for t in long)),
                ops.project_int4(first, q, torch.ones(48, 2, device="cuda"), w[:48, 0].contiguous(), group=32)]
    native = run("plain")
    assert ops._held, "tensors are not read natively here"
    other = run("subclass")
    monkeypatch.setattr(ops, "_held", None)
    python = run("plain")
    for n, o, p in zip(native, other, python):
        assert torch.equal(n, o.as_subclass(torch.Tensor)) and torch.equal(n, p)


def test_refusals_of_device_tensors():
    """What the native reading leaves alone is refused with the reason, and nothing is launched."""
    x, w = torch.zeros(4, 64, device="cuda"), torch.zeros(64, 4, device="cuda")
    q, s = torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.zeros(8, 2, device="cuda")
    maps, a = torch.zeros(4, 1, 8, device="cuda"), torch.zeros(8, 64, device="cuda")
    for call, words in [
            (lambda: ops.causal_conv(x, w.cpu()), "weight must be"), (lambda: ops.causal_conv(x.cpu(), w), "weight must be"),
            (lambda: ops.causal_conv(x.double(), w), "x must be"), (lambda: ops.causal_conv(x[:, ::2], w[:32]), "adjacent"),
            (lambda: ops.causal_conv(x, w.t().contiguous().t()), "weight must be"),
            (lambda: ops.causal_conv(x, w, activation="snake"), "activation"),
            (lambda: ops.causal_conv(x, w, out=torch.zeros(4, 64, device="cuda", dtype=F16)), "out must be"),
            (lambda: ops.causal_conv(x, w, out=torch.zeros(4, 64)), "out must be"),
            (lambda: ops.selective_scan(x, x.half(), a, maps, maps), "dt must be"),
            (lambda: ops.selective_scan(x, x, a, maps, maps.cpu()), "c must be"),
            (lambda: ops.selective_scan(x, x, a[:, :32], maps, maps), "a must be"),
            (lambda: ops.causal_conv(None, w), "x must be"), (lambda: ops.causal_conv(x, None), "weight must"),
            (lambda: ops.selective_scan(x, None, a, maps, maps), "dt must be"),
            (lambda: ops.selective_scan(x, x, None, maps, maps), "a must have"),
            (lambda: ops.selective_scan(x, x, a, None, maps), "b must have"),
            (lambda: ops.selective_scan(x, x, a, maps, None), "c must be"),
            (lambda: ops.group_norm(None, 4), "x must be"), (lambda: ops.project_int4(None, q, s, group=32), "x must be"),
            (lambda: ops.project_int4(x, None, s, group=32), "weight must be"),
            (lambda: ops.project_int4(x, q, None, group=32), "scales are required"),
            (lambda: ops.group_norm(x, 3), "divides"), (lambda: ops.group_norm(x, 4, eps=float("nan")), "eps"),
            (lambda: ops.group_norm(x, 4, w[:, 0]), "weight must be"),
            (lambda: ops.project_int4(x, q, s, group=64), "scales must be"),
            (lambda: ops.project_int4(x, q.char(), s, group=32), "weight must be"),
            (lambda: ops.project_int4(x, q, s, s[:, 0], group=32), "bias must be")]:
        with pytest.raises(ValueError, match=words):
            call()
    grad = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.group_norm(grad, 4)
    with torch.no_grad():
        assert torch.equal(ops.group_norm(grad, 4), x)
    with pytest.raises(_native.NativeError):   # rows that share memory
        ops.causal_conv(x[:1].expand(4, 64), w)


def test_a_parameter_is_a_tensor():
    x = torch.ones(3, 64, device="cuda")
    w = torch.nn.Parameter(torch.ones(64, 2, device="cuda"))
    with torch.inference_mode():
        assert torch.equal(ops.causal_conv(x.view(1, 3, 64), w)[0, :, 0].cpu(), torch.tensor([1.0, 2.0, 2.0]))


def test_calls_follow_the_current_stream():
    """A call on a side stream waits for that stream's earlier work alone."""
    g = gen(12)
    x, w = normal(g, 40, 64).cuda(), normal(g, 64, 4).cuda()
    want = ops.causal_conv(x.view(1, 40, 64) * 2, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            y = ops.causal_conv(x.view(1, 40, 64) * 2, w)
    side.synchronize()
    assert torch.equal(y, want)


def test_captured_graphs_keep_their_own_workspaces():
    """Two captured prompts (split scans and norms, which need workspaces or clusters), replayed in turn."""
    g = gen(13)
    inputs = [{k: v.cuda().unflatten(0, (1, 2000)) if k in ("x", "dt", "b", "c", "z") else v.cuda()
               for k, v in scan_inputs(g, 2000, 64, 16, 1, F32, True).items()} for _ in range(2)]
    def run(i):
        y = ops.selective_scan(**inputs[i])
        return y, ops.group_norm(y, 8, activation="silu")
    want = [run(i) for i in range(2)]
    graphs, got = [], []
    for i in range(2):
        side, captured = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(captured, stream=side):
            got.append(run(i))
        torch.cuda.current_stream().wait_stream(side)
        graphs.append(captured)
    for _ in range(3):
        for captured in graphs:
            captured.replay()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_more_than_two_to_the_31_elements():
    """The last rows of arrays of 2.4e9 elements are those of a short call."""
    rows, channels = 1_200_000, 2048
    x = torch.zeros(rows, channels, dtype=BF16, device="cuda")
    tail = normal(gen(14), 40, channels, dtype=BF16).cuda()
    x[-40:] = tail
    w = normal(gen(15), channels, 4).cuda()
    y = ops.causal_conv(x.unsqueeze(0), w, activation="silu")[0]
    assert torch.equal(y[-36:], ops.causal_conv(tail.unsqueeze(0), w, activation="silu")[0, -36:])
    assert not y[:-40].any()
    y = ops.group_norm(x, 16, activation="silu", out=y)
    assert torch.equal(y[-40:], ops.group_norm(tail, 16, activation="silu"))
    y = ops.group_norm(x, 16, offsets=torch.tensor([rows - 40, rows], dtype=torch.int32, device="cuda"), out=y)
    want, tol = ref.group_norm(tail.cpu(), 16, None, None, 1e-5, None, None, None, [(0, 40)])
    close(y[-40:], want, tol)
    del y
    maps = torch.ones(rows, 1, 4, dtype=BF16, device="cuda")
    a = -torch.ones(4, channels, device="cuda")
    y = ops.selective_scan(x, x, a, maps, maps, offsets=torch.tensor([0, rows - 40, rows], dtype=torch.int32, device="cuda"))
    short = ops.selective_scan(tail, tail, a, maps[:40], maps[:40],
                               offsets=torch.tensor([0, 40], dtype=torch.int32, device="cuda"))
    assert (y[-40:].float() - short.float()).abs().max() <= short.float().abs().max() * 2 ** -7   # pieces end elsewhere


def test_argument_structures_are_the_native_ones():
    """A zero-row call of each operator passes its checks through the C ABI."""
    lib = _native.load_library()
    stream = ct.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.fav_group_norm(ct.byref(_native.NormArgs(channels=8, groups=2, length=1)), stream) == 0
    assert lib.fav_group_norm(ct.byref(_native.NormArgs(channels=8, groups=3, length=1)), stream) == 1
