"""The stream operators at the ends of their range, on a B200 (``-m gpu``): far means, large sizes, extreme values."""
import threading
import time

import pytest
import torch

from fast_audiovae import _native, build, ops
import ops_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module", autouse=True)
def library():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if not build.LIBRARY.exists():
        build.build()
    assert _native.load_library().fav_device_supported()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def close(got, want, tol):
    excess = (got.cpu().to(torch.float64) - want).abs() - tol
    assert not torch.isnan(excess).any()
    assert excess.max() <= 0, float(excess.max())


# -------------------------------------------------------------- group_norm
# Shape, groups, type, and the additions that a value passes through at most: the
# vectors of a thread (two sums each), its warp, the block's warps and the cluster.
# A cluster may have half the 16 CTAs that are asked for.
FAR = [
    ((1, 6000, 2048), 1, F32, 1600),   # 12.3e6 values, 8 or 16 x 512 threads, 4 a vector: 750 or 1500
    ((1, 6000, 2048), 8, BF16, 400),   # 1.5e6 values, 16 or 8 CTAs of 128 threads at least, 8 a vector: 380
    ((2, 750, 512), 1, F32, 100),
    ((1, 3000, 32), 32, F32, 200),     # several groups a block: 8 threads a group
    ((40, 100, 96), 8, F32, 200),
    ((3, 333, 330), 11, F16, 200),
    ((3, 40000), 1, F32, 200),         # single rows
    ((5, 2048), 1, F32, 64),
    ((7, 66), 22, F32, 64),
]


def norm_far_from_zero(x, groups, weight, bias, adds):
    """The norm in float64 and a bound in which the mean enters by the square of a rounding alone.

    A first sum errs by A = adds U of the values' size m, and so does the mean that the differences
    are taken from: e = A m. Their own mean errs by A of the differences' size, spread + e, and so
    does what is left of the mean. The squares err by A of their sum, which holds e^2.
    """
    u, wide = ref.U, x.to(ref.WIDE)
    a = adds * u
    part = wide.reshape(x.shape[0], -1, groups, x.shape[-1] // groups) if x.dim() == 3 else wide.reshape(
        x.shape[0], 1, groups, -1)
    mean = part.mean((1, 3), keepdim=True)
    centred = part - mean
    spread, size = (centred ** 2).mean((1, 3), keepdim=True), centred.abs().mean((1, 3), keepdim=True)
    e = a * mean.abs()
    left = (a + 2 * u) * (size + e)
    spread_off = 3 * a * spread + 2 * left ** 2 + 4 * a * e ** 2
    rstd = 1 / torch.sqrt(spread + 1e-5)
    norm = centred * rstd
    far = rstd * (left + 2 * u * (centred.abs() + e)) + norm.abs() * (spread_off * rstd ** 2 / 2 + 4 * u)
    norm, far, e = ((t + 0 * part).reshape(x.shape) for t in (norm, far, e * rstd))
    w, b = weight.to(ref.WIDE), bias.to(ref.WIDE)
    y = norm * w + b
    return y, far * w.abs() + 4 * u * ((norm * w).abs() + b.abs() + e * w.abs()) + ref.half_step(y, x.dtype)


@pytest.mark.parametrize("shape,groups,dtype,adds", FAR)
@pytest.mark.parametrize("value,spread", [(1000.1, 0.0), (10.1, 0.0), (1000.1, 0.01), (-300.7, 1.0)])
def test_a_mean_far_from_zero_costs_group_norm_no_digits(shape, groups, dtype, adds, value, spread):
    g = gen(sum(shape))
    x = (value + spread * torch.randn(*shape, generator=g)).to(dtype)
    weight, bias = torch.randn(shape[-1], generator=g), torch.randn(shape[-1], generator=g)
    want, tol = norm_far_from_zero(x, groups, weight, bias, adds)
    close(ops.group_norm(x.cuda(), groups, weight.cuda(), bias.cuda()), want, tol)


# Rows that fill a CTA's shared memory to within 15 bytes of what it may ask for.
@pytest.mark.parametrize("shape,groups", [((1, 54576, 48), 16), ((1, 81904, 20), 2), ((1, 6, 20477), 1)])
def test_group_norm_of_rows_that_fill_the_shared_memory(shape, groups):
    x = torch.randn(*shape, generator=gen(shape[1])).to(BF16)
    want, tol = ref.group_norm(x[0], groups, None, None, 1e-5, None, None, None, [(0, shape[1])])
    close(ops.group_norm(x.cuda(), groups)[0], want, tol)


@pytest.mark.parametrize("offsets,code", [([0, 0, 0], 0), ([0, 0, 5], 0x201), ([3, 0], 0x201)])
def test_group_norm_checks_the_offsets_of_no_rows(offsets, code):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.group_norm(torch.empty(0, 64, device="cuda"), 4, offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"),
                   status=status)
    assert status.item() == code


# ---------------------------------------------------------- selective_scan
def test_selective_scan_of_over_two_to_the_30_rows():
    """The last sequences of 20 million of 64 rows are those of a short call."""
    n, length, last = 20_000_000, 64, 3
    g = gen(30)
    x, dt, b, c = (torch.zeros(n, length, *shape, dtype=BF16, device="cuda") for shape in ((1,), (1,), (1, 1), (1, 1)))
    for t in (x, dt, b, c):
        t[-last:] = torch.randn(last, *t.shape[1:], generator=g).to(BF16).cuda()
    a = torch.tensor([[-0.5]], device="cuda")
    y = ops.selective_scan(x, dt, a, b, c, out=torch.full_like(x, 7.0))
    assert torch.equal(y[-last:], ops.selective_scan(*(t[-last:].contiguous() for t in (x, dt)), a,
                                                     *(t[-last:].contiguous() for t in (b, c))))
    assert not y[:-last].any()


@pytest.mark.parametrize("rate,softplus", [(4.0, True), (-4.0, False)])
def test_selective_scan_of_states_that_grow_late(rate, softplus):
    """A state of zero stays zero however much it would grow; what grows at the end of a long prompt is finite.

    Few prompts are cut into pieces of 32 rows, over which a state would grow by e^90, out of fp32's range; the
    ten last rows, the only ones with inputs, let it grow by e^30.
    """
    rows, channels, states = 200, 64, 16
    g = gen(31)
    x, dt = torch.zeros(1, rows, channels), torch.rand(1, rows, channels, generator=g) * 0.1
    x[:, -10:] = torch.randn(10, channels, generator=g)
    a = torch.full((states, channels), rate)
    if not softplus:
        dt = -0.7 - dt
    b, c = torch.randn(1, rows, 1, states, generator=g), torch.randn(1, rows, 1, states, generator=g)
    want, tol, _, _ = ref.selective_scan(x[0], dt[0], a, b[0], c[0], None, None, None, softplus, [(0, rows)],
                                         [torch.zeros(states, channels, dtype=ref.WIDE)])
    close(ops.selective_scan(*(t.cuda() for t in (x, dt, a, b, c)), softplus=softplus)[0], want, tol)


def test_selective_scan_of_states_that_fade():
    """A large state without new inputs fades over a piece of a prompt as it does row by row, and no further."""
    rows, channels, states = 200, 64, 16
    x, maps, dt = torch.zeros(1, rows, channels), torch.ones(1, rows, 1, states), torch.zeros(1, rows, channels)
    dt[:, 32:66] = 3.2     # 2^-148 over the second 32 rows
    a = -torch.ones(states, channels)
    pool = torch.full((1, 2, states, channels), 2.0 ** 120)
    want, tol, new, new_tol = ref.selective_scan(x[0], dt[0], a, maps[0], maps[0], None, None, None, False, [(0, rows)],
                                                 ref.states_before(pool, [0]))
    dev = pool.cuda()
    y = ops.selective_scan(*(t.cuda() for t in (x, dt, a, maps, maps)), softplus=False, state=dev,
                           codes=torch.zeros(1, dtype=torch.int32, device="cuda"))
    close(y[0], want, tol)
    assert (new[0] > 1e-12).all()
    close(dev[0, 1], new[0], new_tol[0])


# ------------------------------------------------------------ project_int4
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,out,depth,group", [(1, 333, 2048, 64), (9, 40, 608, 96), (20, 5000, 512, 128)])
def test_project_int4_of_inputs_near_the_largest(rows, out, depth, group, dtype):
    """Inputs of 10^38, whose sums times whole codes overflow, give their finite outputs; other rows keep their bits."""
    g = gen(rows)
    x = torch.randn(rows, depth, generator=g)
    x[rows // 2] = (torch.rand(depth, generator=g) * 2 - 1) * 1e38
    x = x.to(dtype)
    weight = torch.randint(0, 256, (out, depth // 2), generator=g, dtype=torch.uint8)
    scales = torch.rand(out, -(-depth // group), generator=g) * 0.001
    bias = torch.randn(out, generator=g)
    want, tol = ref.project_int4(x, weight, scales, bias, group)
    assert want.abs().max() < 3e37
    got = ops.project_int4(x.cuda(), weight.cuda(), scales.cuda(), bias.cuda(), group=group)
    close(got, want, tol)
    x[rows // 2] = 0
    other = ops.project_int4(x.cuda(), weight.cuda(), scales.cuda(), bias.cuda(), group=group)
    keep = [i for i in range(rows) if i != rows // 2]
    assert torch.equal(got[keep], other[keep])


@pytest.mark.parametrize("group", [2 ** 31 - 32, 2 ** 31 - 128, 2 ** 30])
def test_project_int4_of_one_large_group(group):
    """A group wider than the depth is one scale a row, however wide."""
    g = gen(40)
    x, weight = torch.randn(3, 96, generator=g).cuda(), torch.randint(0, 256, (70, 48), generator=g, dtype=torch.uint8)
    scales = torch.rand(70, 1, generator=g)
    want, tol = ref.project_int4(x.cpu(), weight, scales, None, 96)
    close(ops.project_int4(x, weight.cuda(), scales.cuda(), group=group), want, tol)


def test_numbers_beyond_32_bits_are_not_cut():
    x = torch.randn(3, 64, device="cuda")
    weight, scales = torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.ones(8, 2, device="cuda")
    with pytest.raises(ValueError, match="divides the channels"):
        ops.group_norm(x, 2 ** 32 + 4)
    with pytest.raises(ValueError, match="scales must be"):
        ops.project_int4(x, weight, scales, group=2 ** 32 + 32)
    for group in (2 ** 31, 2 ** 32 + 32):
        assert torch.equal(ops.project_int4(x, weight, scales[:, 0].unsqueeze(1).contiguous(), group=group),
                           ops.project_int4(x, weight, scales[:, 0].unsqueeze(1).contiguous(), group=128))


def test_forward_derivatives_of_device_tensors_are_refused():
    x, w, state = torch.ones(2, 64, device="cuda"), torch.ones(64, 4, device="cuda"), ops.conv_state(2, 64, 4, dtype=F32)
    want = ops.causal_conv(x, w)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no gradients"):
            ops.causal_conv(torch.autograd.forward_ad.make_dual(x, x), w)
        assert torch.equal(ops.causal_conv(x, w), want)
    with pytest.raises(RuntimeError, match="no gradients"):
        torch.func.jvp(lambda t: ops.causal_conv(t, w), (x,), (x,))
    codes = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.causal_conv(x, w, state=state.requires_grad_(), codes=codes)
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.causal_conv(x, w, out=torch.empty_like(x).requires_grad_())


def test_device_tensors_without_plain_memory_are_refused():
    x, w = torch.ones(6, 64, device="cuda"), torch.ones(64, 4, device="cuda")
    for call in (lambda: ops.causal_conv(x.to_sparse(), w), lambda: ops.causal_conv(x, w.to_sparse()),
                 lambda: ops.causal_conv(x, w, out=x.to_sparse()), lambda: ops.group_norm(x.to_sparse(), 4),
                 lambda: ops.group_norm(x, 4, w[:, 0].to_sparse()),
                 lambda: ops.project_int4(x.to_sparse(), torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), w[:8, :2], group=32)):
        with pytest.raises(ValueError, match="must be"):
            call()


def test_negated_views_of_device_tensors_are_refused():
    """The imaginary part of conjugated numbers: its memory holds the opposite sign. Other strided rows of one run."""
    z = torch.complex(torch.arange(6.0), torch.arange(6.0)).cuda()
    w = torch.tensor([[0.0, 1.0]], device="cuda")
    assert torch.equal(ops.causal_conv(z.imag[:, None], w), z.imag[:, None])
    for call in (lambda: ops.causal_conv(z.conj().imag[:, None], w),
                 lambda: ops.causal_conv(z.imag[:, None], w, z[:1].conj().imag),
                 lambda: ops.causal_conv(z.imag[:, None], w, out=z.conj().imag[:, None])):
        with pytest.raises(ValueError, match="must be"):
            call()


def test_other_threads_run_while_a_call_waits_for_the_queue():
    """Calls into a full queue wait for the device, but not with the interpreter's lock."""
    x, w, out = torch.ones(2, 64, device="cuda"), torch.ones(64, 4, device="cuda"), torch.empty(2, 64, device="cuda")
    ops.causal_conv(x, w, out=out)
    torch.cuda.synchronize()
    done, gaps = threading.Event(), []

    def tick():
        last = time.perf_counter()
        while not done.is_set():
            time.sleep(0.002)
            now = time.perf_counter()
            gaps.append(now - last)
            last = now

    thread = threading.Thread(target=tick)
    thread.start()
    torch.cuda._sleep(1_500_000_000)   # most of a second, and it ends by itself
    begin = time.perf_counter()
    for _ in range(8000):
        ops.causal_conv(x, w, out=out)
    took = time.perf_counter() - begin
    done.set()
    thread.join()
    torch.cuda.synchronize()
    assert took > 0.4, "the queue never filled"
    assert max(gaps) < 0.2, max(gaps)


def test_codes_do_not_wait_for_the_device():
    """Codes of many steps, made while the stream is busy, arrive as they were."""
    slots, streams = ops.StreamSlots(512), list(range(512))
    out = torch.empty(512, dtype=torch.int32, device="cuda")
    slots.codes(streams)
    torch.cuda.synchronize()
    torch.cuda._sleep(1_000_000_000)   # about half a second
    begin, got, want = time.perf_counter(), [], []
    for step in range(40):
        got.append(slots.codes(streams) if step % 2 else slots.codes(streams, out=out).clone())
        want.append([i << 2 | (0 if step else 2) | step % 2 for i in streams])
        slots.commit(streams)
    assert time.perf_counter() - begin < 0.2
    assert torch.equal(torch.stack(got).cpu(), torch.tensor(want, dtype=torch.int32))


def test_codes_are_no_part_of_a_capture():
    slots, x, graph = ops.StreamSlots(4), torch.zeros(2, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="before it"):
            slots.codes([0, 1])
    graph.replay()
    assert x.tolist() == [1.0, 1.0]


def test_a_scan_asks_for_small_workspaces_natively_too():
    """A prompt of one channel and two states needs 36 bytes."""
    ops.group_norm(torch.ones(1, 64, device="cuda"), 4)
    x, maps = torch.ones(1, 65, 1, device="cuda"), torch.ones(1, 65, 1, 2, device="cuda")
    args = x, x, -torch.ones(2, 1, device="cuda"), maps, maps, *[None] * 7
    assert ops._held.fav_selective_scan_tensors(*args, None, torch.empty_like(x), False) > 64


@pytest.mark.parametrize("native", [True, False])
def test_calls_see_what_their_own_stream_wrote(native, monkeypatch):
    """On a busy side stream an input is written late, with other data each time: a call that did not wait for
    that stream would read what was there before (NaN at first), whichever way its tensors are read."""
    g = gen(50)
    if not native:
        monkeypatch.setattr(ops, "_held", None)
    w, a = torch.randn(64, 4, generator=g).cuda(), -torch.rand(4, 64, generator=g).cuda()
    weight, scales = torch.randint(0, 256, (40, 32), generator=g, dtype=torch.uint8).cuda(), torch.ones(40, 2, device="cuda")
    data = torch.randn(5, 400, 64, generator=g).cuda()
    x = torch.empty(400, 64, device="cuda")
    pool, codes = torch.zeros(400, 2, 3, 64, device="cuda"), (torch.arange(400, dtype=torch.int32) << 2).cuda()

    def run():
        maps = x[:, :4].unsqueeze(1)
        return [ops.causal_conv(x, w, state=pool, codes=codes), pool, ops.causal_conv(x[None], w), ops.group_norm(x, 8),
                ops.group_norm(x[None], 8), ops.selective_scan(x, x, a, maps, maps),
                ops.selective_scan(x[None], x[None], a, maps[None], maps[None]),   # cut into pieces, two launches
                ops.project_int4(x, weight, scales, group=32)]

    want = []
    for rows in data:
        x.copy_(rows)
        want.append([t.clone() for t in run()])
    x.fill_(float("nan"))
    torch.cuda.synchronize()
    side, got = torch.cuda.Stream(), []
    with torch.cuda.stream(side):
        for rows in data:
            torch.cuda._sleep(20_000_000)   # ten milliseconds
            x.copy_(rows)
            got.append([t.clone() for t in run()])
            x.fill_(float("nan"))
    side.synchronize()
    for one, other in zip(want, got):
        for t, u in zip(one, other):
            assert torch.equal(t, u)


def test_silu_in_fp32_keeps_its_digits():
    """The same few roundings for any argument, by every operator that has it.

    2^x errs by 2 units in the last place (4 U), the factor that corrects its argument and the product with it
    by one rounding each, the sum by one, 1/x by a unit (2 U) and the product by one: 10 U. Below -87 the hardware
    takes e^-v for infinity or its inverse, under 2^-126, for zero: 100 * 2^-126 is below 2e-36.
    """
    v = torch.cat([torch.linspace(-120, 120, 20_000), torch.linspace(-1, 1, 476),
                   torch.tensor([-float("inf"), -3e38, -1e5, 3e38])]).view(1, -1)
    wide = v.to(ref.WIDE).clamp(min=-500)   # the limit is zero
    want = wide * torch.sigmoid(wide)
    tol = 10 * ref.U * want.abs() * (1 + 1e-6) + 2e-36
    n = v.shape[1]
    one, d = torch.ones(1, n, device="cuda"), v.cuda()
    close(ops.causal_conv(d, torch.tensor([[0.0, 1.0]], device="cuda").expand(n, 2).contiguous(), activation="silu"),
          want, tol)
    close(ops.causal_conv(d[None].expand(1, 1, n).repeat(1, 3, 1), torch.tensor([[0.0, 1.0]], device="cuda").expand(n, 2)
                          .contiguous(), activation="silu")[0, :1], want, tol)   # behind it 0 * inf is no number
    close(ops.group_norm(one, n // 8, None, d[0], activation="silu"), want, tol)
    close(ops.group_norm(one.repeat(1, 3, 1), n // 8, None, d[0], activation="silu")[0, 1:2], want, tol)
    none = torch.zeros(3, 1, 4, device="cuda")
    close(ops.selective_scan(one, one, -torch.ones(4, n, device="cuda"), none[:1], none[:1], d=one[0], z=d), want, tol)
    close(ops.selective_scan(*(one.repeat(1, 3, 1),) * 2, -torch.ones(4, n, device="cuda"), none[None], none[None], d=one[0],
                             z=d.repeat(1, 3, 1))[0, 1:2], want, tol)


def test_outputs_may_lie_between_other_rows():
    """Coefficients in the columns that a strided output leaves free, and in a single row of them."""
    buffer = torch.zeros(8, 256, device="cuda")
    x = torch.randn(8, 64, device="cuda")
    bias = buffer[3, 64:128]
    bias.normal_()
    assert torch.equal(ops.group_norm(x, 4, None, bias, out=buffer[:, :64]), ops.group_norm(x, 4, None, bias.clone()))
    assert torch.equal(ops.group_norm(x, 4, None, bias, out=buffer[:, 192:]), ops.group_norm(x, 4, None, bias.clone()))
    row = buffer[4:5, 64:128]
    assert torch.equal(ops.group_norm(row, 4, out=buffer[4:5, 128:192]), ops.group_norm(row.clone(), 4))
    with pytest.raises(_native.NativeError):
        ops.group_norm(x, 4, None, bias, out=buffer[:, 64:128])


def test_two_threads_call_at_once():
    """Calls give the interpreter's lock back while they launch; each thread's stream and tensors are its own."""
    g = gen(60)
    w, a = torch.randn(64, 4, generator=g).cuda(), -torch.rand(4, 64, generator=g).cuda()
    weight, scales = torch.randint(0, 256, (40, 32), generator=g, dtype=torch.uint8).cuda(), torch.ones(40, 2, device="cuda")

    def run(x):
        maps = x[:, :4].unsqueeze(1)
        return [ops.causal_conv(x, w), ops.group_norm(x[None], 8), ops.selective_scan(x[None], x[None], a, maps[None], maps[None]),
                ops.project_int4(x, weight, scales, group=32)]

    data = torch.randn(2, 300, 64, generator=g).cuda()
    want = [run(x) for x in data]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(100):
                got = run(data[i])
                if not all(torch.equal(t, u) for t, u in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
