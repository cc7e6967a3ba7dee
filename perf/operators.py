"""Cases of the stream operators: causal convolution, selective scan, group norm and 4-bit projection.

Sizes are the decoder's own: its channel counts (32 to 2048), up to 512 streams
of one 40 ms frame each, clips of up to 750 frames (30 s at 25 Hz), one clip of
minutes. ``run`` computes an operator in elementary torch operations, or with
``own`` through ``fast_audiovae.ops``.
"""
import math
import os
import sys

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEVICE = "cuda"


def listed():
    return [
        # One speaker's 40 ms step: the smallest call, where only latency counts.
        dict(name="conv 1 stream", op="conv", dtype="bf16", n=1, longest=1, ragged=False, channels=1024, taps=4,
             silu=True),
        # A server's step: one frame of every stream.
        dict(name="conv 512 streams", op="conv", dtype="bf16", n=512, longest=1, ragged=False, channels=2048, taps=4,
             silu=True),
        # Prompts of a batch of new and continued streams, packed without padding.
        dict(name="conv ragged prompts", op="conv", dtype="bf16", n=33, longest=750, ragged=True, channels=2048, taps=4,
             silu=True),
        # The recurrent step of one stream and of a full server.
        dict(name="scan 1 stream", op="scan", dtype="bf16", n=1, longest=1, ragged=False, channels=1024, states=16,
             groups=1, gate=True),
        dict(name="scan 512 streams", op="scan", dtype="bf16", n=512, longest=1, ragged=False, channels=2048, states=16,
             groups=1, gate=True),
        # One prompt of four minutes: few rows, a long axis.
        dict(name="scan one long prompt", op="scan", dtype="bf16", n=1, longest=6000, ragged=False, channels=1024,
             states=16, groups=1, gate=True),
        # A batch of 30 s prompts of unlike length, in full precision, with grouped input and output maps.
        dict(name="scan ragged prompts", op="scan", dtype="fp32", n=32, longest=750, ragged=True, channels=1536,
             states=16, groups=2, gate=True),
        # The norm of one frame of every stream, each frame by itself.
        dict(name="norm 512 frames", op="norm", dtype="bf16", n=512, longest=1, ragged=False, channels=2048, groups=16,
             activation="silu"),
        # Whole clips, statistics over each clip: the batch decoder's 64 clips of 30 s.
        dict(name="norm 64 clips", op="norm", dtype="fp32", n=64, longest=750, ragged=False, channels=512, groups=32,
             activation="snake"),
        # A few clips of unlike length at an odd width.
        dict(name="norm ragged clips", op="norm", dtype="fp16", n=7, longest=333, ragged=True, channels=330, groups=11,
             activation="silu"),
        # The projections of a step: one stream, and a few.
        dict(name="int4 1 stream", op="int4", dtype="bf16", n=1, rows=4096, depth=2048, group=64),
        dict(name="int4 16 streams", op="int4", dtype="fp16", n=16, rows=8192, depth=4096, group=128),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    """A channel count: two of three a multiple of 8, the others any number."""
    value = _spread(rng, low, high)
    return max(low, value // 8 * 8) if rng.random() < 0.67 else value


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm", "int4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "int4":
        return dict(op=op, dtype=dtype, n=_spread(rng, 1, 48), rows=_width(rng, 64, 8192),
                    depth=32 * _spread(rng, 2, 128), group=rng.choice([32, 64, 128]))
    shape = rng.choice(["step", "batch", "ragged", "long"])
    if shape == "step":
        n, longest = _spread(rng, 1, 512), 1
    elif shape == "long":
        n, longest = 1, _spread(rng, 750, 6000)
    else:
        n, longest = _spread(rng, 2, 32 if shape == "ragged" else 16), _spread(rng, 2, 750)
    case = dict(op=op, dtype=dtype, n=n, longest=longest, ragged=shape == "ragged")
    if op == "conv":
        case.update(channels=_width(rng, 32, 2048), taps=rng.randint(2, 8), silu=rng.random() < 0.7)
    elif op == "scan":
        groups = rng.choice([1, 1, 2, 4])
        case.update(channels=groups * _width(rng, 32, 1536 // groups),
                    states=rng.choice([4, 8, 16, 16, 16, rng.randint(1, 64) if n * longest <= 2000 else 16]),
                    groups=groups, gate=rng.random() < 0.7)
    else:
        groups = _spread(rng, 1, 32)
        case.update(channels=groups * max(1, _width(rng, 32, 2048) // groups), groups=groups,
                    activation=rng.choice(["none", "silu", "snake"]))
    return case


def _lengths(case):
    """Sequence lengths: the longest for all, or any from none to the longest (which one of them has)."""
    n, longest = case["n"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    gen = torch.Generator().manual_seed(1000 * n + longest)
    lengths = torch.randint(0, longest + 1, (n,), generator=gen).tolist()
    lengths[0] = longest
    return lengths


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    rand = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(*shape, generator=rand, device=DEVICE) * scale).to(kind)

    f32 = torch.float32
    state = dict(case)
    if case["op"] == "int4":
        n, rows, depth, group = case["n"], case["rows"], case["depth"], case["group"]
        state.update(
            x=normal(n, depth),
            weight=torch.randint(0, 256, (rows, depth // 2), generator=rand, device=DEVICE, dtype=torch.uint8),
            scales=torch.rand(rows, -(-depth // group), generator=rand, device=DEVICE) * 0.02 + 0.001,
            bias=normal(rows, scale=0.1, kind=f32))
        return state
    lengths = _lengths(case)
    n, total, channels = case["n"], sum(lengths), case["channels"]
    offsets = [0]
    for length in lengths:
        offsets.append(offsets[-1] + length)
    state["total"] = total
    state["starts"] = torch.tensor(offsets, dtype=torch.int32, device=DEVICE)
    # What the call is told: offsets of packed sequences, or the shape alone.
    state["offsets"] = state["starts"] if case["ragged"] else None
    shape = (total,) if case["ragged"] or case["longest"] == 1 else (n, case["longest"])
    if case["op"] == "norm":
        state.update(x=normal(*shape, channels) + 0.5, weight=1 + normal(channels, scale=0.1, kind=f32),
                     bias=normal(channels, scale=0.1, kind=f32),
                     alpha=torch.rand(channels, generator=rand, device=DEVICE) + 0.5)
        state["reciprocal"] = 1.0 / (state["alpha"] + 1e-9)
        return state
    # Streams hold slots of a pool in any order; one in four starts afresh.
    slots = torch.randperm(n, generator=gen)
    fresh = torch.randint(0, 4, (n,), generator=gen) == 0
    table = torch.randint(0, 2, (n,), generator=gen)
    state["codes"] = ((slots << 2) | (fresh.long() << 1) | table).to(torch.int32).to(DEVICE)
    if case["op"] == "conv":
        taps = case["taps"]
        state.update(x=normal(*shape, channels), weight=normal(channels, taps, scale=taps ** -0.5, kind=f32),
                     bias=normal(channels, scale=0.1, kind=f32), pool=normal(n, 2, taps - 1, channels))
        return state
    states, groups = case["states"], case["groups"]
    # Steps of a thousandth to a tenth and decays of 1 to the state count, as such models start from.
    step = torch.exp(torch.rand(channels, generator=rand, device=DEVICE) * math.log(100) + math.log(1e-3))
    decay = torch.arange(1, states + 1, device=DEVICE, dtype=f32)[:, None] * torch.exp(
        normal(states, channels, scale=0.1, kind=f32))
    state.update(
        x=normal(*shape, channels), dt=normal(*shape, channels, scale=0.5), a=-decay,
        b=normal(*shape, groups, states), c=normal(*shape, groups, states), d=normal(channels, kind=f32),
        z=normal(*shape, channels) if case["gate"] else None, dt_bias=step + torch.log(-torch.expm1(-step)),
        pool=normal(n, 2, states, channels, scale=0.3, kind=f32))
    return state


def _sequences(s):
    """Per packed row: its sequence and its place in it; per sequence: slot, read table, whether it starts afresh."""
    starts = s["starts"].long()
    rows = torch.arange(s["total"], device=DEVICE)
    seq = torch.searchsorted(starts[1:], rows, right=True)
    codes = s["codes"].long()
    return starts, seq, rows - starts[seq], codes >> 2, codes & 1, (codes & 2) != 0


def _silu(v):
    return v / (1 + torch.exp(-v))


def _plain_conv(s):
    taps, channels, pool = s["taps"], s["channels"], s["pool"]
    starts, seq, place, slot, table, fresh = _sequences(s)
    x = s["x"].reshape(s["total"], channels)
    old = pool[slot, table] * ~fresh[:, None, None]
    # Row p of a sequence's extended input: its history, then its rows. Tap j of row t reads row t + j.
    base = torch.arange(len(slot), device=DEVICE) * (taps - 1)
    extended = torch.cat([old.reshape(-1, channels), x])
    shift = torch.arange(taps, device=DEVICE)
    reach = place[:, None] + shift - (taps - 1)
    index = torch.where(reach >= 0, len(slot) * (taps - 1) + starts[seq][:, None] + reach,
                        base[seq][:, None] + reach + taps - 1)
    y = (extended[index].float() * s["weight"].t()).sum(1) + s["bias"]
    if s["silu"]:
        y = _silu(y)
    last = (starts[1:] - starts[:-1])[:, None] + shift[:-1] - (taps - 1)
    index = torch.where(last >= 0, len(slot) * (taps - 1) + starts[:-1][:, None] + last, base[:, None] + last + taps - 1)
    pool[slot, 1 - table] = extended[index]
    return y.to(x.dtype).reshape(s["x"].shape), pool


def _plain_scan(s):
    total, channels, states, groups, pool = s["total"], s["channels"], s["states"], s["groups"], s["pool"]
    starts, seq, place, slot, table, fresh = _sequences(s)
    x = s["x"].reshape(total, channels).float()
    v = s["dt"].reshape(total, channels).float() + s["dt_bias"]
    delta = torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))
    b = s["b"].reshape(total, groups, states).float().transpose(1, 2).repeat_interleave(channels // groups, 2)
    c = s["c"].reshape(total, groups, states).float().transpose(1, 2).repeat_interleave(channels // groups, 2)
    keep = torch.exp(delta[:, None] * s["a"])
    h = (delta * x)[:, None] * b
    del b
    old = pool[slot, table] * ~fresh[:, None, None]
    first = starts[:-1][starts[1:] > starts[:-1]]
    held = old[starts[1:] > starts[:-1]]
    h[first] += keep[first] * held
    keep[first] = 0
    # h[t] = keep[t] h[t - 1] + h[t], by doubling: every pass joins a row with the one `reach` rows before.
    reach = 1
    while reach < s["longest"]:
        h[reach:] += keep[reach:] * h[:-reach].clone()
        keep[reach:] *= keep[:-reach].clone()
        reach *= 2
    y = (h * c).sum(1) + s["d"] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].reshape(total, channels).float())
    ended = (starts[1:] - 1).clamp(min=0)
    new = torch.where((starts[1:] > starts[:-1])[:, None, None], h[ended], old)
    pool[slot, 1 - table] = new
    return y.to(s["x"].dtype).reshape(s["x"].shape), pool


def _plain_norm(s):
    channels, groups, total = s["channels"], s["groups"], s["total"]
    starts = s["starts"].long()
    x = s["x"].reshape(total, groups, channels // groups).float()
    counts = (starts[1:] - starts[:-1]).clamp(min=1) * (channels // groups)
    seq = torch.searchsorted(starts[1:], torch.arange(total, device=DEVICE), right=True)

    def over_sequences(v):
        if s["ragged"]:
            return torch.zeros(s["n"], groups, device=DEVICE).index_add_(0, seq, v.sum(2)) / counts[:, None]
        return v.sum(2).reshape(s["n"], -1, groups).sum(1) / counts[:, None]

    centred = x - over_sequences(x)[seq][:, :, None]
    spread = over_sequences(centred * centred)
    y = centred * torch.rsqrt(spread + 1e-5)[seq][:, :, None]
    y = y.reshape(total, channels) * s["weight"] + s["bias"]
    if s["activation"] == "silu":
        y = _silu(y)
    elif s["activation"] == "snake":
        wave = torch.sin(s["alpha"] * y)
        y = y + s["reciprocal"] * wave * wave
    return y.to(s["x"].dtype).reshape(s["x"].shape)


def _plain_int4(s):
    packed, rows, depth = s["weight"], s["rows"], s["depth"]
    q = torch.stack([packed & 15, packed >> 4], 2).reshape(rows, depth).float() - 8
    w = q * s["scales"].repeat_interleave(s["group"], 1)[:, :depth]
    return (s["x"].float() @ w.t() + s["bias"]).to(s["x"].dtype)


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fast-audiovae_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from fast_audiovae import ops
    return ops


def run(state):
    s = state
    if not own:
        return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm, "int4": _plain_int4}[s["op"]](s)
    ops = s.get("ops") or s.setdefault("ops", _ops())
    if s["op"] == "conv":
        y = ops.causal_conv(s["x"], s["weight"], s["bias"], activation="silu" if s["silu"] else None,
                            offsets=s["offsets"], state=s["pool"], codes=s["codes"])
        return y, s["pool"]
    if s["op"] == "scan":
        y = ops.selective_scan(s["x"], s["dt"], s["a"], s["b"], s["c"], d=s["d"], z=s["z"], dt_bias=s["dt_bias"],
                               softplus=True, offsets=s["offsets"], state=s["pool"], codes=s["codes"])
        return y, s["pool"]
    if s["op"] == "norm":
        activation, wave = s["activation"], {}
        if activation == "snake":
            wave = dict(alpha=s["alpha"], reciprocal=s["reciprocal"])
        return ops.group_norm(s["x"], s["groups"], s["weight"], s["bias"], eps=1e-5,
                              activation=None if activation == "none" else activation, offsets=s["offsets"], **wave)
    return ops.project_int4(s["x"], s["weight"], s["scales"], s["bias"], group=s["group"])


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    n = case["n"]
    if case["op"] == "int4":
        rows, depth = case["rows"], case["depth"]
        return dict(bytes=rows * depth / 2 + 4 * rows * (-(-depth // case["group"]) + 1) + size * n * (rows + depth),
                    flops=2.0 * n * rows * depth)
    total = sum(_lengths(case))
    values = total * case["channels"]
    if case["op"] == "norm":
        return dict(bytes=2 * values * size + 16 * case["channels"], flops=12.0 * values)
    if case["op"] == "conv":
        # One stream in four starts afresh and has no history to read.
        history = 1.75 * n * (case["taps"] - 1) * case["channels"] * size
        return dict(bytes=2 * values * size + history + 4 * case["channels"] * (case["taps"] + 1),
                    flops=values * (2.0 * case["taps"] + 4))
    states = case["states"]
    return dict(bytes=values * size * (4 if case["gate"] else 3) + 2 * total * case["groups"] * states * size
                + 1.75 * n * states * case["channels"] * 4 + 4 * case["channels"] * (states + 2),
                flops=values * (states * 7.0 + 12))


def exact(case, seed):
    s = prepare(case, seed)
    wide = torch.float64
    if case["op"] == "int4":
        byte = s["weight"].to(torch.int64)
        value = torch.empty(case["rows"], case["depth"], dtype=wide, device=DEVICE)
        value[:, 0::2], value[:, 1::2] = byte % 16 - 8, byte // 16 - 8
        for k in range(0, case["depth"], case["group"]):
            value[:, k:k + case["group"]] *= s["scales"][:, k // case["group"]].to(wide)[:, None]
        return torch.einsum("mk,nk->mn", s["x"].to(wide), value) + s["bias"].to(wide)
    bounds = s["starts"].tolist()
    channels = case["channels"]
    x = s["x"].to(wide).reshape(-1, channels)
    out = torch.zeros_like(x)
    if case["op"] == "norm":
        width = channels // case["groups"]
        for begin, end in zip(bounds, bounds[1:]):
            if begin == end:
                continue
            part = x[begin:end].reshape(end - begin, case["groups"], width)
            spread, mean = torch.var_mean(part, dim=(0, 2), correction=0, keepdim=True)
            y = ((part - mean) / torch.sqrt(spread + 1e-5)).reshape(end - begin, channels)
            y = y * s["weight"].to(wide) + s["bias"].to(wide)
            if case["activation"] == "silu":
                y = y * torch.sigmoid(y)
            elif case["activation"] == "snake":
                y = y + s["reciprocal"].to(wide) * torch.sin(s["alpha"].to(wide) * y) ** 2
            out[begin:end] = y
        return out.reshape(s["x"].shape)
    pool = s["pool"].to(wide)
    codes = s["codes"].tolist()
    held = [torch.zeros_like(pool[0, 0]) if code & 2 else pool[code >> 2, code & 1] for code in codes]
    if case["op"] == "conv":
        taps, w = case["taps"], s["weight"].to(wide)
        for begin, end, code, old in zip(bounds, bounds[1:], codes, held):
            line = torch.cat([old, x[begin:end]])
            y = s["bias"].to(wide) + sum(w[:, j] * line[j:j + end - begin] for j in range(taps))
            out[begin:end] = y * torch.sigmoid(y) if case["silu"] else y
            pool[code >> 2, 1 - (code & 1)] = line[end - begin:]
        return out.reshape(s["x"].shape), pool
    width, groups, states = channels // case["groups"], case["groups"], case["states"]
    v = s["dt"].to(wide).reshape(-1, channels) + s["dt_bias"].to(wide)
    delta = torch.logaddexp(v, torch.zeros_like(v))
    b, c = (s[k].to(wide).reshape(-1, groups, 1, states) for k in "bc")
    a = s["a"].to(wide).t().reshape(groups, width, states)
    # All sequences side by side, one row of each at a time.
    first, last = torch.tensor(bounds[:-1], device=DEVICE), torch.tensor(bounds[1:], device=DEVICE)
    h = torch.stack(held).transpose(1, 2).reshape(-1, groups, width, states).clone()
    for t in range(case["longest"]):
        live = (first + t < last).nonzero()[:, 0] if case["ragged"] else slice(None)
        row = first[live] + t
        step = delta[row].reshape(-1, groups, width, 1)
        now = torch.exp(step * a) * h[live] + step * x[row].reshape(-1, groups, width, 1) * b[row]
        h[live] = now
        out[row] = (now * c[row]).sum(3).reshape(-1, channels)
    out += s["d"].to(wide) * x
    if s["z"] is not None:
        z = s["z"].to(wide).reshape(-1, channels)
        out *= z * torch.sigmoid(z)
    for i, code in enumerate(codes):
        pool[code >> 2, 1 - (code & 1)] = h[i].reshape(channels, states).t()
    return out.reshape(s["x"].shape), pool
