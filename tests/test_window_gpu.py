"""Windowed attention (forward, backward, single tokens over a cache) against a 64-bit restatement, on a GPU."""

import ctypes as C
import math

import pytest
import torch

import mcsparse_b200 as mc
from mcsparse_b200 import capi
from mcsparse_b200.capi import lib
from tests import operators_reference as ref

pytestmark = pytest.mark.gpu

# (query lengths, key lengths, window, sinks)
SHAPES = {
    "one token": ([1], [1], 1, 0),
    "self only": ([70], [70], 1, 0),
    "causal": ([300], [300], 1 << 40, 0),
    "window": ([513], [513], 100, 0),
    "first tokens": ([700], [700], 130, 3),
    "many first tokens": ([650], [650], 33, 200),
    "first tokens meet the window": ([400], [400], 129, 128),
    "edges of tiles": ([127, 128, 129, 255, 256, 257], [127, 128, 129, 255, 256, 257], 128, 1),
    "ragged with empty": ([0, 5, 0, 131, 1, 0], [3, 5, 0, 131, 1, 0], 64, 2),
    "cached": ([3, 130, 1], [900, 400, 77], 256, 4),
    "rows that see nothing": ([200, 9], [130, 0], 50, 2),
    "long": ([1500], [1700], 384, 5),
    "long reach of the first": ([2300], [2300], 64, 130),
}
HEADS = [(1, 1, 128), (4, 2, 64), (6, 2, 96), (8, 1, 128), (2, 2, 32), (3, 3, 72), (2, 1, 8)]


def offsets(lengths, device):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=device)


def normal(shape, dtype, device, gen):
    return torch.empty(shape, dtype=dtype, device=device).normal_(generator=gen)


def check(handle, q, k, v, lq, lk, window, sinks, scale=None, dout=None, tail=0):
    """Runs forward (and backward) on given tensors and compares every sequence; `tail` rows belong to no sequence."""
    device, dtype = q.device, q.dtype
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    w = mc.Window(window, sinks, hq, hk, d, dtype, scale=scale)
    qo, ko = offsets(lq, device), offsets(lk, device)
    out = torch.full(q.shape, 7.0, dtype=dtype, device=device)
    lse = torch.full((hq, q.shape[0]), 7.0, device=device)
    mc.window_attention(handle, w, q, k, v, out, lse, q_offsets=qo, k_offsets=ko)
    grads = {}
    if dout is not None:
        grads = {n: torch.full(x.shape, 7.0, dtype=dtype, device=device) for n, x in (("dq", q), ("dk", k), ("dv", v))}
        buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, len(lq), q.shape[0], k.shape[0]), dtype=torch.uint8,
                          device=device).fill_(0xA5)
        mc.window_attention_backward(handle, w, q, k, v, out, lse, dout, grads["dq"], grads["dk"], grads["dv"], buf, q_offsets=qo,
                                     k_offsets=ko)
    q0 = k0 = 0
    for b, (n, m) in enumerate(zip(lq, lk)):
        qs, ks = slice(q0, q0 + n), slice(k0, k0 + m)
        want = ref.attention(q[qs], k[ks], v[ks], min(window, 1 << 40), sinks, w.scale, None if dout is None else dout[qs])
        got = dict(out=out[qs], lse=lse[:, qs], **{name: x[qs if name == "dq" else ks] for name, x in grads.items()})
        for name in want:
            ref.close(got[name], want[name], f"sequence {b}: {name}")
        q0, k0 = q0 + n, k0 + m
    for x, n in [(out, q0), (lse.t(), q0)] + [(x, q0 if name == "dq" else k0) for name, x in grads.items()]:
        assert bool((x[n:] == 7.0).all()), "rows behind the last sequence are left as they were"
    return out, lse, grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_backward(handle, device, dtype, heads, shape):
    lq, lk, window, sinks = SHAPES[shape]
    hq, hk, d = heads
    gen = torch.Generator(device=device).manual_seed(17)
    tq, tk = sum(lq) + 3, sum(lk) + 5
    q, k, v, dout = (normal((n, h, d), dtype, device, gen) for n, h in ((tq, hq), (tk, hk), (tk, hk), (tq, hq)))
    for x, n in ((q, sum(lq)), (dout, sum(lq)), (k, sum(lk)), (v, sum(lk))):
        x[n:] = float("nan")  # rows in no sequence are not looked at
    check(handle, q, k, v, lq, lk, window, sinks, dout=dout)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("layout", ["heads first", "packed", "one key head for all", "odd start", "odd strides"])
def test_strides(handle, device, dtype, layout):
    gen = torch.Generator(device=device).manual_seed(23)
    n, hq, hk, d = 333, 4, 2, 64
    if layout == "heads first":
        q, k, v, g = (normal((h, n, d), dtype, device, gen).transpose(0, 1) for h in (hq, hk, hk, hq))
    elif layout == "packed":
        whole = normal((n, hq + 2 * hk, d), dtype, device, gen)
        q, k, v, g = whole[:, :hq], whole[:, hq:hq + hk], whole[:, hq + hk:], normal((n, hq, d), dtype, device, gen)
    elif layout == "one key head for all":  # broadcast inputs: a head stride of 0; the gradients have rows of their own
        q, g = normal((n, hq, d), dtype, device, gen), normal((1, hq, d), dtype, device, gen).expand(n, hq, d)
        k, v = (normal((n, 1, d), dtype, device, gen).expand(n, hk, d) for _ in range(2))
    elif layout == "odd start":
        q, k, v, g = (normal((n * h * d + 1,), dtype, device, gen)[1:].view(n, h, d) for h in (hq, hk, hk, hq))
    else:
        q, k, v, g = (normal((n, h, d + 3), dtype, device, gen)[..., :d] for h in (hq, hk, hk, hq))
    check(handle, q, k, v, [n], [n], 90, 2, dout=g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
def test_unseen_tokens_may_hold_anything(handle, device, dtype):
    """Keys before the first query's window and behind the first tokens, and the neighbours of a sequence, are NaN or inf."""
    gen = torch.Generator(device=device).manual_seed(29)
    lq, lk, window, sinks, d = [40, 200, 3], [1000, 300, 700], 200, 3, 128
    q, k, v, g = (normal((n, 2, d), dtype, device, gen) for n in (sum(lq), sum(lk), sum(lk), sum(lq)))
    k0 = 0
    for n, m in zip(lq, lk):
        hidden = torch.ones(m, dtype=torch.bool, device=device)
        hidden[:sinks] = False
        hidden[max(0, m - n - window + 1):] = False
        k[k0:k0 + m][hidden] = float("nan")
        v[k0:k0 + m][hidden] = float("inf")
        k0 += m
    out, lse, grads = check(handle, q, k, v, lq, lk, window, sinks, dout=g)
    # a sequence of NaN between two others stays alone
    q[40:240], k[1000:1300], v[1000:1300], g[40:240] = (float("nan"),) * 4
    w = mc.Window(window, sinks, 2, 2, d, dtype)
    qo, ko = offsets(lq, device), offsets(lk, device)
    out2, lse2 = torch.empty_like(out), torch.empty_like(lse)
    mc.window_attention(handle, w, q, k, v, out2, lse2, q_offsets=qo, k_offsets=ko)
    again = {n: torch.empty_like(x) for n, x in grads.items()}
    buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 3, q.shape[0], k.shape[0]), dtype=torch.uint8, device=device)
    mc.window_attention_backward(handle, w, q, k, v, out2, lse2, g, again["dq"], again["dk"], again["dv"], buf, q_offsets=qo, k_offsets=ko)
    rows, keys = torch.ones(len(q), dtype=torch.bool), torch.ones(len(k), dtype=torch.bool)
    rows[40:240], keys[1000:1300] = False, False
    assert torch.equal(out2[rows], out[rows]) and torch.equal(lse2[:, rows], lse[:, rows])
    assert torch.equal(again["dq"][rows], grads["dq"][rows])
    assert torch.equal(again["dk"][keys], grads["dk"][keys]) and torch.equal(again["dv"][keys], grads["dv"][keys])
    assert bool(out2[40:240].isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=lambda t: str(t)[6:])
def test_large_scores(handle, device, dtype):
    """Scores that grow along the sequence, up to several hundred: the running maximum has to follow them."""
    gen = torch.Generator(device=device).manual_seed(31)
    n, d = 600, 64
    q, k, v, g = (normal((n, 2, d), dtype, device, gen) for _ in range(4))
    k[:, 0] *= torch.linspace(0.1, 30, n, device=device)[:, None].to(dtype)
    k[:, 1] *= torch.linspace(30, 0.1, n, device=device)[:, None].to(dtype)
    check(handle, q, k, v, [n], [n], 300, 4, dout=g)
    check(handle, q, k, v, [n], [n], 300, 4, scale=0.0, dout=g)
    check(handle, q, k, v, [n], [n], 300, 4, scale=-0.2, dout=g)


def test_gradients_against_differences(handle, device):
    """Central differences of sum(out * g), in fp32, along random directions of q, k and v."""
    gen = torch.Generator(device=device).manual_seed(37)
    lq, lk, window, sinks = [19, 45], [30, 45], 12, 2
    q, k, v, g = (normal((n, h, 16), torch.float32, device, gen) for n, h in ((64, 4), (75, 2), (75, 2), (64, 4)))
    _, _, grads = check(handle, q, k, v, lq, lk, window, sinks, dout=g)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        direction = normal(x.shape, torch.float32, device, gen)
        step, values = 2.0 ** -6, []
        for sign in (1, -1):
            moved = dict(q=q, k=k, v=v)
            moved[name[1]] = x + sign * step * direction
            out, _, _ = check(handle, moved["q"], moved["k"], moved["v"], lq, lk, window, sinks)
            values.append(float((out.double() * g.double()).sum()))
        slope = (values[0] - values[1]) / (2 * step)
        want = float((grads[name].double() * direction.double()).sum())
        # third-order term: step^2 / 6 times a third derivative; |x| and |direction| are near 1, so it is below
        # step^2 * (number of values) in any case; fp32 rounding: 2^-24 * |out * g| / step
        allowed = step ** 2 * x.numel() ** 0.5 * 4 + 2.0 ** -24 * float((out * g).abs().sum()) / step
        assert abs(slope - want) <= allowed, (name, slope, want, allowed)


def test_gradients_are_repeatable_and_streams_are_kept(device):
    stream = torch.cuda.Stream()
    handle = mc.Handle(stream)
    gen = torch.Generator(device=device).manual_seed(41)
    n, w = 2000, mc.Window(200, 4, 8, 2, 128, torch.bfloat16)
    q, k, v, g = (normal((n, h, 128), torch.bfloat16, device, gen) for h in (8, 2, 2, 8))
    out, lse = torch.empty_like(q), torch.empty(8, n, device=device)
    buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 1, n, n), dtype=torch.uint8, device=device)
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        grads = [torch.empty_like(x) for x in (q, k, v)]
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(2_000_000)
            out.fill_(float("nan"))
        mc.window_attention(handle, w, q, k, v, out, lse)
        mc.window_attention_backward(handle, w, q, k, v, out, lse, g, *grads, buf)
        stream.synchronize()
        results.append([out.clone(), lse.clone()] + grads)
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
    handle.close()


def test_captured_and_replayed(device):
    """A training step captured as a graph, a second one with the same work buffer, replayed in turn with new inputs."""
    stream = torch.cuda.Stream()
    handle = mc.Handle(stream)
    gen = torch.Generator(device=device).manual_seed(43)
    sets = []
    for n, window, heads in ((300, 64, (4, 2, 64)), (777, 200, (2, 1, 128))):
        hq, hk, d = heads
        w = mc.Window(window, 3, hq, hk, d, torch.bfloat16)
        t = [torch.empty(n, h, d, dtype=torch.bfloat16, device=device) for h in (hq, hk, hk, hq)]
        sets.append((w, n, t, torch.empty_like(t[0]), torch.empty(hq, n, device=device), [torch.empty_like(x) for x in t[:3]], window))
    size = max(mc.window_attention_backward_buffer_size(handle, w, 1, n, n) for w, n, *_ in sets)
    buf = torch.empty(size, dtype=torch.uint8, device=device)
    torch.cuda.synchronize()
    graphs = []
    for w, n, t, out, lse, grads, _ in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            mc.window_attention(handle, w, *t[:3], out, lse)
            mc.window_attention_backward(handle, w, *t[:3], out, lse, t[3], *grads, buf)
        graphs.append(graph)
    with torch.cuda.stream(stream):
        for _ in range(2):
            for (w, n, t, out, lse, grads, window), graph in zip(sets, graphs):
                for x in t:
                    x.normal_(generator=gen)
                graph.replay()
                want = ref.attention(*t[:3], window, 3, w.scale, t[3])
                for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
                    ref.close(x, want[name], name)
        stream.synchronize()
    handle.close()


def test_two_calls_at_once(device):
    """Two handles on two streams, each with a buffer of its own."""
    gen = torch.Generator(device=device).manual_seed(47)
    work = []
    for i in range(2):
        stream = torch.cuda.Stream()
        handle = mc.Handle(stream)
        n = 700 + 300 * i
        w = mc.Window(150, 2, 4, 4, 64, torch.float16)
        t = [normal((n, 4, 64), torch.float16, device, gen) for _ in range(4)]
        buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 1, n, n), dtype=torch.uint8, device=device)
        work.append((stream, handle, n, w, t, [torch.empty_like(t[0]) for _ in range(4)], torch.empty(4, n, device=device), buf))
    torch.cuda.synchronize()
    for _ in range(4):
        for stream, handle, n, w, t, o, lse, buf in work:
            mc.window_attention(handle, w, *t[:3], o[0], lse)
            mc.window_attention_backward(handle, w, *t[:3], o[0], lse, t[3], *o[1:], buf)
    torch.cuda.synchronize()
    for stream, handle, n, w, t, o, lse, buf in work:
        want = ref.attention(*t[:3], 150, 2, w.scale, t[3])
        for name, x in zip(("out", "dq", "dk", "dv"), o):
            ref.close(x, want[name], name)
        handle.close()


@pytest.mark.parametrize("sinks", [900, 1024, 1025, 5000])
def test_many_first_tokens_of_a_long_sequence(handle, device, sinks):
    """First tokens on either side of the number whose far queries are cut into pieces, two sequences of different length."""
    gen = torch.Generator(device=device).manual_seed(51)
    lengths = [3300, 1500]
    q, k, v, g = (normal((sum(lengths), h, 64), torch.bfloat16, device, gen) for h in (2, 1, 1, 2))
    check(handle, q, k, v, lengths, lengths, 100, sinks, dout=g)


@pytest.mark.parametrize("dtype,heads", [(torch.bfloat16, (16, 4, 128)), (torch.float16, (18, 6, 64)), (torch.bfloat16, (12, 12, 40))], ids=str)
def test_more_work_than_blocks_run_at_once(handle, device, dtype, heads):
    """Every thread block takes over others' places: long work next to short, sequences without queries or keys, queries that see
    nothing, in changing order; the order in which blocks take over is no part of the result."""
    hq, hk, d = heads
    lengths = [(0, 7), (1, 1), (300, 300), (0, 0), (65, 20), (40, 0), (1400, 1400), (257, 400), (5, 0), (128, 128), (1, 900), (640, 64)]
    lengths = lengths * 2 + lengths[::-1] * 2
    lq, lk = [a for a, _ in lengths], [b for _, b in lengths]
    gen = torch.Generator(device=device).manual_seed(53)
    q, k, v, g = (normal((n, h, d), dtype, device, gen) for n, h in ((sum(lq), hq), (sum(lk), hk), (sum(lk), hk), (sum(lq), hq)))
    first = check(handle, q, k, v, lq, lk, 200, 3, dout=g)
    again = check(handle, q, k, v, lq, lk, 200, 3, dout=g)
    for a, b in zip(first[:2] + tuple(first[2].values()), again[:2] + tuple(again[2].values())):
        assert torch.equal(a, b)


def test_offsets_past_32_bits(handle, device):
    """2.4e9 values per tensor of queries: the last sequence lies behind 2^31 of them."""
    gen = torch.Generator(device=device).manual_seed(54)
    lengths, hq, d, window = [139_800, 300], 136, 128, 40
    total = sum(lengths)
    assert lengths[0] * hq * d > 1 << 31
    q, g = (normal((total, hq, d), torch.bfloat16, device, gen) for _ in range(2))
    k, v = (normal((total, 1, d), torch.bfloat16, device, gen) for _ in range(2))
    w, off = mc.Window(window, 2, hq, 1, d, torch.bfloat16), offsets(lengths, device)
    out, dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    lse = torch.empty(hq, total, device=device)
    mc.window_attention(handle, w, q, k, v, out, lse, q_offsets=off)
    buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 2, total, total), dtype=torch.uint8, device=device)
    mc.window_attention_backward(handle, w, q, k, v, out, lse, g, dq, dk, dv, buf, q_offsets=off)
    last = slice(lengths[0], total)
    want = ref.attention(q[last], k[last], v[last], window, 2, w.scale, g[last])
    for name, x in (("out", out[last]), ("lse", lse[:, last]), ("dq", dq[last]), ("dk", dk[last]), ("dv", dv[last])):
        ref.close(x, want[name], name)


def test_infinite_and_nan_scores_stay_in_their_row(handle, device):
    """A query with an infinite or a NaN value gives a row of NaN, as a softmax does, and no other row notices."""
    gen = torch.Generator(device=device).manual_seed(55)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        q, k, v = (normal((400, 2, 64), dtype, device, gen) for _ in range(3))
        w = mc.Window(90, 2, 2, 2, 64, dtype)
        plain, bad = torch.empty_like(q), torch.empty_like(q)
        mc.window_attention(handle, w, q, k, v, plain)
        q[37, 0, 5], q[200, 1, 9] = float("nan"), float("inf")
        mc.window_attention(handle, w, q, k, v, bad)
        assert bool(bad[37, 0].isnan().all()) and bool(bad[200, 1].isnan().all())
        bad[37, 0], bad[200, 1] = plain[37, 0], plain[200, 1]
        assert torch.equal(bad, plain)


def test_waits_that_run_out_are_reported(device):
    """With a wait limit of one clock every block gives up; the call after the next synchronisation says so, once, and with the
    limit back the same handle computes what it should."""
    handle = mc.Handle()
    gen = torch.Generator(device=device).manual_seed(52)
    n, w = 900, mc.Window(200, 4, 4, 2, 128, torch.bfloat16)
    q, k, v, g = (normal((n, h, 128), torch.bfloat16, device, gen) for h in (4, 2, 2, 4))
    out, lse = torch.empty_like(q), torch.empty(4, n, device=device)
    grads = [torch.empty_like(x) for x in (q, k, v)]
    buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 1, n, n), dtype=torch.uint8, device=device)
    for step in ("forward", "backward"):
        mc.window_attention(handle, w, q, k, v, out, lse)
        torch.cuda.synchronize()
        capi.check(lib.mcsparseB200SetDeviceWaitLimit(handle.h, 1, 0))
        if step == "forward":
            mc.window_attention(handle, w, q, k, v, out, lse)
        else:
            mc.window_attention_backward(handle, w, q, k, v, out, lse, g, *grads, buf)
        torch.cuda.synchronize()
        capi.check(lib.mcsparseB200SetDeviceWaitLimit(handle.h, 40_000_000, 0))
        with pytest.raises(mc.McsparseError) as e:
            mc.window_attention(handle, w, q, k, v, out, lse)
        assert e.value.status == capi.MCSPARSE_STATUS_EXECUTION_FAILED
    mc.window_attention(handle, w, q, k, v, out, lse)
    mc.window_attention_backward(handle, w, q, k, v, out, lse, g, *grads, buf)
    want = ref.attention(q, k, v, 200, 4, w.scale, g)
    for name, x in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        ref.close(x, want[name], name)
    handle.close()


def test_offsets_that_lie_stay_inside(handle, device):
    """Offsets that do not ascend or leave the tensors: rows of no meaning, but nothing outside the outputs is written."""
    gen = torch.Generator(device=device).manual_seed(53)
    n, d = 300, 64
    q, k, v = (normal((n, 2, d), torch.bfloat16, device, gen) for _ in range(3))
    whole = torch.full((n + 400, 2, d), 7.0, dtype=torch.bfloat16, device=device)
    w = mc.Window(64, 2, 2, 2, d, torch.bfloat16)
    for bad in ([0, 250, 100, 5000], [-70, 90, 2 ** 31 - 1, 300], [300, 200, 100, 0]):
        o = torch.tensor(bad, dtype=torch.int32, device=device)
        grads = [torch.empty_like(x) for x in (q, k, v)]
        buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 3, n, n), dtype=torch.uint8, device=device)
        lse = torch.zeros(2, n, device=device)
        mc.window_attention(handle, w, q, k, v, whole[200:200 + n], lse, q_offsets=o, k_offsets=o)
        mc.window_attention_backward(handle, w, q, k, v, whole[200:200 + n], lse, q, *grads, buf, q_offsets=o, k_offsets=o)
        torch.cuda.synchronize()
        assert bool((whole[:200] == 7.0).all()) and bool((whole[200 + n:] == 7.0).all())


# ----------------------------------------------------------------------------- single tokens

def decode_case(device, dtype, lengths, page, hq, hk, d, gen, window, sinks, layout="plain"):
    batch, longest = len(lengths), max(max(lengths), 1)
    per = -(-longest // page) if page else 1
    size = page or longest
    pages = batch * per + 3
    shape = (pages, size, hk, d) if layout != "heads first" else (pages, hk, size, d)
    if layout == "odd":
        k, v = (normal((*shape[:3], d + 1), dtype, device, gen)[..., 1:] for _ in range(2))
    else:
        k, v = (normal(shape, dtype, device, gen) for _ in range(2))
    if layout == "heads first":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    table = None
    if page:
        table = torch.randperm(pages, generator=torch.Generator().manual_seed(3))[:batch * per].view(batch, per).to(torch.int32).to(device)
    return normal((batch, hq, d), dtype, device, gen), k, v, table


def decode_check(handle, q, k, v, table, lengths, window, sinks):
    device, dtype = q.device, q.dtype
    w = mc.Window(window, sinks, q.shape[1], k.shape[2], q.shape[2], dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device=device)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=device)
    per = 1 if table is None else table.shape[1]
    buf = torch.empty(mc.window_attention_decode_buffer_size(handle, w, len(lengths), per, k.shape[1]), dtype=torch.uint8,
                      device=device).fill_(0xA5)
    mc.window_attention_decode(handle, w, q, k, v, n, out, lse, buf, page_table=table)
    room = per * k.shape[1]
    for b, m in enumerate(lengths):
        m = max(0, min(m, room))
        j = torch.arange(m, device=device)
        seen = (j > m - 1 - window) | (j < sinks)
        j = j[seen]
        page = torch.full_like(j, b) if table is None else table[b].long()[j // k.shape[1]]
        fine = (page >= 0) & (page < k.shape[0])
        j, page = j[fine], page[fine]
        at = j % k.shape[1]
        # the seen keys alone, all visible to the one query
        want = ref.attention(q[b:b + 1], k[page, at], v[page, at], 1 << 40, 0, w.scale)
        ref.close(out[b:b + 1], want["out"], f"sequence {b}: out")
        ref.close(lse[b][:, None], want["lse"], f"sequence {b}: lse")
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("heads", HEADS + [(32, 8, 128), (48, 2, 64), (17, 1, 80)], ids=str)
@pytest.mark.parametrize("page", [0, 1, 16, 37, 128])
def test_decode(handle, device, dtype, heads, page):
    gen = torch.Generator(device=device).manual_seed(59)
    for lengths, window, sinks in (([1], 1, 0), ([0, 5, 129], 64, 2), ([700, 1, 333, 0, 2100], 256, 5), ([1500], 1 << 40, 0),
                                   ([900, 131], 70, 130)):
        q, k, v, table = decode_case(device, dtype, lengths, page, *heads, gen, window, sinks)
        decode_check(handle, q, k, v, table, lengths, window, sinks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("layout", ["heads first", "odd"])
def test_decode_strides(handle, device, dtype, layout):
    gen = torch.Generator(device=device).manual_seed(61)
    for page in (0, 16):
        q, k, v, table = decode_case(device, dtype, [600, 44], page, 4, 2, 64, gen, 200, 3, layout)
        decode_check(handle, q, k, v, table, [600, 44], 200, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=lambda t: str(t)[6:])
def test_decode_pages_out_of_use(handle, device, dtype):
    """Page numbers outside the cache are not seen where the window reaches them and not looked at elsewhere; tokens behind
    a length and evicted pages hold NaN."""
    gen = torch.Generator(device=device).manual_seed(67)
    lengths, window, sinks = [1000, 70, 512], 100, 4
    q, k, v, table = decode_case(device, dtype, lengths, 16, 8, 2, 128, gen, window, sinks)
    for b, n in enumerate(lengths):
        for page in range(table.shape[1]):
            first, last = page * 16, page * 16 + 15
            if first >= n or (last <= n - 1 - window and first >= sinks):
                number = int(table[b, page])
                k[number], v[number] = float("nan"), float("inf")
                table[b, page] = [-1, 2 ** 31 - 1, number][page % 3]
            else:
                for at in range(16):
                    j = first + at
                    if j >= n or (j <= n - 1 - window and j >= sinks):
                        k[int(table[b, page]), at], v[int(table[b, page]), at] = float("nan"), float("nan")
    out, _ = decode_check(handle, q, k, v, table, lengths, window, sinks)
    assert bool(out.isfinite().all())
    table[0, 999 // 16], table[1, 0] = -5, k.shape[0]  # in reach, but no page of the cache
    decode_check(handle, q, k, v, table, lengths, window, sinks)
    table.fill_(-1)
    out, lse = decode_check(handle, q, k, v, table, lengths, window, sinks)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    decode_check(handle, q, k, v, table, [5000, -3, 1 << 30], window, sinks)


def test_decode_long_cache(handle, device):
    """A cache whose offsets pass 32 bits: the sequence's pages lie at its end."""
    pages, page = 17000, 128
    k = torch.zeros(pages, page, 8, 128, dtype=torch.bfloat16, device=device)
    v = torch.zeros_like(k)
    assert k.numel() > 1 << 31
    gen = torch.Generator(device=device).manual_seed(71)
    k[-20:].normal_(generator=gen)
    v[-20:].normal_(generator=gen)
    table = torch.arange(pages - 20, pages, dtype=torch.int32, device=device)[None]
    q = normal((1, 16, 128), torch.bfloat16, device, gen)
    decode_check(handle, q, k, v, table, [2500], 2000, 3)


def test_decode_captured(device):
    """A captured step whose lengths move on between replays."""
    stream = torch.cuda.Stream()
    handle = mc.Handle(stream)
    gen = torch.Generator(device=device).manual_seed(73)
    q, k, v, table = decode_case(device, torch.bfloat16, [900, 900], 16, 8, 2, 128, gen, 300, 4)
    w = mc.Window(300, 4, 8, 2, 128, torch.bfloat16)
    n = torch.tensor([5, 600], dtype=torch.int32, device=device)
    out, lse = torch.empty_like(q), torch.empty(2, 8, device=device)
    buf = torch.empty(mc.window_attention_decode_buffer_size(handle, w, 2, table.shape[1], 16), dtype=torch.uint8, device=device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        mc.window_attention_decode(handle, w, q, k, v, n, out, lse, buf, page_table=table)
    with torch.cuda.stream(stream):
        for lengths in ([5, 600], [6, 601], [900, 1], [0, 320]):
            n.copy_(torch.tensor(lengths, dtype=torch.int32))
            graph.replay()
            stream.synchronize()
            got = out.clone(), lse.clone()
            want = decode_check(handle, q, k, v, table, lengths, 300, 4)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    stream.synchronize()
    handle.close()


def test_decode_continues_forward(handle, device):
    """The last row of a forward pass is what the decode call gives on the same keys."""
    gen = torch.Generator(device=device).manual_seed(79)
    n, w = 777, mc.Window(200, 4, 8, 2, 128, torch.bfloat16)
    q, k, v = (normal((n, h, 128), torch.bfloat16, device, gen) for h in (8, 2, 2))
    out = torch.empty_like(q)
    mc.window_attention(handle, w, q, k, v, out)
    one = torch.empty(1, 8, 128, dtype=torch.bfloat16, device=device)
    lengths = torch.tensor([n], dtype=torch.int32, device=device)
    buf = torch.empty(mc.window_attention_decode_buffer_size(handle, w, 1, 1, n), dtype=torch.uint8, device=device)
    mc.window_attention_decode(handle, w, q[-1:], k[None], v[None], lengths, one, buffer=buf)
    want = ref.attention(q[-1:], k, v, 200, 4, w.scale)["out"]
    ref.close(one, want, "decode")
    ref.close(out[-1:], want, "forward")


# ----------------------------------------------------------------------------- together, and refusals

def test_tokens_to_gradients_of_the_table(handle, device):
    """Token ids -> rows of a table -> windowed attention (q = k = v) -> gradients back to the table, as a model chains them."""
    gen = torch.Generator(device=device).manual_seed(83)
    rows, heads, d, lengths = 50, 4, 32, [120, 33]
    n = sum(lengths)
    table = normal((rows, heads * d), torch.float32, device, gen)
    ids = torch.randint(0, rows, (n,), device=device, generator=gen)
    ids[5] = -1
    x = torch.empty(n, heads * d, device=device)
    alpha = 0.5
    mc.embedding_lookup(handle, ids, mc.DnMat(table, rows, heads * d, heads * d), mc.DnMat(x, n, heads * d, heads * d), alpha=alpha)
    w, off = mc.Window(20, 2, heads, heads, d, torch.float32), offsets(lengths, device)
    x3 = x.view(n, heads, d)
    out, lse, g = torch.empty_like(x3), torch.empty(heads, n, device=device), normal((n, heads, d), torch.float32, device, gen)
    mc.window_attention(handle, w, x3, x3, x3, out, lse, q_offsets=off)
    grads = [torch.empty_like(x3) for _ in range(3)]
    buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 2, n, n), dtype=torch.uint8, device=device)
    mc.window_attention_backward(handle, w, x3, x3, x3, out, lse, g, *grads, buf, q_offsets=off)
    total = (grads[0] + grads[1] + grads[2]).view(n, heads * d)
    dtable = torch.empty_like(table)
    m_y, m_e = mc.DnMat(total, n, heads * d, heads * d), mc.DnMat(dtable, rows, heads * d, heads * d)
    ebuf = torch.empty(mc.embedding_gradient_buffer_size(handle, ids, m_y, m_e), dtype=torch.uint8, device=device)
    mc.embedding_gradient(handle, ids, m_y, m_e, ebuf, alpha=alpha)

    t = table.double().requires_grad_()
    e = torch.where((ids >= 0)[:, None], t[ids.clamp(min=0)] * alpha, 0.0).view(n, heads, d)
    loss, at = 0.0, 0
    for m in lengths:
        y = e[at:at + m]
        s = torch.einsum("ihd,jhd->hij", y, y) * w.scale
        s = s.masked_fill(~ref.positions(m, m, 20, 2, device), -torch.inf)
        loss = loss + (torch.einsum("hij,jhd->ihd", torch.softmax(s, -1), y) * g[at:at + m].double()).sum()
        at += m
    loss.backward()
    # fp32 throughout: sums of at most 200 terms of size near 1 and a chain of four products; 2^-24 * 1000 of the scale
    scale = float(t.grad.abs().max())
    assert float((dtable.double() - t.grad).abs().max()) <= 1000 * ref.U32 * scale


def test_refusals(handle, device):
    n, hq, hk, d = 20, 4, 2, 64
    w = mc.Window(8, 1, hq, hk, d, torch.bfloat16)
    q, k = torch.zeros(n, hq, d, dtype=torch.bfloat16, device=device), torch.zeros(n, hk, d, dtype=torch.bfloat16, device=device)
    off = offsets([n], device)
    invalid, refused = capi.MCSPARSE_STATUS_INVALID_VALUE, capi.MCSPARSE_STATUS_NOT_SUPPORTED

    def heads(t, token=None, head=None, p=None):
        return capi.Heads(t.data_ptr() if p is None else p, t.stride(0) if token is None else token, t.stride(1) if head is None else head)

    def forward(h=handle.h, descr=w.d, batch=1, qo=off.data_ptr(), ko=off.data_ptr(), tq=n, tk=n, a=None, b=None, o=None, lse=None):
        a, b, o = a or heads(q), b or heads(k), o or heads(torch.zeros_like(q))
        return lib.mcsparseB200WindowAttention(h, descr, batch, qo, ko, tq, tk, C.byref(a), C.byref(b), C.byref(b), C.byref(o), lse)

    out = torch.zeros_like(q)
    assert forward(o=heads(out)) == 0
    assert forward(h=None) == capi.MCSPARSE_STATUS_NOT_INITIALIZED
    assert forward(descr=None) == invalid
    assert forward(batch=-1) == invalid and forward(tq=-1) == invalid
    assert forward(tk=1 << 31) == refused and forward(batch=1 << 31) == refused
    assert forward(qo=None) == invalid and forward(ko=None) == invalid
    assert forward(qo=None, ko=None, batch=2) == invalid
    assert forward(qo=off.data_ptr() + 2) == invalid
    assert forward(a=heads(q, p=0)) == invalid and forward(b=heads(k, p=k.data_ptr() + 1)) == invalid
    assert forward(a=heads(q, token=-1)) == invalid and forward(b=heads(k, head=1 << 33)) == invalid
    assert forward(o=heads(out, head=d - 1)) == invalid and forward(o=heads(out, token=0)) == invalid
    assert forward(lse=3) == invalid
    size = C.c_size_t()
    assert lib.mcsparseB200WindowAttentionBackward_bufferSize(handle.h, w.d, 1, n, n, None) == invalid
    assert lib.mcsparseB200WindowAttentionBackward_bufferSize(handle.h, None, 1, n, n, C.byref(size)) == invalid
    a, b = C.byref(heads(q)), C.byref(heads(k))
    assert lib.mcsparseB200WindowAttentionBackward(handle.h, w.d, 1, None, None, n, n, a, b, b, a, None, a, a, b, b, 256) == invalid
    assert lib.mcsparseB200WindowAttentionBackward(handle.h, w.d, 1, None, None, n, n, a, b, b, a, 256, a, a, b, b, None) == invalid
    cache = capi.Cache(k.data_ptr(), n * hk * d, hk * d, d)

    def decode(batch=1, lengths=off.data_ptr(), pages=1, size=n, table=None, per=1, buf=256, c=None):
        c = c or cache
        return lib.mcsparseB200WindowAttentionDecode(handle.h, w.d, batch, lengths, a, C.byref(c), C.byref(c), pages, size, table, per,
                                                     C.byref(heads(out)), None, buf)

    assert decode(batch=-1) == invalid and decode(size=0) == invalid and decode(pages=-1) == invalid
    assert decode(per=2) == invalid, "without a table a sequence has one page"
    assert decode(per=1 << 20, size=1 << 20, table=256) == refused
    assert decode(lengths=None) == invalid and decode(buf=None) == invalid and decode(lengths=off.data_ptr() + 1) == invalid
    assert decode(c=capi.Cache(0, 1, 1, 1)) == invalid and decode(c=capi.Cache(k.data_ptr(), -1, 1, 1)) == invalid
    lse = torch.zeros(hq, n, device=device)
    with pytest.raises(ValueError):
        mc.window_attention(handle, w, q.half(), k, k, out)
    with pytest.raises(ValueError):
        mc.window_attention(handle, w, q, q, k, out)
    with pytest.raises(ValueError):
        mc.window_attention(handle, w, q.cpu(), k, k, out)
    with pytest.raises(ValueError):
        mc.window_attention(handle, w, q, k, k, out, lse.t())
    with pytest.raises(ValueError):
        mc.window_attention(handle, w, q, k, k, out, q_offsets=off.long())
    with pytest.raises(ValueError):
        mc.window_attention(handle, w, q, k, k, out, k_offsets=off)
    with pytest.raises(ValueError):
        mc.window_attention_backward(handle, w, q, k, k, out, None, q, q, k, k, torch.empty(1 << 20, dtype=torch.uint8, device=device))


def test_a_short_wait_limit_does_not_count_the_launch_ahead(device):
    """Backward: the keys' launch comes up while the queries' launch still runs on one SM for milliseconds. Its blocks start with
    keys that no query sees, which need no loads; waiting for the launch ahead must not use up the limit of their own waits."""
    handle = mc.Handle()
    d, unseen, long_keys, rows = 64, 148 * 8 * 128, 1 << 20, 128
    n = unseen + long_keys
    w = mc.Window(1 << 40, 0, 1, 1, d, torch.bfloat16)
    gen = torch.Generator(device=device).manual_seed(61)
    q, g = (normal((rows, 1, d), torch.bfloat16, device, gen) for _ in range(2))
    k, v = (normal((n, 1, d), torch.bfloat16, device, gen) for _ in range(2))
    qo = torch.tensor([0, 0, rows], dtype=torch.int32, device=device)
    ko = torch.tensor([0, unseen, n], dtype=torch.int32, device=device)
    out, lse = torch.empty_like(q), torch.empty(1, rows, device=device)
    buf = torch.empty(mc.window_attention_backward_buffer_size(handle, w, 2, rows, n), dtype=torch.uint8, device=device)
    mc.window_attention(handle, w, q, k, v, out, lse, q_offsets=qo, k_offsets=ko)
    results = []
    for limit in (40_000_000, 60_000):  # 64 times that: over a second, and 2 ms
        grads = [torch.full_like(x, 7.0) for x in (q, k, v)]
        torch.cuda.synchronize()
        capi.check(lib.mcsparseB200SetDeviceWaitLimit(handle.h, limit, 0))
        mc.window_attention_backward(handle, w, q, k, v, out, lse, g, *grads, buf, q_offsets=qo, k_offsets=ko)
        torch.cuda.synchronize()
        capi.check(lib.mcsparseB200SetDeviceWaitLimit(handle.h, 40_000_000, 0))
        mc.window_attention(handle, w, q, k, v, out, lse, q_offsets=qo, k_offsets=ko)  # raises if a block gave up
        results.append(grads)
    for name, x, y in zip(("dq", "dk", "dv"), *results):
        assert torch.equal(x, y), name
    for x in results[1][1:]:
        assert not bool(x[:unseen].any()), "keys that no query sees get zeros"
        assert bool(x[unseen:].isfinite().all()) and bool(x[unseen:].any())
    handle.close()


def test_each_kind_of_call_reports_its_own_waits(device):
    """An attention call that gave up is not reported by mcsparseSpMV, nor the other way round; both are reported once."""
    handle = mc.Handle()
    gen = torch.Generator(device=device).manual_seed(67)
    n, w = 300, mc.Window(50, 1, 2, 2, 64, torch.bfloat16)
    q, k, v = (normal((n, 2, 64), torch.bfloat16, device, gen) for _ in range(3))
    out, one = torch.empty_like(q), torch.empty(1, 2, 64, dtype=torch.bfloat16, device=device)
    room = torch.empty(mc.window_attention_decode_buffer_size(handle, w, 1, 1, n), dtype=torch.uint8, device=device)
    length = torch.tensor([n], dtype=torch.int32, device=device)
    rows = 20000  # a diagonal of ones and one below it
    ptr = (2 * torch.arange(rows + 1, device=device)).int()
    col = (torch.arange(2 * rows, device=device) // 2 - (torch.arange(2 * rows, device=device) % 2)).clamp_min(0).int()
    A = mc.CsrMatrix(rows, rows, ptr, col, torch.ones(2 * rows, device=device))
    x, y = mc.DnVec(torch.ones(rows, device=device)), mc.DnVec(torch.zeros(rows, device=device))
    buf = torch.empty(max(mc.spmv_buffer_size(handle, A, x, y), 16), dtype=torch.uint8, device=device)

    def limit(clocks, withhold):
        torch.cuda.synchronize()
        capi.check(lib.mcsparseB200SetDeviceWaitLimit(handle.h, clocks, withhold))

    attention = lambda: mc.window_attention(handle, w, q, k, v, out)
    spmv = lambda: mc.spmv(handle, A, x, y, buf)
    others = lambda: mc.window_attention_decode(handle, w, q[-1:], k[None], v[None], length, one, buffer=room)
    attention(), spmv(), others()
    for fails, clocks, withhold, fine in ((attention, 1, 0, spmv), (spmv, 100_000, 1, attention)):
        limit(clocks, withhold)
        fails()
        limit(40_000_000, 0)
        fine(), others()
        with pytest.raises(mc.McsparseError) as e:
            fails()
        assert e.value.status == capi.MCSPARSE_STATUS_EXECUTION_FAILED
        fails(), fine()
    torch.cuda.synchronize()
    assert bool((y.values == 2).all())
    want = ref.attention(q, k, v, 50, 1, w.scale)
    ref.close(out, want["out"], "out")
    handle.close()


def decode_parts(handle, batch, hq, hk, d, dtype, window, sinks, per, page):
    """Parts of a sequence, by the room that their sums take in the work buffer (0: at most 8, which take none)."""
    size = mc.window_attention_decode_buffer_size(handle, mc.Window(window, sinks, hq, hk, d, dtype), batch, per, page)
    tiles = -(-(hq // hk) // 16)
    return (size - 256) // (batch * hk * tiles * 16 * ((64 if d <= 64 else 128) + 2) * 4)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 40), (torch.float16, 72)], ids=str)
@pytest.mark.parametrize("page", [0, 16, 37])
@pytest.mark.parametrize("heads,lengths,window,sinks,parts", [
    ((16, 16), [8192], 1 << 40, 0, 16),             # the fewest visible keys that take the work buffer
    ((32, 8), [9001, 0, 3, 700, 8193], 8500, 5, 8),  # (five sequences: a cluster each)
    ((32, 8), [9001], 8500, 5, 32),
    ((18, 1), [30011, 1], 20000, 130, 64),          # two tiles of query heads
    ((4, 1), [65536], 1 << 40, 0, 64),
], ids=str)
def test_decode_over_many_parts(handle, device, dtype, d, page, heads, lengths, window, sinks, parts):
    """Long visible caches: the parts of a sequence are joined through the work buffer. What no query sees is NaN."""
    gen = torch.Generator(device=device).manual_seed(71)
    q, k, v, table = decode_case(device, dtype, lengths, page, *heads, d, gen, window, sinks)
    per = 1 if table is None else table.shape[1]
    got = decode_parts(handle, len(lengths), *heads, d, dtype, window, sinks, per, k.shape[1])
    assert (got if parts > 8 else max(got, 8)) == parts
    seen = torch.zeros(k.shape[:2], dtype=torch.bool, device=device)
    for b, n in enumerate(lengths):
        j = torch.arange(n, device=device)
        j = j[(j > n - 1 - window) | (j < sinks)]
        seen[torch.full_like(j, b) if table is None else table[b].long()[j // k.shape[1]], j % k.shape[1]] = True
    k[~seen] = float("nan")
    v[~seen] = float("inf")
    out, lse = decode_check(handle, q, k, v, table, lengths, window, sinks)
    again = decode_check(handle, q, k, v, table, lengths, window, sinks)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1]), "equal inputs, equal bits"
    if page:  # pages outside the cache are not seen, whichever part they fall to
        table[0, ::3] = -1
        table[0, 1::9] = k.shape[0]
        decode_check(handle, q, k, v, table, lengths, window, sinks)
