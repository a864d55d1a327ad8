"""mcsparseB200EmbeddingLookup / EmbeddingGradient against a 64-bit restatement, on a GPU."""

import ctypes as C

import pytest
import torch

import mcsparse_b200 as mc
from mcsparse_b200 import capi
from mcsparse_b200.capi import lib
from tests import operators_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
         (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]


def mat(t):
    return mc.DnMat(t, t.shape[0], t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1])


def ids_for(count, rows, kind, device, seed=1, index=torch.int64, base=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":  # one token fills the batch
        ids = torch.full((count,), rows // 2)
    elif kind == "each":  # no token twice
        ids = torch.randperm(max(rows, count), generator=g)[:count] % rows
    elif kind == "outside":  # half of them padding, on both sides of the table
        ids = torch.randint(-rows, 2 * rows, (count,), generator=g)
    elif kind == "edges":
        ids = torch.randint(0, 2, (count,), generator=g) * (rows - 1)
    else:
        ids = (torch.rand(count, generator=g) ** 4 * rows).long()
    return (ids + base).to(index).to(device)


def strided(rows, cols, dtype, device, pad, offset, gen):
    """A rows x cols view with a leading dimension of cols + pad, starting `offset` elements into its storage."""
    whole = torch.empty(offset + rows * (cols + pad) + 16, dtype=dtype, device=device).normal_(generator=gen)
    return whole, whole[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
@pytest.mark.parametrize("width,pad,offset", [(1, 0, 0), (64, 0, 0), (1000, 24, 8), (777, 2, 0), (4096, 0, 0), (256, 1, 1)])
@pytest.mark.parametrize("count", [1, 65])
def test_lookup(handle, device, types, width, pad, offset, count):
    te, ty = types
    gen = torch.Generator(device=device).manual_seed(7)
    rows, base = 37, count % 2
    _, table = strided(rows, width, te, device, pad, offset, gen)
    whole, out = strided(count, width, ty, device, pad, offset, gen)
    before = whole.clone()
    ids = ids_for(count, rows, "outside", device, index=torch.int32 if width % 2 else torch.int64, base=base)
    mc.embedding_lookup(handle, ids, mat(table), mc.DnMat(out, count, width, width + pad), alpha=1.7, base=base)
    i = ids.long() - base
    ok = (i >= 0) & (i < rows)
    # alpha reaches the kernel as an fp32 number
    want = torch.where(ok[:, None], table.double()[i.clamp(0, rows - 1)] * float(torch.tensor(1.7)), 0.0)
    ref.close(out, (want, (ref.U[ty] + 2 * ref.U32) * want.abs() + ref.TINY[ty]), "lookup")
    after = whole.clone()
    inside = torch.zeros_like(whole, dtype=torch.bool)
    inside[offset:offset + count * (width + pad)].view(count, width + pad)[:, :width] = True
    assert torch.equal(after[~inside], before[~inside]), "wrote outside its rows"


def test_lookup_keeps_bits_and_device_alpha(handle, device):
    table = torch.randn(500, 264, device=device, dtype=torch.bfloat16)
    table[3] = float("nan")
    table[4] = float("inf")
    ids = torch.randint(5, 500, (300,), device=device)
    out = torch.empty(300, 264, device=device, dtype=torch.bfloat16)
    mc.embedding_lookup(handle, ids, mat(table), mat(out), alpha=2.0)
    assert torch.equal(out, table[ids] * 2)
    handle.set_pointer_mode(capi.MCSPARSE_POINTER_MODE_DEVICE)
    try:
        alpha = torch.full((1,), float("inf"), device=device)
        ids[::3] = -1
        mc.embedding_lookup(handle, ids, mat(table), mat(out), alpha=alpha)
    finally:
        handle.set_pointer_mode(capi.MCSPARSE_POINTER_MODE_HOST)
    assert bool((out[::3] == 0).all()), "padding is zero whatever alpha is"


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
def test_lookup_of_more_rows_than_l2_holds(handle, device, types):
    """A result of more than 64 MB is written past L2."""
    te, ty = types
    gen = torch.Generator(device=device).manual_seed(9)
    count = (80 << 20) // (2048 * torch.finfo(ty).bits // 8)
    table = torch.empty(3000, 2048, dtype=te, device=device).normal_(generator=gen)
    ids = ids_for(count, 3000, "outside", device)
    out = torch.empty(count, 2048, dtype=ty, device=device)
    mc.embedding_lookup(handle, ids, mat(table), mat(out), alpha=0.5)
    ok = (ids >= 0) & (ids < 3000)
    want = torch.where(ok[:, None], table[ids.clamp(0, 2999)].float() * 0.5, 0.0)  # exact: a power of two
    assert torch.equal(out, want.to(ty))


def run_gradient(handle, ids, dy, table, alpha=1.0, beta=0.0, base=0):
    m_y, m_e = mc.DnMat(dy, dy.shape[0], dy.shape[1], dy.stride(0)), mc.DnMat(table, *table.shape, table.stride(0))
    buf = torch.empty(mc.embedding_gradient_buffer_size(handle, ids, m_y, m_e), dtype=torch.uint8, device=dy.device)
    buf.fill_(0xA5)
    mc.embedding_gradient(handle, ids, m_y, m_e, buf, alpha=alpha, beta=beta, base=base)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: f"{str(t[0])[6:]}-{str(t[1])[6:]}")
@pytest.mark.parametrize("kind", ["one", "each", "outside", "edges", "skewed"])
@pytest.mark.parametrize("count,rows,width", [(1, 1, 1), (7, 300, 40), (513, 301, 136), (4099, 97, 72), (3000, 5000, 515)])
def test_gradient(handle, device, types, kind, count, rows, width):
    te, ty = types
    gen = torch.Generator(device=device).manual_seed(11)
    index, base = (torch.int32, 1) if width % 2 else (torch.int64, 0)
    ids = ids_for(count, rows, kind, device, index=index, base=base)
    dy = torch.empty(count, width, dtype=ty, device=device).normal_(generator=gen)
    for beta in (0.0, 1.0, -0.5):
        table = torch.empty(rows, width, dtype=te, device=device).normal_(generator=gen)
        if beta == 0.0:
            table.fill_(float("nan"))  # not read
        want = ref.gradient(ids, dy, rows, 0.75, beta, table, base)
        run_gradient(handle, ids, dy, table, 0.75, beta, base)
        ref.close(table, want, f"beta {beta}")


@pytest.mark.parametrize("count", [2047, 2049, 16384, 16385, 40000, 131072, 140001])
def test_gradient_long_batches(handle, device, count):
    gen = torch.Generator(device=device).manual_seed(count)
    ids = ids_for(count, 70000, "skewed", device, seed=count)
    dy = torch.empty(count, 24, dtype=torch.bfloat16, device=device).normal_(generator=gen)
    table = torch.empty(70000, 24, dtype=torch.float32, device=device)
    run_gradient(handle, ids, dy, table)
    ref.close(table, ref.gradient(ids, dy, 70000, 1.0, 0.0, table), "gradient")
    again = torch.empty_like(table)
    run_gradient(handle, ids, dy, again)
    assert torch.equal(table, again), "equal inputs, equal bits"


@pytest.mark.parametrize("width", [24, 33, 264])
@pytest.mark.parametrize("run", [1, 7, 8, 9, 16, 63, 64, 65, 512, 2048, 2049, 6000, 30000])
def test_gradient_of_runs_of_one_length(handle, device, run, width):
    """Every id occurs `run` times, so that sums begin and end on, before and behind the places where the work is cut."""
    gen = torch.Generator(device=device).manual_seed(run)
    rows = max(30000 // run, 1)
    ids = torch.arange(rows, device=device).repeat_interleave(run)
    ids = ids[torch.randperm(len(ids), generator=gen, device=device)] if run % 2 else ids
    dy = torch.empty(len(ids), width, dtype=torch.bfloat16, device=device).normal_(generator=gen)
    for beta in (0.0, 1.0):
        table = torch.empty(rows + 3, width, device=device).normal_(generator=gen)
        want = ref.gradient(ids, dy, rows + 3, 1.0, beta, table)
        run_gradient(handle, ids, dy, table, beta=beta)
        ref.close(table, want, f"beta {beta}")


def test_gradient_strides_and_untouched_rows(handle, device):
    gen = torch.Generator(device=device).manual_seed(3)
    for pad, offset in ((8, 8), (3, 1)):
        whole_y, dy = strided(600, 136, torch.bfloat16, device, pad, offset, gen)
        whole, table = strided(90, 136, torch.float32, device, pad, offset, gen)
        table[7] = float("nan")  # a row without tokens
        ids = ids_for(600, 90, "skewed", device, index=torch.int32)
        ids[ids == 7] = 8
        before = whole.clone()
        want = ref.gradient(ids, dy, 90, 1.0, 1.0, table)
        run_gradient(handle, ids, dy, table, 1.0, 1.0)
        keep = torch.ones(90, dtype=torch.bool, device=device)
        keep[7] = False
        ref.close(table[keep], (want[0][keep], want[1][keep]), "strided")
        inside = torch.zeros_like(whole, dtype=torch.bool)
        touched = torch.bincount(ids.long(), minlength=90) > 0
        inside[offset:offset + 90 * (136 + pad)].view(90, 136 + pad)[:, :136] = touched[:, None]
        same = (whole == before) | (whole.isnan() & before.isnan())
        assert bool(same[~inside].all()), "beta = 1 leaves rows without tokens as they were"


@pytest.mark.parametrize("rows", [300_000, 1 << 28])
@pytest.mark.parametrize("count", [500, 5000])
def test_gradient_of_a_tall_table(handle, device, rows, count):
    """Ids of 19 and 29 bits: three and four passes of the sort, an odd and an even number."""
    gen = torch.Generator(device=device).manual_seed(13)
    ids = torch.randint(0, rows, (count,), device=device, generator=gen)
    ids[::3] = ids[0]
    ids[1::7] = rows - 1
    dy = torch.empty(count, 2, dtype=torch.float32, device=device).normal_(generator=gen)
    table = torch.zeros(rows, 2, device=device)
    run_gradient(handle, ids, dy, table, beta=1.0)
    touched, inverse = torch.unique(ids, return_inverse=True)
    value, allowed = ref.gradient(inverse, dy, len(touched), 1.0, 0.0, torch.zeros(len(touched), 2, device=device))
    ref.close(table[touched], (value, allowed), "gradient")
    table[touched] = 0
    assert not bool(table.any()), "wrote a row nobody named"


def test_gradient_with_scalars_on_the_device(handle, device):
    gen = torch.Generator(device=device).manual_seed(14)
    ids = ids_for(700, 200, "outside", device)
    dy = torch.empty(700, 64, dtype=torch.bfloat16, device=device).normal_(generator=gen)
    handle.set_pointer_mode(capi.MCSPARSE_POINTER_MODE_DEVICE)
    try:
        for a, b in ((0.75, 0.0), (2.0, 1.0), (-1.0, 0.5)):
            table = torch.empty(200, 64, device=device).normal_(generator=gen)
            want = ref.gradient(ids, dy, 200, a, b, table)
            run_gradient(handle, ids, dy, table, torch.full((1,), a, device=device), torch.full((1,), b, device=device))
            ref.close(table, want, f"{a} {b}")
    finally:
        handle.set_pointer_mode(capi.MCSPARSE_POINTER_MODE_HOST)


def test_no_rows(handle, device):
    """A table without rows: every index lies outside it."""
    ids = torch.zeros(5, dtype=torch.int32, device=device)
    table = mc.DnMat(torch.zeros(1, 16, device=device), 0, 16, 16)
    out = torch.full((5, 16), 7.0, device=device)
    mc.embedding_lookup(handle, ids, table, mat(out))
    assert bool((out == 0).all())
    buf = torch.empty(mc.embedding_gradient_buffer_size(handle, ids, mat(out), table), dtype=torch.uint8, device=device)
    mc.embedding_gradient(handle, ids, mat(out), table, buf)


def test_gradient_empty(handle, device):
    table = torch.randn(5, 8, device=device)
    ids = torch.empty(1, dtype=torch.int64, device=device)[:0]
    dy = torch.empty(1, 8, device=device)
    m_y, m_e = mc.DnMat(dy, 0, 8, 8), mat(table)
    buf = torch.empty(mc.embedding_gradient_buffer_size(handle, ids, m_y, m_e), dtype=torch.uint8, device=device)
    before = table.clone()
    mc.embedding_gradient(handle, ids, m_y, m_e, buf, beta=1.0)
    assert torch.equal(table, before)
    mc.embedding_gradient(handle, ids, m_y, m_e, buf, beta=2.0)
    assert torch.equal(table, before * 2)
    mc.embedding_gradient(handle, ids, m_y, m_e, buf, beta=0.0)
    assert bool((table == 0).all())
    mc.embedding_lookup(handle, ids, m_e, m_y)


def test_gradient_captured_and_replayed(device):
    """Two graphs that share one work buffer, replayed in turn on a stream of their own."""
    stream = torch.cuda.Stream()
    handle = mc.Handle(stream)
    gen = torch.Generator(device=device).manual_seed(5)
    sets = []
    for n in (900, 2500):
        ids = ids_for(n, 400, "skewed", device, seed=n)
        dy = torch.empty(n, 128, dtype=torch.float16, device=device).normal_(generator=gen)
        sets.append((ids, dy, torch.empty(400, 128, device=device)))
    plans = [(i, mat(y), mat(e)) for i, y, e in sets]
    buf = torch.empty(max(mc.embedding_gradient_buffer_size(handle, *p) for p in plans), dtype=torch.uint8, device=device)
    graphs = []
    torch.cuda.synchronize()
    for p in plans:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            mc.embedding_gradient(handle, *p, buf)
        graphs.append(g)
    with torch.cuda.stream(stream):
        for turn in range(3):
            for (ids, dy, e), g in zip(sets, graphs):
                dy.normal_(generator=gen)
                ids.copy_(ids_for(ids.numel(), 400, ["skewed", "one", "outside"][turn], device, seed=turn))
                e.fill_(float("nan"))
                g.replay()
                stream.synchronize()
                ref.close(e, ref.gradient(ids, dy, 400, 1.0, 0.0, e), f"replay {turn}")
    handle.close()


def test_refusals(handle, device):
    E, Y = torch.zeros(10, 16, device=device), torch.zeros(4, 16, device=device)
    ids = torch.zeros(4, dtype=torch.int64, device=device)
    one = C.c_float(1.0)
    p1 = C.cast(C.byref(one), C.c_void_p)

    def lookup(h=handle.h, alpha=p1, count=4, i=ids.data_ptr(), it=capi.MCSPARSE_INDEX_64I, base=0, e=None, y=None):
        e, y = e or mat(E), y or mat(Y)
        return lib.mcsparseB200EmbeddingLookup(h, alpha, count, i, it, base, e.d, y.d)

    assert lookup() == 0
    assert lookup(h=None) == capi.MCSPARSE_STATUS_NOT_INITIALIZED
    invalid, refused = capi.MCSPARSE_STATUS_INVALID_VALUE, capi.MCSPARSE_STATUS_NOT_SUPPORTED
    assert lookup(alpha=None) == invalid
    assert lookup(i=None) == invalid
    assert lookup(i=ids.data_ptr() + 4) == invalid
    assert lookup(count=-1) == invalid
    assert lookup(count=3) == invalid
    assert lookup(base=2) == invalid
    assert lookup(it=capi.MCSPARSE_INDEX_16U) == refused
    assert lookup(e=mc.DnMat(E, 10, 16, 15)) == invalid
    assert lookup(y=mc.DnMat(Y, 4, 8, 16)) == invalid
    assert lookup(e=mc.DnMat(E, 10, 16, 16, order=capi.MCSPARSE_ORDER_COL)) == refused
    assert lookup(e=mc.DnMat(E.double(), 10, 16, 16)) == refused
    half, brain = mat(E.half()), mat(Y.bfloat16())
    assert lookup(e=half, y=brain) == refused
    size = C.c_size_t()
    assert lib.mcsparseB200EmbeddingGradient_bufferSize(handle.h, 4, 3, mat(Y).d, mat(E).d, None) == invalid
    assert lib.mcsparseB200EmbeddingGradient_bufferSize(handle.h, 4, 3, mat(Y).d, None, C.byref(size)) == invalid
    m_y, m_e = mat(Y), mat(E)
    assert lib.mcsparseB200EmbeddingGradient(handle.h, p1, 4, ids.data_ptr(), 3, 0, m_y.d, p1, m_e.d, None) == invalid
    assert lib.mcsparseB200EmbeddingGradient(handle.h, p1, 4, ids.data_ptr(), 3, 0, m_y.d, None, m_e.d, 256) == invalid
    with pytest.raises(ValueError):
        mc.embedding_lookup(handle, ids.cpu(), m_e, m_y)
    with pytest.raises(ValueError):
        mc.embedding_lookup(handle, ids.float(), m_e, m_y)
    with pytest.raises(ValueError):
        mc.embedding_gradient(handle, ids, m_y, m_e, torch.empty(8, dtype=torch.uint8, device=device))


def test_matrices_without_values_are_refused(handle, device):
    """mcsparseDnMatSetValues may take a descriptor's values away: refused on the host, as the library's other products do."""
    E, Y = torch.full((10, 16), 7.0, device=device), torch.full((4, 16), 7.0, device=device)
    ids = torch.zeros(4, dtype=torch.int64, device=device)
    m_e, m_y = mat(E), mat(Y)
    buf = torch.empty(mc.embedding_gradient_buffer_size(handle, ids, m_y, m_e), dtype=torch.uint8, device=device)
    for m in (m_e, m_y):
        capi.check(lib.mcsparseDnMatSetValues(m.d, None))
        for call in (lambda: mc.embedding_lookup(handle, ids, m_e, m_y), lambda: mc.embedding_gradient(handle, ids, m_y, m_e, buf)):
            with pytest.raises(mc.McsparseError) as e:
                call()
            assert e.value.status == capi.MCSPARSE_STATUS_INVALID_VALUE
        capi.check(lib.mcsparseDnMatSetValues(m.d, m.values.data_ptr()))
    torch.cuda.synchronize()
    assert bool((E == 7.0).all()) and bool((Y == 7.0).all())
    # none are missing where there are none
    capi.check(lib.mcsparseDnMatSetValues(m_y.d, None))
    empty = mc.DnMat(Y, 0, 16, 16)
    capi.check(lib.mcsparseDnMatSetValues(empty.d, None))
    mc.embedding_lookup(handle, ids[:0], m_e, empty)
    mc.embedding_gradient(handle, ids[:0], empty, m_e, buf, beta=1.0)
    torch.cuda.synchronize()
    assert bool((E == 7.0).all())


def gradient_time(handle, device, count, width, hot):
    """Median milliseconds of a gradient (beta = 1) of `count` tokens, a share `hot` of them with one id, the others spread."""
    rows = 50000
    gen = torch.Generator(device=device).manual_seed(count)
    ids = torch.randint(0, rows, (count,), device=device, generator=gen)
    ids[torch.rand(count, device=device, generator=gen) < hot] = 7
    dy, table = torch.ones(count, width, dtype=torch.bfloat16, device=device), torch.zeros(rows, width, device=device)
    m_y, m_e = mat(dy), mat(table)
    buf = torch.empty(mc.embedding_gradient_buffer_size(handle, ids, m_y, m_e), dtype=torch.uint8, device=device)
    times = []
    for _ in range(7):
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        start.record()
        mc.embedding_gradient(handle, ids, m_y, m_e, buf, beta=1.0)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    return sorted(times)[3]


def test_time_of_a_run_grows_with_its_length(handle, device):
    """Eight times as many tokens of one id cost about eight times as much (with chunks that look for each other's ends one after
    the other: 21 times)."""
    short, long = (gradient_time(handle, device, n, 512, 1.0) for n in (1 << 19, 1 << 22))
    assert long < 13 * short, f"{short} ms and {long} ms"


@pytest.mark.parametrize("types,width", [((torch.float32, torch.bfloat16), 8), ((torch.float32, torch.float32), 140), ((torch.float32, torch.bfloat16), 264),
                                         ((torch.float32, torch.float16), 131)], ids=str)
def test_gradient_of_runs_over_many_chunks(handle, device, types, width):
    """Sums over 1 to 2250 chunks of 8 tokens, at the numbers of chunks where their groups change, and beginning and ending anywhere in
    a chunk. Whole numbers whose sums stay below 2^24: every order of additions gives the same bits, and a chunk that is
    missing or counted twice shows."""
    gen = torch.Generator(device=device).manual_seed(width)
    parts = [1, 2, 63, 64, 65, 66, 80, 81, 255, 256, 257, 258, 271, 272, 273, 1024, 1025]
    runs = [8 * n + e for n in parts for e in (-3, 0, 5)]
    te, ty = types
    batches = [[]]
    for n in runs + [18000]:
        if sum(batches[-1]) + n > 18000:
            batches.append([])
        batches[-1].append(n)
    for lengths in batches:
        ids = torch.repeat_interleave(torch.arange(len(lengths), device=device), torch.tensor(lengths, device=device))
        ids = ids[torch.randperm(len(ids), generator=gen, device=device)]
        assert len(ids) * -(-width // 256) // (148 * 16) < 16, "chunks of 8 tokens"
        dy = torch.randint(-8, 9, (len(ids), width), device=device, generator=gen).to(ty)
        table = torch.randint(-8, 9, (len(lengths), width), device=device, generator=gen).to(te)
        want = table.double().index_add(0, ids, 2.0 * dy.double())
        run_gradient(handle, ids, dy, table, alpha=2.0, beta=1.0)
        assert torch.equal(table.double(), want)


def test_one_id_in_all_tokens_costs_little_more_than_spread_ids(handle, device):
    """(One warp for all the partial sums of a row: 11 times as much.)"""
    spread, one = (gradient_time(handle, device, 1 << 22, 512, hot) for hot in (0.0, 1.0))
    assert one < 3 * spread, f"{spread} ms and {one} ms"


@pytest.mark.parametrize("count", [100, 5000, 140001])
def test_gradient_buffer_does_not_grow_with_the_table(handle, device, count):
    """The sort needs room for the tokens, not for the rows (it once reserved a word for each of them, a gigabyte at 2^28)."""
    ids = torch.zeros(count, dtype=torch.int32, device=device)
    dy, table = torch.empty(count, 2, device=device), torch.empty(1, 2, device=device)  # (sizes alone are looked at)
    sizes = [mc.embedding_gradient_buffer_size(handle, ids, mat(dy), mc.DnMat(table, rows, 2, 2)) for rows in (10, 50000, 1 << 28)]
    assert sizes[0] == sizes[1] == sizes[2], sizes


@pytest.mark.parametrize("kind", ["one", "outside", "edges", "skewed"])
@pytest.mark.parametrize("index,base", [(torch.int32, 1), (torch.int64, 0)], ids=str)
@pytest.mark.parametrize("rows", [200, 70000, 1 << 26])
def test_gradient_of_more_tokens_than_one_cluster_sorts(handle, device, kind, index, base, rows):
    """140001 tokens, ids of one to four digits, and those outside the table, whose key is the number of rows."""
    count = 140001
    gen = torch.Generator(device=device).manual_seed(rows)
    ids = ids_for(count, rows, kind, device, seed=3, index=index, base=base)
    dy = torch.randint(-4, 5, (count, 8), device=device, generator=gen).bfloat16()  # whole numbers: any order of additions is exact
    table = torch.zeros(rows, 8, device=device)
    run_gradient(handle, ids, dy, table, beta=1.0, base=base)
    i = ids.long() - base
    ok = (i >= 0) & (i < rows)
    want = torch.zeros(rows, 8, device=device).index_add_(0, i[ok], dy[ok].float())
    assert torch.equal(table, want)
