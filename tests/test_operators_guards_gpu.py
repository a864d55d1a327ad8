"""Outputs and work buffers of the embedding and attention calls inside larger blocks of memory: each call writes nothing beside
them, the work buffers having exactly the bytes that were asked for."""

import pytest
import torch

import mcsparse_b200 as mc

pytestmark = pytest.mark.gpu

GUARD, FILL = 1 << 16, 0x5A


class Guards:
    """Tensors with GUARD bytes of FILL on both sides."""

    def __init__(self, device):
        self.device, self.blocks = device, []

    def tensor(self, shape, dtype, shift=0):
        """`shift`: bytes past a 256-byte boundary."""
        n = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
        whole = torch.full((2 * GUARD + shift + n,), FILL, dtype=torch.uint8, device=self.device)
        self.blocks.append((whole, GUARD + shift, n))
        return whole[GUARD + shift:GUARD + shift + n].view(dtype).view(shape)

    def check(self):
        torch.cuda.synchronize()
        for i, (whole, at, n) in enumerate(self.blocks):
            assert bool((whole[:at] == FILL).all()) and bool((whole[at + n:] == FILL).all()), f"tensor {i} of {len(self.blocks)}"


def mat(t):
    return mc.DnMat(t, *t.shape, t.shape[1])


@pytest.mark.parametrize("types", [(torch.float32, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32)], ids=str)
@pytest.mark.parametrize("count,rows,width", [(1, 1, 1), (100, 37, 771), (257, 5001, 136), (5000, 300, 64), (20000, 1000, 24), (140001, 513, 40),
                                              (140001, 513, 33)])
@pytest.mark.parametrize("kind", ["one", "mixed"])
def test_embedding(handle, device, types, count, rows, width, kind):
    te, ty = types
    gen = torch.Generator(device=device).manual_seed(count)
    ids = torch.randint(-3, rows + 3, (count,), device=device, generator=gen)
    if kind == "one":
        ids.fill_(rows - 1)
    for shift in (0, 4):
        g = Guards(device)
        table, y = g.tensor((rows, width), te, shift).normal_(generator=gen), g.tensor((count, width), ty, shift)
        mc.embedding_lookup(handle, ids, mat(table), mat(y))
        buf = g.tensor((mc.embedding_gradient_buffer_size(handle, ids, mat(y), mat(table)),), torch.uint8, shift)
        for beta in (0.0, 1.0, 0.5):
            mc.embedding_gradient(handle, ids, mat(y), mat(table), buf, beta=beta)
        g.check()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 72), (torch.float16, 33), (torch.float32, 48)], ids=str)
@pytest.mark.parametrize("lq,lk,window,sinks", [([1], [1], 1, 0), ([0, 130, 5, 0], [9, 130, 77, 0], 64, 2), ([257, 1023], [257, 1023], 100, 0),
                                                ([5000, 700], [5000, 700], 64, 130), ([3000], [2500], 200, 1024)], ids=str)
def test_attention(handle, device, dtype, dim, lq, lk, window, sinks):
    """Forward and backward, with pieces of first tokens' queries (5000 tokens, 130 first ones) and without."""
    hq, hk = 4, 2
    gen = torch.Generator(device=device).manual_seed(dim)
    qo, ko = (torch.tensor([0] + torch.tensor(x).cumsum(0).tolist(), dtype=torch.int32, device=device) for x in (lq, lk))
    tq, tk = sum(lq), sum(lk)
    g = Guards(device)
    q, go = (torch.empty(tq, hq, dim, dtype=dtype, device=device).normal_(generator=gen) for _ in range(2))
    k, v = (torch.empty(tk, hk, dim, dtype=dtype, device=device).normal_(generator=gen) for _ in range(2))
    out, dq, dk, dv = (g.tensor(x.shape, dtype) for x in (q, q, k, v))
    lse = g.tensor((hq, tq), torch.float32, 4)
    w = mc.Window(window, sinks, hq, hk, dim, dtype)
    buf = g.tensor((mc.window_attention_backward_buffer_size(handle, w, len(lq), tq, tk),), torch.uint8, 1)
    mc.window_attention(handle, w, q, k, v, out, lse, q_offsets=qo, k_offsets=ko)
    mc.window_attention_backward(handle, w, q, k, v, out, lse, go, dq, dk, dv, buf, q_offsets=qo, k_offsets=ko)
    g.check()
    for x in (out, dq, dk, dv):
        assert bool(x.isfinite().all())


@pytest.mark.parametrize("offsets", [[0, 2500, 1000, 9000], [-70, 2600, 2 ** 31 - 1, 2900], [3000, 2000, 1000, 0], [5, 5, 5, 5]], ids=str)
@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 20)], ids=str)
def test_offsets_that_lie(handle, device, offsets, dtype, dim):
    """Offsets that do not ascend or leave the tensors: rows of no meaning, but nothing beside any output is written."""
    n, hq, hk = 3000, 4, 2
    gen = torch.Generator(device=device).manual_seed(dim)
    q, go = (torch.empty(n, hq, dim, dtype=dtype, device=device).normal_(generator=gen) for _ in range(2))
    k, v = (torch.empty(n, hk, dim, dtype=dtype, device=device).normal_(generator=gen) for _ in range(2))
    o = torch.tensor(offsets, dtype=torch.int32, device=device)
    plain = torch.tensor([0, 1000, 2000, 3000], dtype=torch.int32, device=device)
    w = mc.Window(64, 130, hq, hk, dim, dtype)
    for qo, ko in ((o, o), (o, plain), (plain, o)):
        g = Guards(device)
        out, dq, dk, dv = (g.tensor(x.shape, dtype) for x in (q, q, k, v))
        out.zero_()
        lse = g.tensor((hq, n), torch.float32)
        lse.zero_()
        buf = g.tensor((mc.window_attention_backward_buffer_size(handle, w, 3, n, n),), torch.uint8)
        mc.window_attention(handle, w, q, k, v, out, lse, q_offsets=qo, k_offsets=ko)
        mc.window_attention_backward(handle, w, q, k, v, out, lse, go, dq, dk, dv, buf, q_offsets=qo, k_offsets=ko)
        g.check()


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 40), (torch.float32, 64), (torch.float16, 33)], ids=str)
@pytest.mark.parametrize("heads,lengths,window,page", [((2, 1), [1, 0], 4, 16), ((32, 8), [2000, 77, 1], 1024, 16), ((17, 1), [9000], 1 << 40, 0),
                                                       ((32, 8), [12000], 1 << 40, 37), ((4, 1), [70000], 1 << 40, 64)], ids=str)
def test_decode(handle, device, dtype, dim, heads, lengths, window, page):
    """Single tokens with parts that join in a cluster and through the work buffer (8192 visible keys and more)."""
    hq, hk = heads
    gen = torch.Generator(device=device).manual_seed(dim)
    batch, longest = len(lengths), max(lengths)
    per, size = (-(-longest // page), page) if page else (1, longest)
    k, v = (torch.empty(batch * per, size, hk, dim, dtype=dtype, device=device).normal_(generator=gen) for _ in range(2))
    q = torch.empty(batch, hq, dim, dtype=dtype, device=device).normal_(generator=gen)
    table = torch.arange(batch * per, dtype=torch.int32, device=device).view(batch, per) if page else None
    w = mc.Window(window, 3, hq, hk, dim, dtype)
    g = Guards(device)
    out, lse = g.tensor(q.shape, dtype), g.tensor((batch, hq), torch.float32, 4)
    buf = g.tensor((mc.window_attention_decode_buffer_size(handle, w, batch, per, size),), torch.uint8, 1)
    mc.window_attention_decode(handle, w, q, k, v, torch.tensor(lengths, dtype=torch.int32, device=device), out, lse, buf, page_table=table)
    g.check()
    assert bool(out.isfinite().all())
