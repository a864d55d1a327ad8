"""The language-model operators of the library on real work: embedding rows and their gradient, windowed attention
forward, in a training step, and for single tokens over a cache.

A case is a dict of plain values. ``run`` computes it either with elementary torch operations in 32 bits (``own``
false) or with the calls a user makes of the library (``own`` true).
"""

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}


# ----------------------------------------------------------------------------- cases

def listed():
    """kind "lookup": rows of a table; "gradient": the table's gradient; "attention": forward over ragged sequences;
    "training": forward and backward; "decode": one token per sequence over a cache."""
    return [
        # the rows for one decoding step of a small batch: latency
        dict(name="lookup step", kind="lookup", count=61, rows=32000, width=4096, table="bf16", out="bf16", index64=True),
        # the rows for a large prompt batch: bandwidth
        dict(name="lookup prompt", kind="lookup", count=65536, rows=128000, width=4096, table="bf16", out="bf16", index64=True),
        # gradient of a small table with an odd width
        dict(name="gradient small", kind="gradient", count=257, rows=5001, width=771, grad="fp32", table="fp32", index64=False, parts=1),
        # gradient of a training step, fp32 master gradient from bf16 activations
        dict(name="gradient step", kind="gradient", count=16384, rows=50257, width=2048, grad="bf16", table="fp32", index64=True, parts=1),
        # the same accumulated over two micro-batches, a large vocabulary
        dict(name="gradient accumulated", kind="gradient", count=65536, rows=128000, width=2048, grad="bf16", table="fp32", index64=True, parts=2),
        # a handful of short requests in one ragged batch: latency
        dict(name="attention short", kind="attention", lengths="1,37,100,64,200", cached=0, q_heads=8, kv_heads=2, dim=64, window=64, sinks=4, dtype="fp16"),
        # a ragged prompt batch
        dict(name="attention ragged", kind="attention", lengths="4099,257,8001,1023,3004", cached=0, q_heads=16, kv_heads=2, dim=128, window=1024, sinks=16, dtype="bf16"),
        # one long document
        dict(name="attention long", kind="attention", lengths="32768", cached=0, q_heads=32, kv_heads=8, dim=128, window=4096, sinks=4, dtype="bf16"),
        # training on short packed documents with a head size between the powers of two
        dict(name="training packed", kind="training", lengths="700,33,1201,512,555", cached=0, q_heads=12, kv_heads=12, dim=96, window=256, sinks=1, dtype="fp16"),
        # a training step on full sequences with shared key heads
        dict(name="training step", kind="training", lengths="4096,4096,4096,4096", cached=0, q_heads=16, kv_heads=4, dim=128, window=1024, sinks=4, dtype="bf16"),
        # one sequence, one token: latency
        dict(name="decode one", kind="decode", batch=1, longest=5000, page=0, q_heads=32, kv_heads=8, dim=128, window=1024, sinks=4, dtype="bf16"),
        # a serving batch over a paged cache
        dict(name="decode batch", kind="decode", batch=64, longest=8192, page=16, q_heads=32, kv_heads=8, dim=128, window=4096, sinks=4, dtype="bf16"),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["lookup", "gradient", "attention", "training", "decode"])
    if kind in ("lookup", "gradient"):
        width = _log_uniform(rng, 64, 4096)
        rows = _log_uniform(rng, 2000, 128000)
        count = _log_uniform(rng, 1, 65536)
        if kind == "lookup":
            table = rng.choice(["bf16", "fp16", "fp32"])
            return dict(kind=kind, count=count, rows=rows, width=width, table=table,
                        out=rng.choice([table, table, "fp32" if table != "fp32" else "bf16"]), index64=rng.random() < 0.5)
        width = min(width, 2048)
        grad = rng.choice(["bf16", "fp16", "fp32"])
        parts = rng.choice([1, 1, 2])  # several micro-batches accumulate in 32 bits
        return dict(kind=kind, count=count, rows=rows, width=width, grad=grad, table=rng.choice([grad, "fp32"]) if parts == 1 else "fp32",
                    index64=rng.random() < 0.5, parts=parts)
    kv_heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    while kv_heads * group > 32:
        group //= 2
    dim = rng.choice([32, 64, 72, 80, 96, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    window = _log_uniform(rng, 16, 4096)
    sinks = rng.choice([0, 1, 4, 16, 130])
    heads = dict(q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, window=window, sinks=sinks, dtype=dtype)
    if kind == "decode":
        return dict(kind=kind, batch=_log_uniform(rng, 1, 64), longest=_log_uniform(rng, 16, 8192), page=rng.choice([0, 16, 64]), **heads)
    total = _log_uniform(rng, 64, 32768 if kind == "attention" else 12000)
    if window * total > 4096 * 8192:
        heads["window"] = window = max(16, 4096 * 8192 // total)
    sequences = rng.choice([1, 2, 3, 5, 9])
    cuts = sorted(rng.randint(1, max(1, total - 1)) for _ in range(sequences - 1))
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [total])]
    cached = rng.choice([0, 0, 77, 1000]) if kind == "attention" else 0
    return dict(kind=kind, lengths=",".join(str(max(1, n)) for n in lengths), cached=cached, **heads)


# ----------------------------------------------------------------------------- inputs

def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _normal(shape, dtype, gen, scale=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=gen)


def _tokens(case, gen):
    """Token ids as text has them: frequency falls as one over the rank; one in 64 is padding (-1)."""
    u = torch.rand(case["count"], device="cuda", generator=gen, dtype=torch.float64)
    ids = (torch.exp(u * math.log(case["rows"] + 1.0)) - 1.0).floor().clamp_(0, case["rows"] - 1).long()
    ids = torch.where(torch.rand(case["count"], device="cuda", generator=gen) < 1 / 64, torch.full_like(ids, -1), ids)
    return ids if case["index64"] else ids.int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case=case)
    kind = case["kind"]
    if kind == "lookup":
        s["ids"] = _tokens(case, gen)
        s["table"] = _normal((case["rows"], case["width"]), DTYPES[case["table"]], gen, 0.02)
        s["out"] = torch.empty(case["count"], case["width"], dtype=DTYPES[case["out"]], device="cuda")
        s["alpha"] = math.sqrt(case["width"])
    elif kind == "gradient":
        s["ids"] = [_tokens(case, gen) for _ in range(case["parts"])]
        s["dy"] = [_normal((case["count"], case["width"]), DTYPES[case["grad"]], gen) for _ in range(case["parts"])]
        s["dtable"] = torch.empty(case["rows"], case["width"], dtype=DTYPES[case["table"]], device="cuda")
        s["alpha"] = math.sqrt(case["width"])
    else:
        dtype, hq, hk, d = DTYPES[case["dtype"]], case["q_heads"], case["kv_heads"], case["dim"]
        if kind == "decode":
            rng = random.Random(seed)
            b, longest, page = case["batch"], case["longest"], case["page"] or case["longest"]
            lengths = [rng.randint(longest // 2, longest) for _ in range(b)]
            lengths[0] = longest
            per = -(-longest // page)
            s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
            s["pages"] = None
            if case["page"]:
                order = list(range(b * per))
                rng.shuffle(order)
                s["pages"] = torch.tensor(order, dtype=torch.int32, device="cuda").view(b, per)
            s["k"] = _normal((b * per, page, hk, d), dtype, gen)
            s["v"] = _normal((b * per, page, hk, d), dtype, gen)
            s["q"] = _normal((b, hq, d), dtype, gen)
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(b, hq, dtype=torch.float32, device="cuda")
        else:
            lengths = _lengths(case)
            keys = [n + case["cached"] for n in lengths]
            s["q_offsets"] = torch.tensor(np.cumsum([0] + lengths), dtype=torch.int32, device="cuda")
            s["k_offsets"] = torch.tensor(np.cumsum([0] + keys), dtype=torch.int32, device="cuda")
            s["longest"], s["longest_k"] = max(lengths), max(keys)
            tq, tk = sum(lengths), sum(keys)
            s["q"] = _normal((tq, hq, d), dtype, gen)
            s["k"] = _normal((tk, hk, d), dtype, gen)
            s["v"] = _normal((tk, hk, d), dtype, gen)
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(hq, tq, dtype=torch.float32, device="cuda")
            if kind == "training":
                s["dout"] = _normal((tq, hq, d), dtype, gen)
                s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[n]) for n in "qkv")
    return s


# ----------------------------------------------------------------------------- plain forms

def _plain_lookup(s):
    ids = s["ids"].long()
    valid = ids >= 0
    y = s["table"][ids.clamp(min=0)].float() * s["alpha"]
    return torch.where(valid[:, None], y, torch.zeros((), device=y.device)).to(s["out"].dtype)


def _plain_gradient(s):
    rows, width = s["dtable"].shape
    ids = torch.cat(s["ids"]).long()
    ids = torch.where(ids >= 0, ids, rows)
    total = torch.zeros(rows + 1, width, dtype=torch.float32, device=ids.device)
    total.index_add_(0, ids, torch.cat(s["dy"]).float() * s["alpha"])
    return total[:rows].to(s["dtable"].dtype)


def _band(s):
    """Queries and the keys that may be seen, in blocks: positions, flat indices and the mask of every pair.

    The sequences are laid side by side, padded to the longest; a block of queries meets the first tokens and the
    stretch of keys its windows cover."""
    case, dev = s["case"], s["q"].device
    window, sinks = case["window"], case["sinks"]
    lq = (s["q_offsets"][1:] - s["q_offsets"][:-1]).long()
    lk = (s["k_offsets"][1:] - s["k_offsets"][:-1]).long()
    longest = s["longest"]
    whole = s["longest_k"] <= 2048 or 2 * window >= s["longest_k"]
    block = longest if whole else max(256, min(1024, window))
    blocks = -(-longest // block)
    qi = torch.arange(blocks * block, device=dev).view(1, blocks, block)
    pos = qi + (lk - lq)[:, None, None]                                   # [sequences, blocks, block]
    if whole:
        kj = torch.arange(s["longest_k"], device=dev).view(1, 1, -1).expand(len(lq), blocks, -1)
    else:
        back = pos[:, :, :1] - window + 1
        kj = torch.cat([torch.arange(sinks, device=dev).expand(len(lq), blocks, -1),
                        back + torch.arange(window + block - 1, device=dev)], -1)
    first = torch.arange(kj.shape[-1], device=dev) < (0 if whole else sinks)
    i, j = pos[..., :, None], kj[..., None, :]
    near = j > i - window
    # a key that stands in both parts is seen once, in the window's part where it lies there
    seen = torch.where(first, ~near, near | (j < sinks if whole else torch.zeros_like(near)))
    mask = (seen & (j <= i) & (j >= 0) & (j < lk[:, None, None, None]) & (qi < lq[:, None, None])[..., :, None])
    qf = (s["q_offsets"][:-1, None, None].long() + qi).clamp(0, s["q"].shape[0] - 1)
    kf = (s["k_offsets"][:-1, None, None].long() + kj).clamp(0, s["k"].shape[0] - 1)
    return qf, kf, mask, (qi < lq[:, None, None])


def _scores(s, qf, kf, mask):
    case = s["case"]
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    q = s["q"][qf].float().unflatten(-2, (hk, hq // hk))                    # [sequences, blocks, block, hk, group, d]
    k, v = s["k"][kf].float(), s["v"][kf].float()                           # [sequences, blocks, keys, hk, d]
    x = torch.einsum("abihgd,abjhd->abhgij", q, k) * d ** -0.5
    x = x.masked_fill_(~mask[:, :, None, None], -math.inf)
    m = x.amax(-1, keepdim=True).clamp_min_(-1e30)
    p = (x - m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log())[..., 0]
    p /= total.clamp_min(1e-37)
    return q, k, v, p, lse


def _flat_rows(x, qf, real, like):
    """Blocks of rows back to the flat order of the tokens."""
    out = torch.zeros(like.shape, dtype=torch.float32, device=like.device)
    out[qf[real]] = x[real].flatten(1).view(-1, *like.shape[1:])
    return out


def _plain_attention(s):
    qf, kf, mask, real = _band(s)
    real = real.expand(qf.shape)
    q, k, v, p, lse = _scores(s, qf, kf, mask)
    o = torch.einsum("abhgij,abjhd->abihgd", p, v)
    out = _flat_rows(o, qf, real, s["q"])
    flat_lse = _flat_rows(lse.permute(0, 1, 4, 2, 3), qf, real, s["q"][..., 0]).t().contiguous()
    if s["case"]["kind"] == "attention":
        return out.to(s["q"].dtype), flat_lse
    do = s["dout"][qf].float().unflatten(-2, q.shape[-3:-1]) * real[..., None, None, None]
    dv = torch.einsum("abhgij,abihgd->abjhd", p, do)
    dp = torch.einsum("abihgd,abjhd->abhgij", do, v)
    delta = (do * o).sum(-1).permute(0, 1, 3, 4, 2)[..., None]
    ds = p.mul_(dp.sub_(delta)).mul_(s["case"]["dim"] ** -0.5)
    dq = _flat_rows(torch.einsum("abhgij,abjhd->abihgd", ds, k), qf, real, s["q"])
    dk = torch.einsum("abhgij,abihgd->abjhd", ds, q)
    shape = s["k"].shape
    dk = torch.zeros(shape, dtype=torch.float32, device=dk.device).index_add_(0, kf.flatten(), dk.flatten(0, 2))
    dv = torch.zeros(shape, dtype=torch.float32, device=dk.device).index_add_(0, kf.flatten(), dv.flatten(0, 2))
    t = s["q"].dtype
    return out.to(t), flat_lse, dq.to(t), dk.to(t), dv.to(t)


def _plain_decode(s):
    case = s["case"]
    hq, hk, d, window = case["q_heads"], case["kv_heads"], case["dim"], case["window"]
    page = s["k"].shape[1]
    length = s["lengths"].long()[:, None]
    dev = s["q"].device
    sinks, recent = torch.arange(case["sinks"], device=dev), torch.arange(min(window, case["longest"]), device=dev)
    pos = torch.cat([sinks.expand(len(length), -1), length - 1 - recent], 1)
    far = length - window
    seen = torch.where(torch.arange(pos.shape[1], device=dev) < case["sinks"], pos < far, (pos >= 0) & (pos >= far)) & (pos < length)
    at = pos.clamp(0, case["longest"] - 1)
    number = at // page
    if s["pages"] is not None:
        number = s["pages"].long().gather(1, number)
    else:
        number = torch.arange(len(length), device=dev)[:, None].expand_as(number)
    k, v = s["k"][number, at % page].float(), s["v"][number, at % page].float()
    q = s["q"].float().unflatten(1, (hk, hq // hk))
    x = torch.einsum("bhgd,bjhd->bhgj", q, k) * d ** -0.5
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = (x - m).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bhgj,bjhd->bhgd", p, v) / total
    return o.flatten(1, 2).to(s["q"].dtype), (m + total.log())[..., 0].flatten(1)


# ----------------------------------------------------------------------------- the library's calls

_HANDLES = {}


def _library():
    """The package and a handle on the current stream, as a program keeps them."""
    import mcsparse_b200 as mc

    stream = torch.cuda.current_stream()
    key = (stream.device_index, stream.cuda_stream)
    if key not in _HANDLES:
        _HANDLES[key] = mc.Handle(stream)
    return mc, _HANDLES[key]


def _own(s):
    mc, h = _library()
    case = s["case"]
    kind = case["kind"]
    if kind == "lookup":
        if "plan" not in s:
            s["plan"] = mc.DnMat(s["table"], *s["table"].shape, case["width"]), mc.DnMat(s["out"], *s["out"].shape, case["width"])
        table, out = s["plan"]
        mc.embedding_lookup(h, s["ids"], table, out, alpha=s["alpha"])
        return s["out"]
    if kind == "gradient":
        if "plan" not in s:
            dy = [mc.DnMat(t, *t.shape, case["width"]) for t in s["dy"]]
            dtable = mc.DnMat(s["dtable"], *s["dtable"].shape, case["width"])
            size = mc.embedding_gradient_buffer_size(h, s["ids"][0], dy[0], dtable)
            s["plan"] = dy, dtable, torch.empty(size, dtype=torch.uint8, device="cuda")
        dy, dtable, buffer = s["plan"]
        for i, (ids, g) in enumerate(zip(s["ids"], dy)):
            mc.embedding_gradient(h, ids, g, dtable, buffer, alpha=s["alpha"], beta=0.0 if i == 0 else 1.0)
        return s["dtable"]
    if "window" not in s:
        s["window"] = mc.Window(case["window"], case["sinks"], case["q_heads"], case["kv_heads"], case["dim"], s["q"].dtype)
    w = s["window"]
    if kind == "decode":
        if "buffer" not in s:
            size = mc.window_attention_decode_buffer_size(h, w, case["batch"], case["longest"])
            s["buffer"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        mc.window_attention_decode(h, w, s["q"], s["k"], s["v"], s["lengths"], s["out"], s["lse"], s["buffer"], page_table=s["pages"])
        return s["out"], s["lse"]
    mc.window_attention(h, w, s["q"], s["k"], s["v"], s["out"], s["lse"], q_offsets=s["q_offsets"], k_offsets=s["k_offsets"])
    if kind == "attention":
        return s["out"], s["lse"]
    if "buffer" not in s:
        size = mc.window_attention_backward_buffer_size(h, w, s["q_offsets"].numel() - 1, s["q"].shape[0], s["k"].shape[0])
        s["buffer"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    mc.window_attention_backward(h, w, s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"], s["dv"],
                                 s["buffer"], q_offsets=s["q_offsets"], k_offsets=s["k_offsets"])
    return s["out"], s["lse"], s["dq"], s["dk"], s["dv"]


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "lookup":
        return _plain_lookup(state)
    if kind == "gradient":
        return _plain_gradient(state)
    if kind == "decode":
        return _plain_decode(state)
    return _plain_attention(state)


# ----------------------------------------------------------------------------- what a pass cannot do without

def _pairs(lq, lk, window, sinks):
    """Visible (query, key) pairs of one sequence."""
    p = np.arange(lk - lq, lk, dtype=np.int64)
    near = np.minimum(p + 1, window)
    far = np.clip(np.minimum(p - window + 1, sinks), 0, None)
    return int(np.where(p >= 0, near + far, 0).sum())


def _keys_seen(lq, lk, window, sinks):
    """Keys of one sequence that some query sees."""
    low = max(0, lk - lq - window + 1)
    return lk - low + min(sinks, low)


def work(case):
    kind = case["kind"]
    if kind == "lookup":
        n = case["count"] * case["width"]
        # every distinct row is read once: with ids log-uniform over the rows, expected from the distribution
        r = np.arange(case["rows"], dtype=np.float64)
        share = np.log((r + 2) / (r + 1)) / math.log(case["rows"] + 1.0) * (63 / 64)
        distinct = float((1 - np.exp(case["count"] * np.log1p(-share))).sum())
        return {"bytes": n * SIZES[case["out"]] + distinct * case["width"] * SIZES[case["table"]] + case["count"] * (8 if case["index64"] else 4), "flops": n}
    if kind == "gradient":
        n = case["count"] * case["width"] * case["parts"]
        return {"bytes": n * SIZES[case["grad"]] + case["rows"] * case["width"] * SIZES[case["table"]]
                + case["parts"] * case["count"] * (8 if case["index64"] else 4), "flops": 2 * n}
    hq, hk, d, e = case["q_heads"], case["kv_heads"], case["dim"], SIZES[case["dtype"]]
    if kind == "decode":
        # lengths are uniform between half the longest and the longest
        n = np.arange(case["longest"] // 2, case["longest"] + 1, dtype=np.float64)
        low = np.clip(n - case["window"], 0, None)
        seen = float(np.mean(n - low + np.minimum(case["sinks"], low))) * case["batch"]
        return {"bytes": seen * hk * d * 2 * e + case["batch"] * hq * (2 * d * e + 4), "flops": 4 * d * hq * seen}
    lengths = _lengths(case)
    keys = [n + case["cached"] for n in lengths]
    pairs = sum(_pairs(a, b, case["window"], case["sinks"]) for a, b in zip(lengths, keys))
    seen = sum(_keys_seen(a, b, case["window"], case["sinks"]) for a, b in zip(lengths, keys))
    rows = sum(lengths)
    forward = rows * hq * (2 * d * e + 4) + seen * hk * d * 2 * e
    if kind == "attention":
        return {"bytes": forward, "flops": 4 * d * pairs * hq}
    return {"bytes": forward + rows * hq * 2 * d * e + sum(keys) * hk * d * 2 * e, "flops": 14 * d * pairs * hq}


# ----------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "lookup":
        ids = s["ids"].cpu().numpy()
        rows = torch.from_numpy(np.where(ids < 0, 0, ids)).cuda().long()
        return s["table"].index_select(0, rows).double().mul_(s["alpha"]).mul_(torch.from_numpy(ids >= 0).cuda()[:, None])
    if kind == "gradient":
        ids, dy = torch.cat(s["ids"]).long(), torch.cat(s["dy"])
        order = torch.argsort(ids, stable=True)
        number, counts = torch.unique_consecutive(ids[order], return_counts=True)
        out = torch.zeros(case["rows"], case["width"], dtype=torch.float64, device="cuda")
        ends = torch.cumsum(counts, 0)
        for first in range(0, case["width"], 256):  # running sums of slabs of columns: 64 bits leave 2^-53 of the total
            sums = torch.cumsum(dy[:, first:first + 256][order].double(), 0)
            upto = sums[ends - 1]
            each = torch.diff(upto, dim=0, prepend=torch.zeros_like(upto[:1]))
            keep = number >= 0
            out[number[keep], first:first + 256] = each[keep] * s["alpha"]
        return out
    scale = case["dim"] ** -0.5
    group = case["q_heads"] // case["kv_heads"]
    if kind == "decode":
        out, lse = torch.zeros_like(s["q"], dtype=torch.float64), torch.zeros_like(s["lse"], dtype=torch.float64)
        for b, n in enumerate(s["lengths"].tolist()):
            j = torch.arange(n, device="cuda")
            j = j[(j >= n - case["window"]) | (j < case["sinks"])]
            page = s["k"].shape[1]
            at = (torch.full_like(j, b) if s["pages"] is None else s["pages"][b].long()[j // page]) * page + j % page
            k = s["k"].flatten(0, 1)[at].double().repeat_interleave(group, 1)
            v = s["v"].flatten(0, 1)[at].double().repeat_interleave(group, 1)
            x = (k * s["q"][b].double()).sum(-1) * scale
            lse[b] = torch.logsumexp(x, 0)
            out[b] = (torch.exp(x - lse[b])[..., None] * v).sum(0)
        return out, lse
    lengths = _lengths(case)
    pairs = sum(_pairs(n, n + case["cached"], case["window"], case["sinks"]) for n in lengths) * case["q_heads"]
    if pairs * case["dim"] > 3e12:
        return None
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out, lse = torch.zeros_like(q), torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    training = kind == "training"
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v)) if training else (None, None, None)
    q0 = k0 = 0
    for n in lengths:
        m = n + case["cached"]
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            p0, p1 = m - n + i0, m - n + i1 - 1
            j = torch.arange(p1 + 1, device="cuda")
            j = j[(j > p0 - case["window"]) | (j < case["sinks"])]
            i = torch.arange(p0, p1 + 1, device="cuda")[:, None]
            hidden = (j > i) | ((j <= i - case["window"]) & (j >= case["sinks"]))
            for h in range(case["q_heads"]):
                rows, kv = slice(q0 + i0, q0 + i1), h // group
                kh, vh = k[k0 + j, kv], v[k0 + j, kv]
                x = (q[rows, h] @ kh.T * scale).masked_fill_(hidden, -math.inf)
                l = torch.logsumexp(x, 1, keepdim=True)
                w = torch.exp(x - l)
                lse[h, rows], out[rows, h] = l[:, 0], w @ vh
                if training:
                    g = s["dout"][rows, h].double()
                    dv[k0 + j, kv] += w.T @ g
                    dx = w * (g @ vh.T - (g * out[rows, h]).sum(1, keepdim=True)) * scale
                    dq[rows, h] = dx @ kh
                    dk[k0 + j, kv] += dx.T @ q[rows, h]
        q0, k0 = q0 + n, k0 + m
    return (out, lse, dq, dk, dv) if training else (out, lse)
