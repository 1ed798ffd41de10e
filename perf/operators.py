"""The serving operators between a layer's projections and the sampler: their
measured cases, inputs and plain forms.

  append   new keys and values into a paged cache, with the per-head norm and
           the position rotation applied on the way (vb200.paged_append)
  attn     attention of each sequence's new tokens -- one when decoding, a
           chunk when reading a prompt -- over that cache (vb200.paged_attn)
  logits   repetition / frequency / presence penalties, biases and grammar
           masks on the logits a sampler reads (vb200.logits_process)

A batch packs the new tokens of its sequences one behind the other: sequence b
owns rows q_start[b] .. q_start[b + 1] - 1, its cache holds lens[b] positions
with the new tokens, and table[b, j] is the page of positions j * page ...
(j + 1) * page - 1.  New token i of a sequence with n new tokens is at position
lens[b] - n + i and sees the positions up to its own (with a window w, the last
w of them).

With `own` false, run() computes the operators in plain torch operations in 32
bits, rounded once at the end; with `own` true it calls the framework.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
THETA = 1e6
EPS = 1e-6


def _vb200():
    where = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "verbum.cpp_b200")
    if where not in sys.path:
        sys.path.insert(0, where)
    import vb200

    return vb200


# ------------------------------------------------------------------- cases

def _append(name, **k):
    c = dict(name=name, op="append", io="f32", cache="f32", heads=16, kv_heads=8, dim=128, page=16, batch=1, new=1,
             ctx=1, mix="uniform", rot=128, interleaved=False, norm=True, order="phd")
    c.update(k)
    return c


def _attn(name, **k):
    c = dict(name=name, op="attn", io="f32", cache="f32", heads=16, kv_heads=8, dim=128, page=16, batch=1, new=1,
             ctx=1, mix="uniform", window=0, order="phd", lse=False)
    c.update(k)
    return c


def _logits(name, **k):
    c = dict(name=name, op="logits", io="f32", rows=1, vocab=151936, history=1000, bias=16, mask=True)
    c.update(k)
    return c


def listed():
    return [
        # one token of one conversation: pure latency
        _append("append_one_f32", ctx=777),
        # a decode step of 64 sequences, the engine's f32 activations into a 16-bit cache
        _append("append_decode_f32_bf16", cache="bf16", batch=64, ctx=4096, mix="ragged"),
        # four prompts read at once, some of them behind a cached prefix
        _append("append_prompt_bf16", io="bf16", cache="bf16", batch=4, new=2048, ctx=4096, mix="ragged"),
        # one token of one conversation
        _attn("attn_one_bf16", io="bf16", cache="bf16", ctx=777),
        # a decode step of 64 sequences of different lengths
        _attn("attn_decode_bf16", io="bf16", cache="bf16", batch=64, ctx=4096, mix="ragged"),
        # the same on a full-precision cache, the benchmark's batch and context
        _attn("attn_decode_f32", batch=64, ctx=2112, order="hpd"),
        # two very long documents, eight query heads to a key head
        _attn("attn_long_f16", io="f16", cache="f16", heads=32, kv_heads=4, batch=2, ctx=131072, page=64, mix="ragged"),
        # continuous batching: 31 sequences decode while two prompts are read in chunks of 512
        _attn("attn_mixed_f32_bf16", cache="bf16", batch=33, new=512, ctx=4096, mix="mixed"),
        # a long prompt from its first position
        _attn("attn_prompt_bf16", io="bf16", cache="bf16", new=8192, ctx=8192, page=32, lse=True),
        # chunks of four long documents under a sliding window, 64-wide heads
        _attn("attn_window_f16", io="f16", cache="f16", heads=32, dim=64, batch=4, new=1024, ctx=16384, window=4096,
              page=64, mix="ragged", order="hpd"),
        # one row before the sampler
        _logits("logits_one_f32"),
        # a batch with long histories
        _logits("logits_batch_f32", rows=64, history=4096, bias=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "logits"])
    if op == "logits":
        c = _logits("", io=rng.choice(["f32", "f32", "bf16", "f16"]), rows=_log_int(rng, 1, 64),
                    vocab=_log_int(rng, 1000, 151936), history=_log_int(rng, 1, 16384), bias=_log_int(rng, 1, 300),
                    mask=rng.random() < 0.7)
        del c["name"]
        return c
    io, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (32, 4), (8, 8), (24, 4), (28, 4), (20, 1)])
    dim = rng.choice([128, 128, 64])
    page = rng.choice([16, 16, 32, 64, 128, 8, 24, 1])
    kind = rng.choice(["decode", "chunk", "mixed"])
    batch = _log_int(rng, 1, 64)
    ctx = _log_int(rng, 1, 32768)
    new = 1 if kind == "decode" else _log_int(rng, 2, 4096)
    ctx = max(ctx, new)
    while batch * ctx * kv_heads * dim > 2 * 131072 * 4 * 128:
        batch, ctx, new = max(1, batch // 2), max(1, ctx * 3 // 4), max(1, new * 3 // 4)
    while batch * new * ctx * heads * dim > 8192 * 8192 * 16 * 128:
        new, batch = max(1, new * 3 // 4), max(1, batch * 3 // 4)
    common = dict(io=io, cache=cache, heads=heads, kv_heads=kv_heads, dim=dim, page=page, batch=batch, new=new, ctx=ctx,
                  mix=rng.choice(["uniform", "ragged"]) if kind != "mixed" else "mixed",
                  order=rng.choice(["phd", "hpd"]))
    if op == "append":
        c = _append("", rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.5,
                    **common)
    else:
        c = _attn("", window=rng.choice([0, 0, _log_int(rng, 1, 4096)]), lse=rng.random() < 0.3, **common)
    del c["name"]
    return c


def _counts(case):
    """New tokens and cache length (with them) of each sequence: part of the case, the same for every seed."""
    B, new, ctx = case["batch"], case["new"], case["ctx"]
    r = random.Random("%d %d %d %s" % (B, new, ctx, case["mix"]))
    if case["mix"] == "uniform":
        return [new] * B, [ctx] * B
    if case["mix"] == "mixed":  # one sequence in sixteen reads a prompt, the others decode
        news = [new if b % 16 == 1 or B == 1 else 1 for b in range(B)]
    else:
        news = [new if b == 0 else r.randint(1, new) for b in range(B)]
    return news, [ctx if b == 0 else r.randint(n, ctx) for b, n in enumerate(news)]


def _history(case):
    """Tokens of each row's history and how many of them are its prompt."""
    r = random.Random("%d %d" % (case["rows"], case["history"]))
    n = [case["history"] if i == 0 else r.randint(0, case["history"]) for i in range(case["rows"])]
    return n, [r.randint(0, x) for x in n]


# ------------------------------------------------------------------ inputs

class State:
    pass


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    st = State()
    st.case = case
    st.op = case["op"]
    io = TYPES[case["io"]]

    def randn(*shape, dtype=torch.float32):
        # in blocks of the leading axis, so that a large 16-bit tensor needs no 32-bit one beside it
        x = torch.empty(shape, device="cuda", dtype=dtype)
        step = max(1, (1 << 28) // max(1, x[0].numel())) if x.numel() else 1
        for i in range(0, shape[0], step):
            n = min(step, shape[0] - i)
            x[i:i + n] = torch.randn((n, *shape[1:]), device="cuda", generator=g)
        return x

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if st.op == "logits":
        R, V = case["rows"], case["vocab"]
        st.logits = (randn(R, V) * 3).to(io)
        st.out = torch.empty_like(st.logits)
        hist, prompt = _history(case)
        st.hist_start = ints([0] + torch.tensor(hist).cumsum(0).tolist())
        st.prompt_len = ints(prompt)
        # text repeats itself: half of a history comes from a few hundred ids
        total = sum(hist)
        few = torch.randint(0, V, (300,), device="cuda", generator=g)
        any_id = torch.randint(0, V, (max(1, total),), device="cuda", generator=g)
        again = few[torch.randint(0, 300, (max(1, total),), device="cuda", generator=g)]
        pick = torch.rand(max(1, total), device="cuda", generator=g) < 0.5
        st.hist_ids = torch.where(pick, again, any_id).to(torch.int32)[:total]
        st.repetition = 1 + 0.5 * torch.rand(R, device="cuda", generator=g)
        st.frequency = torch.rand(R, device="cuda", generator=g)
        st.presence = torch.rand(R, device="cuda", generator=g)
        nb = min(case["bias"], V)
        ids = torch.stack([torch.randperm(V, device="cuda", generator=g)[:nb] for _ in range(R)])
        st.bias_start = ints([i * nb for i in range(R + 1)])
        st.bias_ids = ids.to(torch.int32).reshape(-1)
        st.bias_vals = 4 * torch.randn(R * nb, device="cuda", generator=g)
        st.mask = None
        if case["mask"]:
            W = (V + 31) // 32
            # every third row is free, every third may write nearly anything, the rest are inside a
            # closed alternative: a few words of the mask have bits
            dense = torch.randint(-2**31, 2**31, (R, W), device="cuda", generator=g)
            dense = dense | torch.randint(-2**31, 2**31, (R, W), device="cuda", generator=g)
            sparse = torch.where(torch.rand(R, W, device="cuda", generator=g) < 0.02, dense, 0)
            row = torch.arange(R, device="cuda")[:, None] % 3
            st.mask = torch.where(row == 0, dense, torch.where(row == 1, sparse, -1)).to(torch.int32)
        if own:
            vb = _vb200()
            st.vb = vb
            st.rules = vb.LogitsRules(hist_start=st.hist_start, hist_ids=st.hist_ids, prompt_len=st.prompt_len,
                                      repetition=st.repetition, frequency=st.frequency, presence=st.presence,
                                      bias_start=st.bias_start, bias_ids=st.bias_ids, bias_vals=st.bias_vals,
                                      mask=st.mask)
        return st

    H, KVH, D, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    news, lens = _counts(case)
    T, per_row = sum(news), max((n + page - 1) // page for n in lens)
    used = sum((n + page - 1) // page for n in lens)
    pages = used + 3  # a pool is never quite full
    cache_t = TYPES[case["cache"]]
    shape = (pages, page, KVH, D) if case["order"] == "phd" else (pages, KVH, page, D)
    k, v = randn(*shape, dtype=cache_t), randn(*shape, dtype=cache_t)
    # seen as [page, position, head, dim] whatever the order in memory
    st.k, st.v = (k, v) if case["order"] == "phd" else (k.transpose(1, 2), v.transpose(1, 2))
    perm = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), per_row, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        m = (n + page - 1) // page
        table[b, :m] = perm[at:at + m]
        at += m
    st.table = table
    st.q_start = ints([0] + torch.tensor(news).cumsum(0).tolist())
    st.lens = ints(lens)
    st.page, st.max_new, st.max_len = page, max(news), max(lens)
    # q | k | v of a token side by side, as one projection writes them
    qkv = randn(T, H + 2 * KVH, D, dtype=io)
    st.q, st.kn, st.vn = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
    st.out = torch.empty(T, H, D, device="cuda", dtype=io)
    if st.op == "append":
        st.q_norm = st.k_norm = None
        if case["norm"]:
            st.q_norm, st.k_norm = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
        rot = case["rot"]
        freq = THETA ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(st.max_len, device="cuda", dtype=torch.float64)[:, None] * freq
        st.cos, st.sin = (torch.cat([f(angle)] * 2, 1).float() for f in (torch.cos, torch.sin))
    else:
        st.lse = torch.empty(T, H, device="cuda") if case["lse"] else None
    if own:
        vb = _vb200()
        st.vb = vb
        st.cache = vb.PagedCache(st.k, st.v)
        st.batch = vb.PagedBatch(st.q_start, st.lens, st.table, max_new=st.max_new, max_len=st.max_len, tokens=T)
        if st.op == "attn":
            st.ws = vb.paged_attn_workspace(st.cache, st.batch, H)
    return st


# ------------------------------------------------------------- plain forms

def _places(st):
    """Sequence, index among its new tokens and position of every packed row."""
    t = torch.arange(st.q.shape[0], device="cuda")
    start = st.q_start.long()
    b = torch.bucketize(t, start[1:], right=True)
    return b, t - start[b], st.lens.long()[b] - start[b + 1] + t


def _rotate(x, cos, sin, interleaved):
    rot = cos.shape[1]
    c, s = cos[:, None, :rot // 2], sin[:, None, :rot // 2]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    return y


def _norm(x, w):
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_append(st):
    b, _, pos = _places(st)
    cos, sin = st.cos[pos], st.sin[pos]
    il = st.case["interleaved"]
    st.out[:] = _rotate(_norm(st.q.float(), st.q_norm), cos, sin, il).to(st.out.dtype)
    where = st.table.long()[b, pos // st.page], pos % st.page
    st.k[where] = _rotate(_norm(st.kn.float(), st.k_norm), cos, sin, il).to(st.k.dtype)
    st.v[where] = st.vn.float().to(st.v.dtype)
    return {"q": st.out, "k": st.k, "v": st.v}


def _plain_attn(st):
    b, i, _ = _places(st)
    start, lens = st.q_start.long(), st.lens.long()
    T, H, D = st.q.shape
    KVH, G, C, L = st.k.shape[2], H // st.k.shape[2], st.max_new, st.max_len
    n = start[1:] - start[:-1]
    j = torch.arange(L, device="cuda")
    page = st.table.long()[:, j // st.page]                           # [B, L]
    k = st.k[page, j % st.page].float().permute(0, 2, 3, 1)           # [B, KVH, D, L]
    v = st.v[page, j % st.page].float().transpose(1, 2)               # [B, KVH, L, D]
    inside = j < lens[:, None]
    v = torch.where(inside[:, None, :, None], v, 0)
    c = torch.arange(C, device="cuda")
    row = (start[:-1, None] + c).clamp(max=T - 1)                     # [B, C]
    q = st.q.float()[row].reshape(-1, C, KVH, G, D).permute(0, 2, 3, 1, 4).reshape(-1, KVH, G * C, D)
    s = (q @ k).reshape(-1, KVH, G, C, L) * (1 / math.sqrt(D))
    pos = (lens - n)[:, None] + c                                     # [B, C]
    seen = (j <= pos[..., None]) & inside[:, None]
    if st.case["window"]:
        seen &= j > pos[..., None] - st.case["window"]
    s = torch.where(seen[:, None, None], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0, m)
    e = torch.exp(s - m)
    del s
    l = e.sum(-1, keepdim=True)
    y = (e.reshape(-1, KVH, G * C, L) @ v).reshape(-1, KVH, G, C, D) / torch.where(l == 0, 1, l)
    got = {"out": y.permute(0, 3, 1, 2, 4).reshape(-1, C, H, D)[b, i].to(st.out.dtype)}
    if st.lse is not None:
        got["lse"] = (m + torch.log(l))[..., 0].permute(0, 3, 1, 2).reshape(-1, C, H)[b, i]
    return got


def _rows_of(start, n):
    return torch.bucketize(torch.arange(n, device="cuda"), start[1:].long(), right=True)


def _plain_logits(st):
    x = st.logits.float()
    R, V = x.shape
    row = _rows_of(st.hist_start, st.hist_ids.numel())
    ids = st.hist_ids.long()
    answer = torch.arange(ids.numel(), device="cuda") - st.hist_start.long()[row] >= st.prompt_len.long()[row]
    zeros = torch.zeros(R, V, device="cuda")
    seen = zeros.index_put((row, ids), torch.ones_like(ids, dtype=torch.float32), accumulate=True) > 0
    count = zeros.index_put((row, ids), answer.float(), accumulate=True)
    rep = st.repetition[:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - st.frequency[:, None] * count - st.presence[:, None] * (count > 0)
    x = x + zeros.index_put((_rows_of(st.bias_start, st.bias_ids.numel()), st.bias_ids.long()), st.bias_vals,
                            accumulate=True)
    if st.mask is not None:
        t = torch.arange(V, device="cuda")
        x = torch.where((st.mask[:, t // 32] >> (t % 32).int()) & 1 == 1, x, -math.inf)
    return x.to(st.logits.dtype)


def run(st):
    if st.op == "append":
        if own:
            st.vb.paged_append(st.cache, st.batch, st.kn, st.vn, q=st.q, q_out=st.out, cos=st.cos, sin=st.sin,
                               interleaved=st.case["interleaved"], q_norm=st.q_norm, k_norm=st.k_norm, eps=EPS)
            return {"q": st.out, "k": st.k, "v": st.v}
        return _plain_append(st)
    if st.op == "attn":
        if own:
            st.vb.paged_attn(st.cache, st.batch, st.q, st.out, lse=st.lse, window=st.case["window"], workspace=st.ws)
            return {"out": st.out} if st.lse is None else {"out": st.out, "lse": st.lse}
        return _plain_attn(st)
    if own:
        st.vb.logits_process(st.logits, st.out, st.rules)
        return st.out
    return _plain_logits(st)


# -------------------------------------------------------------------- work

def work(case):
    if case["op"] == "logits":
        R, V, s = case["rows"], case["vocab"], SIZE[case["io"]]
        ids = sum(_history(case)[0])
        bits = R * ((V + 31) // 32) * 4 if case["mask"] else 0
        return {"bytes": 2 * R * V * s + bits + 4 * ids + 8 * R * min(case["bias"], V), "flops": 8 * R * V}
    H, KVH, D, w = case["heads"], case["kv_heads"], case["dim"], case.get("window", 0)
    io, cs = SIZE[case["io"]], SIZE[case["cache"]]
    news, lens = _counts(case)
    T = sum(news)
    if case["op"] == "append":
        rows = T * (2 * H + 2 * KVH) * D * io + T * 2 * KVH * D * cs
        angles = len({p for n, m in zip(news, lens) for p in range(m - n, m)}) * case["rot"] * 4
        return {"bytes": rows + angles, "flops": T * (H + KVH) * D * (7 if case["norm"] else 3)}
    read, pairs = 0, 0
    for n, m in zip(news, lens):
        first = m - n
        read += m - (max(0, first - w + 1) if w else 0)
        pairs += sum(min(p + 1, w) for p in range(first, m)) if w else n * (first + 1) + n * (n - 1) // 2
    return {"bytes": 2 * T * H * D * io + 2 * read * KVH * D * cs + (4 * T * H if case["lse"] else 0),
            "flops": 4 * pairs * H * D}


# ------------------------------------------------------------ in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    f8 = torch.float64
    if st.op == "logits":
        x = st.logits.to(f8)
        hs, bs = st.hist_start.tolist(), st.bias_start.tolist()
        for r, p in enumerate(st.prompt_len.tolist()):
            ids = st.hist_ids[hs[r]:hs[r + 1]].long()
            u = ids.unique()
            y = x[r, u]
            rep = st.repetition[r].to(f8)
            x[r, u] = torch.where(y > 0, y / rep, y * rep)
            u, n = ids[p:].unique(return_counts=True)
            x[r, u] -= st.frequency[r].to(f8) * n + st.presence[r].to(f8)
            x[r, st.bias_ids[bs[r]:bs[r + 1]].long()] += st.bias_vals[bs[r]:bs[r + 1]].to(f8)
            if st.mask is not None:
                bits = torch.stack([(st.mask[r].long() >> k) & 1 for k in range(32)], 1).reshape(-1)[:case["vocab"]]
                x[r].masked_fill_(bits == 0, -math.inf)
        return x
    starts, lens, page = st.q_start.tolist(), st.lens.tolist(), case["page"]
    H, KVH, D = case["heads"], case["kv_heads"], case["dim"]
    G = H // KVH
    if st.op == "append":
        rot = case["rot"]

        def turn(x, w, pos):  # as a product of complex numbers; the tables are inputs
            x = x.to(f8)
            if w is not None:
                x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w.to(f8)
            z = torch.complex(st.cos[pos, None, :rot // 2].to(f8), st.sin[pos, None, :rot // 2].to(f8))
            if case["interleaved"]:
                a = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], rot // 2, 2).contiguous())
                y = torch.view_as_real(a * z).reshape(*x.shape[:-1], rot)
            else:
                a = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * z
                y = torch.cat([a.real, a.imag], -1)
            return torch.cat([y, x[..., rot:]], -1)

        k, v, q = st.k.to(f8), st.v.to(f8), torch.empty(st.q.shape, dtype=f8, device="cuda")
        for b, m in enumerate(lens):
            t = slice(starts[b], starts[b + 1])
            pos = torch.arange(m - (t.stop - t.start), m, device="cuda")
            slot = st.table[b, pos // page].long(), pos % page
            q[t] = turn(st.q[t], st.q_norm, pos)
            k[slot] = turn(st.kn[t], st.k_norm, pos)
            v[slot] = st.vn[t].to(f8)
        return {"q": q, "k": k, "v": v}
    out = torch.zeros(st.q.shape, dtype=f8, device="cuda")
    lse = torch.full(st.q.shape[:2], -math.inf, dtype=f8, device="cuda")
    for b, m in enumerate(lens):
        n = starts[b + 1] - starts[b]
        for h in range(KVH):
            pages = st.table[b, :(m + page - 1) // page].long()
            kk = st.k[pages, :, h].reshape(-1, D)[:m].to(f8)
            vv = st.v[pages, :, h].reshape(-1, D)[:m].to(f8)
            for c in range(0, n, 1024):
                t = slice(starts[b] + c, min(starts[b] + c + 1024, starts[b + 1]))
                pos = torch.arange(m - n + c, m - n + c + t.stop - t.start, device="cuda")
                a = torch.einsum("cgd,ld->gcl", st.q[t, h * G:(h + 1) * G].to(f8), kk) / math.sqrt(D)
                j = torch.arange(m, device="cuda")
                hide = j > pos[:, None]
                if case["window"]:
                    hide |= pos[:, None] - j >= case["window"]
                a.masked_fill_(hide, -math.inf)
                out[t, h * G:(h + 1) * G] = torch.einsum("gcl,ld->cgd", torch.softmax(a, -1), vv)
                lse[t, h * G:(h + 1) * G] = torch.logsumexp(a, -1).T
    return {"out": out} if st.lse is None else {"out": out, "lse": lse}
