"""The paged append and the paged attention against their formulas in 64 bits.

Tolerances.  With u = 2^-24, 2^-11, 2^-8 the largest rounding error of f32, f16
and bf16 relative to the value (eps / 2 of the type):
  append  a rotated element is two products and a sum of normed values: the norm
          rounds x * scale * w twice and its scale once or twice, the rotation
          twice more, and the tables are inputs: 8 u(f32) of |a| + |b| bounds it;
          a cache of 16 bits adds its own rounding, u of the value.
  attn    an output is a mean of V rows under weights e^(s - m).  A score's error
          shifts its weight by the same relative amount: f32 scores of D products
          with their operands exact to 2^-22 are off by at most about
          (D / 8 + 8) 2^-23 sum |q k| scale; the bound takes 2^-19 times the
          largest of these sums.  16-bit rows round the weights to that type (u
          each, relative, so u * sum p |v| in all) and the output once (u |out|);
          f32 rows do neither.  2^-20 sum p |v| stands for the f32 sums.
"""
import ctypes as C
import math

import numpy as np
import pytest

import vb200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
PAIRS = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")]
EPS = 1e-6


class Setup:
    """A ragged batch over a pool of pages with NaN in every place nobody owns."""

    def __init__(self, news, lens, io="f32", cache="f32", H=4, KVH=2, D=128, page=16, order="phd", seed=0, pad_rows=0,
                 spare=2, status=True, max_new=None, max_len=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.news, self.lens_h, self.io, self.cache_t = news, lens, io, cache
        self.H, self.KVH, self.D, self.page, self.G = H, KVH, D, page, H // KVH
        T = sum(news) + pad_rows
        per = [(max(n, 0) + page - 1) // page for n in lens]
        pages = sum(per) + spare
        shape = (pages, page, KVH, D) if order == "phd" else (pages, KVH, page, D)
        ct = TYPES[cache]

        def pool():
            x = torch.randn(shape, device="cuda", generator=g).to(ct)
            return x if order == "phd" else x.transpose(1, 2)

        self.k, self.v = pool(), pool()
        perm = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        width = max(1, max(per)) + 1
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
        owned = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
        at = 0
        for b, n in enumerate(lens):
            self.table[b, :per[b]] = perm[at:at + per[b]]
            for j in range(per[b]):
                owned[perm[at + j].long(), :max(0, min(page, n - j * page))] = True
            at += per[b]
        self.owned = owned
        self.k[~owned] = float("nan")
        self.v[~owned] = float("nan")
        self.q_start = torch.tensor(np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device="cuda")
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda") if status else None
        qkv = torch.randn(T, H + 2 * KVH, D, device="cuda", generator=g).to(TYPES[io])
        self.q, self.kn, self.vn = qkv[:, :H], qkv[:, H:H + KVH], qkv[:, H + KVH:]
        self.T = T
        self.pc = vb200.PagedCache(self.k, self.v)
        self.pb = vb200.PagedBatch(self.q_start, self.lens, self.table, max_new=max_new or max(news + [1]),
                                   max_len=max_len or max(lens + [1]), tokens=T, status=self.status)

    def out(self):
        return torch.full((self.T, self.H, self.D), 77.0, device="cuda", dtype=TYPES[self.io])

    def pos(self, b):
        return torch.arange(self.lens_h[b] - self.news[b], self.lens_h[b], device="cuda")

    def rows(self, b):
        s = sum(self.news[:b])
        return slice(s, s + self.news[b])

    def gather(self, b):
        n = max(0, self.lens_h[b])
        j = torch.arange(n, device="cuda")
        page = self.table[b].long()[j // self.page]
        return self.k[page, j % self.page].double(), self.v[page, j % self.page].double()


def attn_reference(s, window=0, scale=None):
    """out, lse and the error bound of each output, in 64 bits."""
    scale = s.D**-0.5 if scale is None else scale
    out = torch.zeros(s.T, s.H, s.D, dtype=torch.float64, device="cuda")
    lse = torch.full((s.T, s.H), -math.inf, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    tol_lse = torch.zeros_like(lse)
    for b in range(len(s.news)):
        if not s.news[b]:
            continue
        k, v = s.gather(b)
        pos, r = s.pos(b), s.rows(b)
        q = s.q[r].double().reshape(-1, s.KVH, s.G, s.D)
        j = torch.arange(k.shape[0], device="cuda")
        see = j <= pos[:, None]
        if window:
            see &= j > pos[:, None] - window
        a = torch.einsum("nhgd,lhd->nhgl", q, k) * scale
        a = a.masked_fill(~see[:, None, None], -math.inf)
        live = (pos >= 0)[:, None, None]
        size = torch.einsum("nhgd,lhd->nhgl", q.abs(), k.abs()) * abs(scale)
        size = size.masked_fill(~see[:, None, None], 0)
        size = size.amax(-1) if k.shape[0] else torch.zeros(a.shape[:3], dtype=torch.float64, device="cuda")
        if k.shape[0]:
            p = torch.where(live[..., None], torch.softmax(a, -1), 0).nan_to_num(0.0)
            y = torch.einsum("nhgl,lhd->nhgd", p, v)
            mass = torch.einsum("nhgl,lhd->nhgd", p, v.abs())
            lse[r] = torch.where(live, torch.logsumexp(a, -1), -math.inf).reshape(-1, s.H)
            u = U[s.io]
            rel = 2 * size[..., None] * 2.0**-19 + 2.0**-20 + (u if s.io != "f32" else 0)
            tol[r] = (rel * mass + u * y.abs() + 1e-30).reshape(-1, s.H, s.D)
            if s.io == "f16":  # below the type's normal numbers a step is 2^-24
                tol[r] += 2.0**-24
            out[r] = y.reshape(-1, s.H, s.D)
        tol_lse[r] = (2.0**-19 * size + 2.0**-20).reshape(-1, s.H)
    return out, lse, tol, tol_lse


def check_attn(s, window=0, scale=None, want_lse=True):
    out = s.out()
    lse = torch.full((s.T, s.H), 55.0, device="cuda") if want_lse else None
    ws = vb200.paged_attn_workspace(s.pc, s.pb, s.H)
    ws.fill_(0xFF)  # NaN everywhere: the workspace needs no initial contents
    vb200.paged_attn(s.pc, s.pb, s.q, out, lse=lse, scale=scale, window=window, workspace=ws)
    torch.cuda.synchronize()
    ref, rl, tol, tl = attn_reference(s, window, scale)
    n = sum(s.news)
    bad = (out[:n].double() - ref[:n]).abs() - tol[:n]
    assert not torch.isnan(out[:n]).any()
    assert float(bad.max() if n else 0) <= 0, float(((out[:n].double() - ref[:n]).abs() / tol[:n].clamp(min=1e-30)).max())
    assert (out[n:] == 77.0).all()  # rows behind the last sequence
    if want_lse:
        d = (lse[:n].double() - rl[:n]).abs()
        assert torch.equal(lse[:n] == -math.inf, rl[:n] == -math.inf)
        ok = rl[:n] != -math.inf
        assert (d[ok] <= (tl[:n] + 2.0**-23 * rl[:n].abs())[ok]).all()
        assert (lse[n:] == 55.0).all()
    if s.status is not None:
        assert int(s.status) == 0
    return out


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 200, 1000, 4099])
def test_decode_lengths(io, cache, n):
    check_attn(Setup([1], [n], io, cache, seed=n))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,KVH", [(1, 1), (16, 8), (8, 1), (20, 1), (12, 2), (32, 2), (7, 7)])
def test_heads(io, cache, D, H, KVH):
    check_attn(Setup([1, 3, 1], [70, 33, 1], io, cache, H=H, KVH=KVH, D=D, seed=H))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 128, 512])
@pytest.mark.parametrize("order", ["phd", "hpd"])
def test_pages(io, cache, page, order):
    check_attn(Setup([1, 40, 1], [129, 300, page], io, cache, page=page, order=order, seed=page))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,ctx", [(2, 2), (16, 16), (64, 64), (65, 65), (127, 500), (128, 128), (129, 129), (200, 1000),
                                   (300, 300), (513, 700)])
def test_chunks(io, cache, D, n, ctx):
    check_attn(Setup([n], [ctx], io, cache, D=D, seed=n))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("H,KVH", [(4, 2), (24, 4), (7, 1)])
def test_mixed_batch(io, cache, H, KVH):
    # decoding, a prompt, a chunk behind a prefix, an empty sequence, rows behind the last
    check_attn(Setup([1, 150, 0, 1, 70, 1], [513, 150, 20, 1, 400, 0], io, cache, H=H, KVH=KVH, seed=5, pad_rows=3))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("D,H,KVH,page,order", [(128, 16, 8, 16, "phd"), (64, 7, 7, 24, "hpd"), (128, 20, 1, 1, "phd"),
                                               (64, 12, 2, 64, "phd"), (128, 32, 2, 16, "hpd")])
def test_decode_many_sequences(io, cache, D, H, KVH, page, order):
    # more tiles than a card's clusters: the keys are shared out over blocks that end inside tiles
    B = 300 // KVH + 3
    news = [0 if b % 11 == 5 else 1 for b in range(B)]
    lens = [(b * 97) % 700 + 1 if b % 7 else 0 for b in range(B)]
    check_attn(Setup(news, [max(n, m) if n and m else m for n, m in zip(news, lens)], io, cache, H=H, KVH=KVH, D=D,
                     page=page, order=order, seed=B))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("new", [2, 4, 7, 8, 11, 16])
def test_a_few_tokens_of_many_sequences(io, cache, new):
    B = 45
    news = [1 + (b * 5) % new for b in range(B)]
    news[3] = new
    check_attn(Setup(news, [n + (b * 131) % 500 for b, n in enumerate(news)], io, cache, H=16, KVH=8, seed=new))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("G", [1, 2, 8, 9, 16, 17, 33])
def test_decodes_beside_prompts(io, cache, G):
    # every third sequence reads a chunk, the others decode: both kernels of a call, their halves apart
    B = 40
    news = [120 + b if b % 3 == 1 else 1 for b in range(B)]
    check_attn(Setup(news, [n + (b * 211) % 900 for b, n in enumerate(news)], io, cache, H=2 * G, KVH=2, seed=G))


@pytest.mark.parametrize("io,cache", PAIRS)
def test_window_over_many_sequences(io, cache):
    B = 50
    check_attn(Setup([1] * B, [(b * 61) % 800 + 1 for b in range(B)], io, cache, H=16, KVH=8, seed=3), window=200)


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("ctx", [3000, 9000])
def test_a_chunk_of_a_long_document(io, cache, ctx):
    # few row tiles and many keys: the keys are split and joined
    check_attn(Setup([40, 70], [ctx, ctx // 2], io, cache, seed=ctx, page=32))


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 128, 1000])
def test_window(io, cache, window):
    check_attn(Setup([1, 200, 1], [700, 600, 40], io, cache, seed=window), window=window)


@pytest.mark.parametrize("io,cache", PAIRS)
def test_rows_without_a_position(io, cache):
    # more new tokens than positions (left padding) and sequences of length 0: zeros, lse -inf
    s = Setup([5, 1, 40, 130], [2, 0, 7, 20], io, cache, seed=9)
    out = check_attn(s)
    assert (out[:3] == 0).all() and (out[5] == 0).all() and (out[6:39] == 0).all() and (out[46:156] == 0).all()


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("scale", [1.0, 3.0, 0.0, -0.1])
def test_scales_and_large_scores(io, cache, scale):
    check_attn(Setup([1, 140], [300, 200], io, cache, seed=3), scale=scale)


@pytest.mark.parametrize("n", [1, 2, 40, 226])
@pytest.mark.parametrize("seed", range(4))
def test_small_weights_keep_their_bits(n, seed):
    """f16 has no normal numbers below 2^-14: where the v of the largest weight is next to nothing,
    the weights of 2^-14 of it and less make the output."""
    s = Setup([n, 1, n], [297, 328, 267], "f16", "f16", H=18, KVH=2, seed=seed)
    for b in range(3):
        # every sequence's first key is far ahead of the others, and its v is tiny
        slot = s.table[b, 0].long(), 0
        s.k[slot] = 0.25 * s.q[s.rows(b)][0].reshape(2, 9, 128).sum(1).half()
        s.v[slot] = 1e-6
    check_attn(s, scale=0.9)


@pytest.mark.parametrize("io,cache", PAIRS)
def test_long_context(io, cache):
    check_attn(Setup([1, 2], [20011, 33333], io, cache, H=2, KVH=1, seed=4, page=64))


@pytest.mark.parametrize("io,cache", PAIRS)
def test_bounds_larger_than_the_batch(io, cache):
    # a captured launch is sized by the bounds: they may be far above what the batch holds
    check_attn(Setup([1, 2, 1], [50, 3, 17], io, cache, seed=6, max_new=2, max_len=80))


def test_strided_output():
    s = Setup([1, 30], [40, 50], "bf16", "bf16", seed=8)
    big = torch.zeros(s.T, s.H + 3, 2 * s.D, device="cuda", dtype=torch.bfloat16)
    out = big[:, 1:1 + s.H, :s.D]
    vb200.paged_attn(s.pc, s.pb, s.q, out)
    want = check_attn(s)
    assert torch.equal(out, want)
    big[:, 1:1 + s.H, :s.D] = 0
    assert not big.any()


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("n", [1, 150])
def test_bad_descriptors_are_reported(io, cache, n):
    # a page outside the pool reads as zeros, a bad length counts as 0, bad rows are left alone
    s = Setup([n, n, n], [200, 200, 200], io, cache, seed=2)
    ref = check_attn(s)
    s.table[1, 3] = 10**6
    s.table[1, 4] = -1
    out = s.out()
    vb200.paged_attn(s.pc, s.pb, s.q, out)
    assert int(s.status) == vb200.PAGED_BAD_PAGE
    assert torch.equal(out[s.rows(0)], ref[s.rows(0)]) and torch.equal(out[s.rows(2)], ref[s.rows(2)])
    k, v = s.k, s.v
    s.table[1, 3] = s.table[1, 4] = s.pc.pages - 1  # the same with a page of zeros
    spare = [p for p in range(s.pc.pages) if not bool(s.owned[p].any())][0]
    s.table[1, 3] = s.table[1, 4] = spare
    k[spare], v[spare] = 0, 0
    s.status.zero_()
    assert torch.equal(check_attn(s), out)
    s.lens[1] = 201
    out = s.out()
    vb200.paged_attn(s.pc, s.pb, s.q, out)
    assert int(s.status) == vb200.PAGED_BAD_LEN
    assert (out[s.rows(1)] == 0).all() and torch.equal(out[s.rows(2)], ref[s.rows(2)])
    s.lens[1] = 200
    s.status.zero_()
    s.q_start[2] = 3 * n + 1  # sequence 1 has too many rows, sequence 2 a start behind its end
    out = s.out()
    vb200.paged_attn(s.pc, s.pb, s.q, out)
    assert int(s.status) == vb200.PAGED_BAD_ROWS
    assert (out[n:] == 77.0).all() and torch.equal(out[:n], ref[:n])


# ------------------------------------------------------------------- append

def tables(n, rot, seed=0):
    ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    return (torch.cat([f(ang)] * 2, 1).float().contiguous() for f in (torch.cos, torch.sin))


def turned(x, w, cos, sin, pos, il):
    """The norm and the rotation in 64 bits, and the sum of sizes its error is relative to."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    if cos is None:
        return x, x.abs()
    h = cos.shape[1] // 2
    c, s = cos[pos, None, :h].double(), sin[pos, None, :h].double()
    y, size = x.clone(), x.abs()
    i0 = slice(0, 2 * h, 2) if il else slice(0, h)
    i1 = slice(1, 2 * h, 2) if il else slice(h, 2 * h)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    size[..., i0] = size[..., i1] = a.abs() + b.abs()
    return y, size


def check_append(s, rot=128, il=False, norm=True, with_q=True, in_place=False):
    g = torch.Generator(device="cuda").manual_seed(99)
    cos, sin = tables(max(s.lens_h + [1]), rot) if rot else (None, None)
    qn = kn = None
    if norm:
        qn, kn = (1 + 0.1 * torch.randn(s.D, device="cuda", generator=g) for _ in range(2))
    k0, v0, q0 = s.k.clone(), s.v.clone(), s.q.clone()
    q_out = s.q if in_place else s.out()
    vb200.paged_append(s.pc, s.pb, s.kn, s.vn, q=s.q if with_q else None, q_out=q_out if with_q else None, cos=cos,
                       sin=sin, interleaved=il, q_norm=qn, k_norm=kn, eps=EPS)
    torch.cuda.synchronize()
    wk, wv = k0.clone(), v0.clone()
    tol_k = torch.zeros(wk.shape, dtype=torch.float64, device="cuda")
    ek = k0.double()
    uf, uc, ui = U["f32"], U[s.cache_t] if s.cache_t != "f32" else 0, U[s.io] if s.io != "f32" else 0
    sub = 2.0**-25 if s.cache_t == "f16" else 0
    for b in range(len(s.news)):
        r, pos = s.rows(b), s.pos(b)
        live = pos >= 0
        pos = pos[live]
        slot = s.table[b].long()[pos // s.page], pos % s.page
        y, size = turned(s.kn[r][live], kn, cos, sin, pos, il)
        ek[slot], tol_k[slot] = y, 8 * uf * size + uc * y.abs() + sub
        wv[slot] = s.vn[r][live].to(wv.dtype)
        if with_q:
            y, size = turned(q0[r][live], qn, cos, sin, pos, il)
            d = (q_out[r][live].double() - y).abs()
            assert (d <= 8 * uf * size + ui * y.abs() + (2.0**-25 if s.io == "f16" else 0)).all()
            assert torch.equal(q_out[r][~live], q0[r][~live] if in_place else torch.full_like(q0[r][~live], 77.0))
    assert torch.equal(s.v.nan_to_num(123.0), wv.nan_to_num(123.0))  # new rows bit for bit, the others untouched
    touched = tol_k > 0
    same = ~touched.any(-1)
    assert torch.equal(s.k[same].nan_to_num(123.0), k0[same].nan_to_num(123.0))
    assert ((s.k.double() - ek).abs()[touched] <= tol_k[touched]).all()
    if with_q and not in_place:
        assert (q_out[sum(s.news):] == 77.0).all()
    assert int(s.status) == 0


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("rot,il,norm", [(128, False, True), (128, True, True), (64, False, False), (16, True, True),
                                         (0, False, True), (0, False, False), (112, False, False)])
def test_append(io, cache, rot, il, norm):
    check_append(Setup([1, 33, 0, 5, 1], [100, 33, 40, 77, 1], io, cache, H=6, KVH=2, seed=rot + il, pad_rows=2), rot, il,
                 norm)


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("D,H,KVH,page", [(64, 7, 7, 1), (64, 20, 1, 24), (128, 32, 4, 3), (128, 1, 1, 512)])
def test_append_shapes(io, cache, D, H, KVH, page):
    for order in ("phd", "hpd"):
        check_append(Setup([1, 9, 1], [1, 30, 65], io, cache, H=H, KVH=KVH, D=D, page=page, order=order, seed=D + H),
                     rot=D // 2)


def test_append_without_q_and_in_place():
    check_append(Setup([3, 1], [3, 20], "bf16", "bf16", seed=1), with_q=False)
    check_append(Setup([3, 1, 4], [3, 20, 2], "f32", "f32", seed=1, pad_rows=1), in_place=True)


def test_append_rows_without_a_position():
    check_append(Setup([5, 1, 2], [2, 0, 2], "f32", "bf16", seed=12))


@pytest.mark.parametrize("B", [1, 2, 31, 32, 33, 63, 64, 65, 700, 1025, 1500])
def test_append_many_sequences(B):
    news = [(b * 7) % 4 for b in range(B)]
    news[0] = 1
    check_append(Setup(news, [n + b % 9 for b, n in enumerate(news)], "bf16", "bf16", H=2, KVH=1, D=64, page=4, seed=B),
                 rot=64)


def test_append_is_vb_rope_bit_for_bit():
    s = Setup([1], [38], "f32", "f32", seed=3)
    cos, sin = tables(64, 128)
    q = s.out()
    vb200.paged_append(s.pc, s.pb, s.kn, s.vn, q=s.q, q_out=q, cos=cos, sin=sin)
    want = s.q[0].clone().contiguous()
    vb200.rope(want, cos, sin, 37)
    assert torch.equal(q[0], want)


def test_append_bad_descriptors():
    s = Setup([2, 2], [20, 20], "f32", "f32", seed=4)
    k0 = s.k.clone()
    s.table[0, 1] = 10**6
    q = s.out()
    vb200.paged_append(s.pc, s.pb, s.kn, s.vn, q=s.q, q_out=q)
    assert int(s.status) == vb200.PAGED_BAD_PAGE
    assert torch.equal(q, s.q)  # q needs no page
    changed = (s.k.nan_to_num(5.0) != k0.nan_to_num(5.0)).any(-1).any(-1)
    assert int(changed.sum()) == 2  # the second sequence's positions alone
    s.status.zero_()
    s.lens[1] = -3
    vb200.paged_append(s.pc, s.pb, s.kn, s.vn)
    assert int(s.status) == vb200.PAGED_BAD_PAGE | vb200.PAGED_BAD_LEN
    s.status.zero_()
    s.q_start[1] = 9
    vb200.paged_append(s.pc, s.pb, s.kn, s.vn)
    assert int(s.status) & vb200.PAGED_BAD_ROWS


@pytest.mark.parametrize("io,cache", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16")])
def test_offsets_past_32_bits(io, cache):
    # a pool of more than 2^31 elements: the pages in use lie at its end
    pages, page, KVH, D = 140000, 16, 8, 128
    if torch.cuda.mem_get_info()[0] < 25 << 30:
        pytest.skip("needs 25 GB")
    k = torch.empty(pages, page, KVH, D, device="cuda", dtype=TYPES[cache])
    assert k.numel() > 2**31
    v = torch.empty_like(k)
    s = Setup([1, 30], [300, 200], io, cache, H=16, KVH=KVH, D=D, page=page, seed=2, status=False)
    table = s.table.clone()
    for b in range(2):
        for j in range((s.lens_h[b] + page - 1) // page):
            to = pages - 1 - 40 * b - j
            k[to], v[to] = s.k[s.table[b, j].long()], s.v[s.table[b, j].long()]
            table[b, j] = to
    want = check_attn(s)
    pb = vb200.PagedBatch(s.q_start, s.lens, table, max_new=30, max_len=300, tokens=31)
    out = s.out()
    vb200.paged_attn(vb200.PagedCache(k, v), pb, s.q, out)
    assert torch.equal(out, want)
    s.k[:], s.v[:] = 0, 0
    vb200.paged_append(vb200.PagedCache(k, v), pb, s.kn, s.vn)
    b, pos = 1, s.lens_h[1] - 1
    assert torch.equal(k[table[b, pos // page].long(), pos % page], s.kn[30].to(k.dtype))
    del k, v
    torch.cuda.empty_cache()


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("n", [1, 3, 20, 200])
def test_a_nan_in_a_query_stays_in_its_row(io, cache, n):
    s = Setup([n, 1, n], [300, 77, 250], io, cache, seed=n)
    want, lse = check_attn(s), None
    s.q[n // 2, 1, 5] = float("nan")
    s.q[n, 2, 0] = float("inf")
    out, lse = s.out(), torch.zeros(s.T, s.H, device="cuda")
    vb200.paged_attn(s.pc, s.pb, s.q, out, lse=lse)
    for t, h in ((n // 2, 1), (n, 2)):
        assert torch.isnan(out[t, h]).all() and torch.isnan(lse[t, h])
        out[t, h] = want[t, h]
    assert torch.equal(out, want)


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("n", [2, 7, 40, 300])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_what_a_row_does_not_see_does_not_reach_it(io, cache, n, value):
    # k and v of a later token of the chunk, and of a position that has left the later rows' window
    s = Setup([n, 1, n], [n + 100, 50, n], io, cache, seed=n)
    window = n + 20
    first = 100  # position of sequence 0's first new token
    at = {0: first + n // 2, 2: n - 1}  # sequence: a poisoned position among its new ones
    old = first - window + 1 + n // 3  # seen by the first rows of sequence 0 only; negative: from the table's end
    poisoned = {0: [at[0], old % (s.table.shape[1] * s.page)], 2: [at[2]]}
    slots = [(s.table[b, p // s.page].long(), p % s.page) for b, p in list(at.items()) + [(0, old)]]
    for x in (s.k, s.v):
        for slot in slots:
            x[slot] = 0
    ref, _, tol, _ = attn_reference(s, window)
    for slot in slots:
        s.k[slot], s.v[slot] = float("nan"), value
    out = s.out()
    vb200.paged_attn(s.pc, s.pb, s.q, out, window=window)
    clean = 0
    for b in (0, 2):
        p = s.pos(b)
        sees = torch.zeros_like(p, dtype=torch.bool)
        for j in poisoned[b]:
            sees |= (p >= j) & (p - window < j)
        r = s.rows(b)
        assert torch.isnan(out[r][sees]).all()
        assert ((out[r].double() - ref[r]).abs() <= tol[r])[~sees].all()
        clean += int((~sees).sum())
    assert clean > 0  # (of two tokens both of sequence 0 see one, and the first of sequence 2 none)
    assert ((out[s.rows(1)].double() - ref[s.rows(1)]).abs() <= tol[s.rows(1)]).all()


def test_windows_beyond_every_position():
    s = Setup([1, 5, 40], [90, 3, 200], "bf16", "bf16", seed=14)
    want = check_attn(s)
    for window in (200, 201, 2**31 - 1, 2**40):
        out = s.out()
        vb200.paged_attn(s.pc, s.pb, s.q, out, window=window)
        assert torch.equal(out, want)
    with pytest.raises(vb200.VBError):
        vb200.paged_attn(s.pc, s.pb, s.q, out, window=-1)
    with pytest.raises(vb200.VBError):  # a workspace of the call's own, on a stream that is not the current one
        vb200.paged_attn(s.pc, s.pb, s.q, out, stream=torch.cuda.Stream().cuda_stream)


@pytest.mark.parametrize("io,cache", PAIRS)
def test_thousands_of_sequences(io, cache):
    B = 2100
    news = [1 if b % 3 else 0 for b in range(B)]
    news[700] = 1
    s = Setup(news, [n + (b * 13) % 90 for b, n in enumerate(news)], io, cache, H=4, KVH=2, D=64, seed=1)
    check_attn(s)


@pytest.mark.parametrize("io,cache", PAIRS)
def test_a_captured_mixed_batch(io, cache):
    """The kernels of a call that run beside each other, captured with the append before and replayed."""
    B = 45
    news = [100 if b % 15 == 2 else 1 for b in range(B)]
    lens = [n + (b * 97) % 600 for b, n in enumerate(news)]
    s = Setup(news, lens, io, cache, H=16, KVH=8, seed=77)
    s.table.clamp_(min=0)
    cos, sin = tables(max(lens), 128)
    q, out = s.out(), s.out()
    ws = vb200.paged_attn_workspace(s.pc, s.pb, s.H)

    def step():
        vb200.paged_append(s.pc, s.pb, s.kn, s.vn, q=s.q, q_out=q, cos=cos, sin=sin)
        vb200.paged_attn(s.pc, s.pb, q, out, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    s.k.copy_(torch.randn(s.k.shape, device="cuda"))
    s.v.copy_(torch.randn(s.v.shape, device="cuda"))
    for _ in range(4):
        for x in (s.q, s.kn, s.vn):
            x.copy_(torch.randn(x.shape, device="cuda"))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        keep, s.q = s.q, q
        ref, _, tol, _ = attn_reference(s)
        s.q = keep
        assert ((out.double() - ref).abs() <= tol).all()
    assert int(s.status) == 0


# ------------------------------------------------- as a user runs them together

def test_captured_step_replays_with_new_lengths():
    """Append and attention captured once, replayed for growing sequences of a static batch."""
    s = Setup([1, 1, 1], [40, 5, 90], "bf16", "bf16", seed=21, max_len=96)
    cos, sin = tables(96, 128)
    out, q = s.out(), s.out()
    ws = vb200.paged_attn_workspace(s.pc, s.pb, s.H)

    def step():
        vb200.paged_append(s.pc, s.pb, s.kn, s.vn, q=s.q, q_out=q, cos=cos, sin=sin)
        vb200.paged_attn(s.pc, s.pb, q, out, workspace=ws)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    s.k.copy_(torch.randn(s.k.shape, device="cuda"))
    s.v.copy_(torch.randn(s.v.shape, device="cuda"))
    for it in range(3):
        lens = [40 + it, 5 + it, 90 + it]
        s.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        s.lens_h = lens
        s.q.copy_(torch.randn(s.q.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        keep, s.q = s.q, q
        ref, _, tol, _ = attn_reference(s)
        s.q = keep
        assert ((out.double() - ref).abs() <= tol).all(), it


def test_on_another_stream():
    s = Setup([1, 60], [300, 200], "bf16", "bf16", seed=31)
    want = check_attn(s)
    out = s.out()
    ws = vb200.paged_attn_workspace(s.pc, s.pb, s.H)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        vb200.paged_attn(s.pc, s.pb, s.q, out, workspace=ws)
    st.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("io,cache", PAIRS)
def test_two_calls_at_once(io, cache):
    # a decode batch and a mixed one on two streams of the caller's choice, over and over
    s = [Setup([1] * 50, [(b * 37) % 900 + 1 for b in range(50)], io, cache, H=16, KVH=8, seed=1),
         Setup([1, 90, 1, 40], [800, 300, 1500, 40], io, cache, H=16, KVH=8, seed=2)]
    want = [check_attn(x) for x in s]
    ws = [vb200.paged_attn_workspace(x.pc, x.pb, x.H) for x in s]
    outs = [[x.out() for _ in range(6)] for x in s]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in s]
    for i in range(6):
        for x, st, w, o in zip(s, streams, ws, outs):
            vb200.paged_attn(x.pc, x.pb, x.q, o[i], workspace=w, stream=st.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)


@pytest.mark.parametrize("io,cache", PAIRS)
def test_k_and_v_in_one_pool_and_a_wider_table(io, cache):
    s = Setup([1, 70, 3], [200, 300, 50], io, cache, seed=6)
    want = check_attn(s)
    both = torch.stack([s.k, s.v], 1)  # [page, 2, position, head, dim]
    pc = vb200.PagedCache(both[:, 0], both[:, 1])
    wide = torch.full((3, s.table.shape[1] + 5), -9, dtype=torch.int32, device="cuda")
    wide[:, :s.table.shape[1]] = s.table
    pb = vb200.PagedBatch(s.q_start, s.lens, wide[:, :s.table.shape[1]], max_new=70, max_len=300, tokens=s.T)
    out = s.out()
    vb200.paged_attn(pc, pb, s.q, out)
    assert torch.equal(out, want)
    k, v = s.k.clone(), s.v.clone()
    vb200.paged_append(s.pc, s.pb, s.kn, s.vn)
    vb200.paged_append(pc, pb, s.kn, s.vn)
    for x, y in ((both[:, 0], s.k), (both[:, 1], s.v)):
        assert torch.equal(x.nan_to_num(9.0), y.nan_to_num(9.0))
    assert not torch.equal(k.nan_to_num(9.0), s.k.nan_to_num(9.0)) and not torch.equal(v.nan_to_num(9.0), s.v.nan_to_num(9.0))


def test_the_same_call_gives_the_same_bits():
    s = Setup([1, 130, 1], [3000, 400, 1700], "f32", "f32", seed=41)
    a = check_attn(s)
    for _ in range(3):
        assert torch.equal(check_attn(s), a)


def test_python_refusals():
    s = Setup([1, 2], [20, 30], "bf16", "bf16", seed=1)
    out = s.out()
    for call in (lambda: vb200.paged_attn(s.pc, s.pb, s.q[:2], out), lambda: vb200.paged_attn(s.pc, s.pb, s.q, out[:, :2]),
                 lambda: vb200.paged_attn(s.pc, s.pb, s.q.float(), out), lambda: vb200.paged_attn(s.pc, s.pb, s.q, out.cpu()),
                 lambda: vb200.paged_attn(s.pc, s.pb, s.q, out, lse=torch.zeros(3, 4, device="cuda", dtype=torch.float64)),
                 lambda: vb200.paged_attn(s.pc, s.pb, s.q[..., ::2], out),
                 lambda: vb200.paged_append(s.pc, s.pb, s.kn, s.vn.float()),
                 lambda: vb200.paged_append(s.pc, s.pb, s.kn, s.vn, q=s.q),
                 lambda: vb200.paged_append(s.pc, s.pb, s.kn, s.vn, cos=torch.zeros(64, 128, device="cuda")),
                 lambda: vb200.paged_append(s.pc, s.pb, s.kn, s.vn, k_norm=torch.zeros(64, device="cuda")),
                 lambda: vb200.PagedCache(s.k, s.v[:1]), lambda: vb200.PagedCache(s.k.double(), s.v.double()),
                 lambda: vb200.PagedBatch(s.q_start[:2], s.lens, s.table, max_new=1, max_len=1, tokens=3),
                 lambda: vb200.PagedBatch(s.q_start.long(), s.lens, s.table, max_new=1, max_len=1, tokens=3)):
        with pytest.raises(vb200.VBError):
            call()
    b = vb200.PagedBatch(s.q_start, s.lens, s.table, max_new=2, max_len=10**6, tokens=3)
    with pytest.raises(vb200.VBError):
        vb200.paged_attn(s.pc, b, s.q, out)
