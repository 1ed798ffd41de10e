"""Calls of the paged operators at the edges of what their interface allows."""
import ctypes as C
import math
import random
import time

import pytest

import vb200
from test_gpu_paged import PAIRS, U, Setup, attn_reference, check_attn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------- descriptors

@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("starts", [[0, 1000, 2000], [0, 1000, 1000, 2000, 2000], [0, 1000, 1999]])
def test_a_sequence_behind_the_rows_takes_no_other_ones_place(io, cache, starts):
    # the last rows claimed lie behind `tokens`; sequence 0 has all of its own
    n = len(starts) - 1
    s = Setup([1000] + [0] * (n - 1), [1000] * n, io, cache, seed=3)
    want, _, tol, _ = attn_reference(s)
    s.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
    out = s.out()
    vb200.paged_attn(s.pc, s.pb, s.q, out)
    assert int(s.status) == vb200.PAGED_BAD_ROWS
    assert ((out.double() - want).abs() <= tol).all()


def _status(s, call, q_start=None, lens=None, tokens=None, max_new=None, max_len=None):
    q_start = s.q_start if q_start is None else torch.tensor(q_start, dtype=torch.int32, device="cuda")
    lens = s.lens if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    s.status.zero_()
    pb = vb200.PagedBatch(q_start, lens, s.table, max_new=max_new or s.pb.s.max_new, max_len=s.pb.max_len, tokens=s.T,
                          status=s.status)
    if call == "attn":
        vb200.paged_attn(s.pc, pb, s.q, s.out())
    else:
        vb200.paged_append(s.pc, pb, s.kn, s.vn)
    return int(s.status)


@pytest.mark.parametrize("call", ["attn", "append"])
@pytest.mark.parametrize("kind", ["one", "few", "decode", "prompt", "mixed"])
def test_every_bad_sequence_is_reported(call, kind):
    # whichever kernel takes the batch, and whether or not a row leads to the sequence
    news = {"one": [1], "few": [8, 8], "decode": [1] * 50, "prompt": [200], "mixed": [1, 150, 1, 1]}[kind]
    s = Setup(news, [n + 60 for n in news], "bf16", "bf16", H=16, KVH=8, seed=2)
    starts, lens, B, T = s.q_start.tolist(), s.lens_h, len(news), s.T
    rows, length = vb200.PAGED_BAD_ROWS, vb200.PAGED_BAD_LEN
    assert _status(s, call) == 0
    assert _status(s, call, q_start=starts[:-1] + [T + 1]) == rows            # rows behind the last one
    assert _status(s, call, q_start=starts[:-1] + [T + 10**6]) == rows
    assert _status(s, call, q_start=starts[:-1] + [starts[-2] - 1]) == rows   # fewer than none
    assert _status(s, call, q_start=[-1] + starts[1:]) == rows
    assert _status(s, call, q_start=[T] * B + [T + 7]) == rows                # and no sequence has rows
    assert _status(s, call, lens=lens[:-1] + [-1]) == length
    assert _status(s, call, q_start=[0] * (B + 1), lens=lens[:-1] + [s.pb.max_len + 1]) == length
    if max(news) > 20:
        assert _status(s, call, max_new=max(news) - 1) == rows


def test_python_faces_refuse_with_their_own_error():
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")
    f32 = lambda *shape: torch.zeros(shape, device="cuda")
    s = Setup([1, 2], [20, 30], "bf16", "bf16", seed=1)
    out = s.out()
    x, y = f32(2, 500), f32(2, 500)
    for call in (lambda: vb200.LogitsRules(mask=i32(16)), lambda: vb200.LogitsRules(mask=i32()),
                 lambda: vb200.LogitsRules(mask=i32(2, 4, 4)), lambda: vb200.LogitsRules(prompt_len=i32()),
                 lambda: vb200.LogitsRules(hist_start=i32(3), hist_ids=i32(2, 2)),
                 lambda: vb200.LogitsRules(bias_start=i32(3), bias_ids=i32(4), bias_vals=f32(5)),
                 lambda: vb200.logits_process(x[0], y[0], vb200.LogitsRules()),
                 lambda: vb200.logits_process(x, y[:1], vb200.LogitsRules()),
                 lambda: vb200.paged_attn(s.pc, s.pb, s.q[:, 0], out), lambda: vb200.paged_attn(s.pc, s.pb, s.q, s.q),
                 lambda: vb200.paged_attn(s.pc, s.pb, s.q, out, lse=f32(3)),
                 lambda: vb200.paged_attn(s.pc, s.pb, s.q, out, workspace=torch.zeros(8, dtype=torch.uint8)),
                 lambda: vb200.paged_append(s.pc, s.pb, s.kn[:, 0], s.vn), lambda: vb200.PagedCache(s.k[0], s.v[0]),
                 lambda: vb200.PagedBatch(s.q_start, s.lens, s.table[0], max_new=2, max_len=30, tokens=3),
                 lambda: vb200.PagedBatch(s.q_start, s.lens[0], s.table, max_new=2, max_len=30, tokens=3)):
        with pytest.raises(vb200.VBError):
            call()


# ------------------------------------------------- values that are not finite

def formula(s, window=0):
    """out in 64 bits, the error bound of its finite elements, and lse.  What is seen is multiplied by its
    weight, an infinity by a weight of 0 (a score of -inf) being NaN; what is not seen is not there.
    A row whose scores are all -inf is empty."""
    out = torch.zeros(s.T, s.H, s.D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((s.T, s.H), -math.inf, dtype=torch.float64, device="cuda")  # NaN under a score of +inf, as out
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
        a = torch.einsum("nhgd,lhd->nhgl", q, k.nan_to_num(0, 0, 0)) * s.D**-0.5
        size = torch.einsum("nhgd,lhd->nhgl", q.abs(), k.abs().nan_to_num(0, 0, 0)) * s.D**-0.5
        for n, h, d in torch.nonzero(~torch.isfinite(k)).tolist():  # (one element of a key at most)
            x = q[:, h, :, d] * k[n, h, d]
            a[:, h, :, n] = torch.where(torch.isnan(x) | torch.isinf(x), x, a[:, h, :, n])
        a = a.masked_fill(~see[:, None, None], -math.inf)
        empty = (a == -math.inf).all(-1, keepdim=True)
        p = torch.where(empty, 0, torch.softmax(a, -1))
        fin = torch.isfinite(v)
        y = torch.einsum("nhgl,lhd->nhgd", p, torch.where(fin, v, 0))
        mass = torch.einsum("nhgl,lhd->nhgd", p, torch.where(fin, v, 0).abs())
        for n, h, d in torch.nonzero(~fin).tolist():
            y[:, h, :, d] += torch.where(see[:, n, None], p[:, h, :, n] * v[n, h, d], 0)
        y = torch.where(empty, 0, y)
        size = size.masked_fill(~see[:, None, None], 0).amax(-1)[..., None]
        u = U[s.io]
        out[r] = y.reshape(-1, s.H, s.D)
        lse[r] = torch.where((a == math.inf).any(-1), math.nan, torch.logsumexp(a, -1)).reshape(-1, s.H)
        tol[r] = ((2 * size * 2.0**-19 + 2.0**-20 + (u if s.io != "f32" else 0)) * mass + u * y.abs() + 1e-30 +
                  (2.0**-24 if s.io == "f16" else 0)).reshape(-1, s.H, s.D)
    return out, tol, lse


def check_formula(s, window=0):
    want, tol, wl = formula(s, window)
    out, lse = s.out(), torch.full((s.T, s.H), 55.0, device="cuda")
    vb200.paged_attn(s.pc, s.pb, s.q, out, lse=lse, window=window)
    fin = torch.isfinite(want)
    assert torch.equal(out.double()[~fin].nan_to_num(7.0), want[~fin].nan_to_num(7.0))
    assert ((out.double() - want).abs()[fin] <= tol[fin]).all()
    assert torch.equal(torch.isnan(lse), torch.isnan(wl))
    fin = torch.isfinite(wl)
    assert ((lse.double() - wl).abs()[fin] <= 1e-3).all()
    return out


# B sequences of one new token: clusters; shared-out keys; shared-out keys of a long sequence; the
# kernels of many rows (more query heads a KV head than the other takes)
SEEN = [(2, 300, 16, 8), (50, 700, 16, 8), (1, 9000, 16, 8), (3, 500, 20, 1), (3, 500, 66, 2)]


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,ctx,H,KVH", SEEN)
def test_an_infinity_that_a_decoding_row_sees(io, cache, B, ctx, H, KVH, D):
    s = Setup([1] * B, [ctx - 3 * b for b in range(B)], io, cache, H=H, KVH=KVH, D=D, seed=B)

    def put(x, b, pos, head, d, value):
        x[s.table[b, pos // s.page].long(), pos % s.page, head, d] = value

    put(s.v, 0, ctx // 3, 0, 5, math.inf)
    put(s.v, 0, ctx // 2, 0, 9, -math.inf)
    put(s.v, B - 1, 0, KVH - 1, D - 1, math.inf)
    put(s.v, B - 1, 1, KVH - 1, D - 1, -math.inf)  # both: NaN
    put(s.v, B - 1, 2, KVH - 1, 0, math.nan)
    put(s.v, B // 2, 7, 0, 2, -math.inf)
    out = check_formula(s)
    assert out[0, 0, 5] == math.inf and out[0, 0, 9] == -math.inf and torch.isnan(out[B - 1, H - 1, D - 1])
    assert torch.isfinite(out[0, 0, 3:5]).all()


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("B,ctx,H,KVH", SEEN)
def test_a_key_of_minus_infinity(io, cache, B, ctx, H, KVH):
    # scores of -inf where q is positive: no weight; of +inf (and NaN) where it is negative
    s = Setup([1] * B, [ctx - 3 * b for b in range(B)], io, cache, H=H, KVH=KVH, seed=B + 1)
    s.k[s.table[0, 1].long(), 3, 0, 4] = -math.inf
    s.q[0, :, 4] = s.q[0, :, 4].abs() + 0.5
    s.q[0, 1, 4] *= -1
    out = check_formula(s)
    assert torch.isfinite(out[0, 0]).all() and torch.isnan(out[0, 1]).all()


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("n", [2, 40, 300])
def test_an_infinity_that_rows_of_a_chunk_see(io, cache, n):
    s = Setup([n, 1, n], [n + 500, 60, n], io, cache, seed=n)
    for b, pos, head, d, value in ((0, 3, 0, 5, math.inf), (0, 400, 1, 9, -math.inf), (2, n - 1, 0, 1, math.inf),
                                   (0, 500 + n // 2, 1, 7, math.nan)):
        s.v[s.table[b, pos // s.page].long(), pos % s.page, head, d] = value
    check_formula(s)
    check_formula(s, window=n + 90)


@pytest.mark.parametrize("n", [1, 2, 40, 300])
def test_an_infinity_under_a_weight_that_f16_has_not(n):
    s = Setup([n, 1], [n + 200, 90], "f16", "f16", H=4, KVH=2, seed=n)
    slot = s.table[0, 2].long(), 1  # position 33, seen by all rows of sequence 0
    s.q[:n, :, 0] = 8.0
    s.k[..., 0] = 0.0
    s.k[slot[0], slot[1], :, 0] = -40.0  # 40 * 8 / sqrt(128) = 28 below the others: 2^-40
    s.v[slot[0], slot[1], 0, 3] = math.inf
    out = check_formula(s)
    assert (out[:n, :2, 3] == math.inf).all()


@pytest.mark.parametrize("seed", range(40))
def test_random_batches_with_values_that_are_not_finite(seed):
    r = random.Random(seed)
    io, cache = r.choice(PAIRS)
    kvh, group = r.choice([1, 2, 4, 8]), r.choice([1, 2, 2, 4, 5, 8, 9, 16, 17, 20, 33])
    most = r.choice([1, 1, r.randint(2, 20), r.randint(2, 300)])
    B = min(int(2 ** r.uniform(0, 5)), max(1, 12000 // (most * group * kvh)))
    news = [r.choice([1, most, r.randint(0, most)]) for _ in range(B)]
    news[0] = most
    s = Setup(news, [n + r.randint(0, 600) for n in news], io, cache, H=kvh * group, KVH=kvh, D=r.choice([64, 128]),
              page=r.choice([1, 5, 8, 16, 32, 64, 128]), order=r.choice(["phd", "hpd"]), seed=seed)
    for _ in range(r.randint(0, 6)):
        b = r.randrange(B)
        if s.lens_h[b]:
            p, h = r.randrange(s.lens_h[b]), r.randrange(kvh)
            x = r.choice([s.k, s.v, s.v])[s.table[b, p // s.page].long(), p % s.page, h]
            if torch.isfinite(x).all():
                x[r.randrange(s.D)] = r.choice([math.nan, math.inf, -math.inf])
    check_formula(s, window=r.choice([0, 0, 1, 7, 64, 300]))


def _time(call, n=5):
    call()
    t = []
    for _ in range(n):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        t.append(a.elapsed_time(b))
    return sorted(t)[n // 2]


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("what", ["v", "k", "v element"])
@pytest.mark.parametrize("where", ["first", "own"])
def test_a_nan_that_rows_see_costs_little(io, cache, what, where):
    """One bad row of the cache makes every later output NaN: no reason for a call to take many
    times as long and hold up the other sequences of its batch."""
    n = 4096
    s = Setup([n, 1], [n, 70], io, cache, H=16, KVH=8, seed=1, page=64)
    ws, out = vb200.paged_attn_workspace(s.pc, s.pb, s.H), s.out()
    call = lambda: vb200.paged_attn(s.pc, s.pb, s.q, out, workspace=ws)
    clean = _time(call)
    keep = out.clone()
    x = s.k if what == "k" else s.v
    pos = 0 if where == "first" else n - 130
    dims = slice(9, 10) if what == "v element" else slice(None)
    x[s.table[0, pos // 64].long(), pos % 64, :, dims] = math.nan
    bad = _time(call)
    assert torch.isnan(out[pos:n, :, dims]).all()
    assert torch.equal(out[:pos], keep[:pos]) or (torch.isfinite(out[:pos]).all() and
                                                  (out[:pos].float() - keep[:pos].float()).abs().max() < 0.02)
    if what == "v element":
        assert torch.isfinite(out[:n, :, :9]).all() and torch.isfinite(out[:n, :, 10:]).all()
    assert torch.equal(out[n:], keep[n:])
    print(f"{io} {cache} {what} {where}: {clean:.3f} -> {bad:.3f} ms")
    assert bad < 4 * clean + 3.0, (clean, bad)  # 0.1-1.1 ms; 8-36 where every key was walked by one warp


# ---------------------------------------------------------------- launches

def launches(call):
    """How many nodes a call captures as."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    n = C.c_size_t()
    assert C.CDLL("libcuda.so.1").cuGraphGetNodes(C.c_void_p(graph.raw_cuda_graph()), None, C.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("io,cache", PAIRS)
def test_one_long_prompt_launches_no_join(io, cache):
    # one sequence alone has no keys that are shared out, however many it has
    def count(ctx):
        s = Setup([300], [ctx], io, cache, H=16, KVH=8, seed=1)
        ws, out = vb200.paged_attn_workspace(s.pc, s.pb, s.H), s.out()
        return launches(lambda: vb200.paged_attn(s.pc, s.pb, s.q, out, workspace=ws))

    assert count(5000) == count(4000) >= 2


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("D", [64, 128])
def test_clusters_are_used_while_all_fit_the_card(io, cache, D):
    # one launch; shared-out keys take a second one, the join
    def count(B):
        s = Setup([1] * B, [300] * B, io, cache, H=2, KVH=1, D=D, seed=B)
        check_attn(s)
        ws, out = vb200.paged_attn_workspace(s.pc, s.pb, s.H), s.out()
        return launches(lambda: vb200.paged_attn(s.pc, s.pb, s.q, out, workspace=ws))

    most = 15 if cache == "f32" and D == 128 else 37
    assert count(most) == 1 and count(most + 1) == 2


# ------------------------------------------------------ a wait that gives up

@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("news,lens,D,status", [([200], [200], 128, True), ([1, 40], [30, 3000], 64, False),
                                                ([1, 1, 150], [60, 700, 150], 128, True)])
def test_a_wait_runs_out(io, cache, news, lens, D, status):
    # the first block of the kernel of many rows: the last sequence's last tile, one KV head and split of it
    s = Setup(news, lens, io, cache, H=16, KVH=8, D=D, seed=5, status=status)
    ws = vb200.paged_attn_workspace(s.pc, s.pb, s.H)

    def call():
        out, lse = s.out(), torch.full((s.T, s.H), 55.0, device="cuda")
        vb200.paged_attn(s.pc, s.pb, s.q, out, lse=lse, workspace=ws)
        torch.cuda.synchronize()
        return out, lse

    want, wl = call()
    vb200.debug_arm_fault(3)
    t0 = time.time()
    out, lse = call()
    took = time.time() - t0
    assert 1.5 < took < 30.0, took
    if status:
        assert int(s.status) == vb200.PAGED_TIMEOUT
        s.status.zero_()
    hit = torch.zeros_like(lse, dtype=torch.bool)
    hit[s.T - news[-1]:, :2] = True
    assert torch.equal(lse[~hit], wl[~hit]) and torch.equal(out[~hit], want[~hit])
    # NaN, or taken again from the keys themselves: never what the output or a workspace held before
    for x, w in ((lse, wl), (out, want)):
        x, w = x[hit].float(), w[hit].float()
        assert (torch.isnan(x) | ((x - w).abs() < 0.02)).all()
    out, lse = call()  # one launch only
    assert torch.equal(out, want) and torch.equal(lse, wl)
    assert not status or int(s.status) == 0


def test_a_captured_call_is_never_the_armed_one():
    s = Setup([200], [200], "bf16", "bf16", seed=5)
    ws, want = vb200.paged_attn_workspace(s.pc, s.pb, s.H), check_attn(s)
    out = s.out()
    graph = torch.cuda.CUDAGraph()
    vb200.debug_arm_fault(3)
    try:
        with torch.cuda.graph(graph):
            vb200.paged_attn(s.pc, s.pb, s.q, out, workspace=ws)
    finally:
        vb200.debug_arm_fault(0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and int(s.status) == 0
