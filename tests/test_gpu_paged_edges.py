"""Calls of the paged operators at the edges of what their interface allows."""
import time

import pytest

import vb200
from test_gpu_paged import PAIRS, Setup, attn_reference, check_attn

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
    lost = torch.isnan(lse)
    assert lost.any() and not lost[:, 2:].any() and not lost[:s.T - news[-1]].any()
    assert torch.equal(lse[~lost], wl[~lost]) and torch.equal(out[~lost], want[~lost])
    # NaN, or taken again from the keys themselves: never what the output or a workspace held before
    left = out[lost].float()
    assert (torch.isnan(left) | ((left - want[lost].float()).abs() < 0.02)).all()
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
