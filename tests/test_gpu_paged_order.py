"""Layers one after the other on one stream, with nothing but this library's launches between
them: every launch may start before the one ahead of it has ended, and each layer's append
writes the q that its attention reads into the buffer that the layer before has just read."""
import pytest

import vb200
from test_gpu_paged import PAIRS, Setup, tables

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

LAYERS = 12
BATCHES = {
    "mixed": [100 if b % 15 == 2 else 1 for b in range(45)],  # both kernels of a call
    "decode": [1] * 45,
    "short": [1, 1],
    "prompts": [150, 90],
}


@pytest.mark.parametrize("io,cache", PAIRS)
@pytest.mark.parametrize("kind", list(BATCHES))
def test_layers_share_their_buffers(io, cache, kind):
    news = BATCHES[kind]
    lens = [n + (b * 97) % 600 for b, n in enumerate(news)]
    s = Setup(news, lens, io, cache, H=16, KVH=8, seed=7)
    s.table.clamp_(min=0)
    cos, sin = tables(max(lens), 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    pools, rows = [], []
    for _ in range(LAYERS):
        k, v = (torch.randn(s.k.shape, device="cuda", generator=g).to(s.k.dtype) for _ in range(2))
        pools.append((vb200.PagedCache(k, v), k.clone(), v.clone()))
        rows.append([torch.randn(x.shape, device="cuda", generator=g).to(x.dtype) for x in (s.q, s.kn, s.vn)])
    q, ws = s.out(), vb200.paged_attn_workspace(s.pc, s.pb, s.H)
    outs = [s.out() for _ in range(LAYERS)]

    def layer(i, sync=False):
        qi, kn, vn = rows[i]
        vb200.paged_append(pools[i][0], s.pb, kn, vn, q=qi, q_out=q, cos=cos, sin=sin)
        if sync:
            torch.cuda.synchronize()
        vb200.paged_attn(pools[i][0], s.pb, q, outs[i], workspace=ws)
        if sync:
            torch.cuda.synchronize()

    for i in range(LAYERS):
        layer(i, sync=True)
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(LAYERS):
            layer(i)
    for turn in range(6):
        for o, (pc, k, v) in zip(outs, pools):
            o.fill_(float("nan"))
            pc.k.copy_(k)
            pc.v.copy_(v)
        ws.view(torch.int32).fill_(1 if turn % 2 else -1)  # whatever an earlier user of the workspace left
        if turn < 3:
            for i in range(LAYERS):
                layer(i)
        else:
            graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
    assert int(s.status) == 0
