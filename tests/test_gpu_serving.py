"""The paged calls and the logits rules as a server of requests runs them: a small
Qwen3-shaped model stepped through the library's own kernels over a paged cache --
prompts of different lengths read in chunks while other sequences decode -- against
the engine, which keeps one contiguous cache a sequence.

Both compute in f32; the tolerance is the one the engine's steps are held to
against the oracle (1e-3 on logits), tokens are the same.
"""
import numpy as np
import pytest

import vb200
import vbsynth

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class PagedModel:
    """The decoder over a shared pool of pages: everything a step does is a call of the library."""

    def __init__(self, cfg, weights, pages=64, page=8, cache=torch.float32):
        self.c = cfg
        self.H, self.KVH = cfg["num_attention_heads"], cfg["num_key_value_heads"]
        self.D, self.hid = cfg["head_dim"], cfg["hidden_size"]
        self.w = {k: torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32)).cuda() for k, v in weights.items()}
        self.page = page
        L = cfg["num_hidden_layers"]
        self.caches = [vb200.PagedCache(*(torch.full((pages, page, self.KVH, self.D), float("nan"), device="cuda",
                                                     dtype=cache) for _ in range(2))) for _ in range(L)]
        pos = torch.arange(512, device="cuda", dtype=torch.float64)[:, None]
        inv = cfg["rope_theta"] ** (-torch.arange(0, self.D, 2, device="cuda", dtype=torch.float64) / self.D)
        self.cos, self.sin = (torch.cat([f(pos * inv)] * 2, 1).float().contiguous() for f in (torch.cos, torch.sin))
        self.free = list(range(pages))[::-1]
        self.pages_of, self.len_of = {}, {}

    def _mm(self, x, name):
        w = self.w[name]
        y = torch.empty(x.shape[0], w.shape[0], device="cuda")
        vb200.matmul_nt_f32(x, w, y)
        return y

    def _norm(self, x, name):
        y = torch.empty_like(x)
        vb200.rmsnorm(x, self.w[name], y, self.c["rms_norm_eps"])
        return y

    def step(self, new):
        """new: {sequence: its new tokens}; the logits behind each one's last token."""
        q_start, lens, tables, ids = [0], [], [], []
        for s, toks in new.items():
            self.len_of[s] = self.len_of.get(s, 0) + len(toks)
            own = self.pages_of.setdefault(s, [])
            while len(own) * self.page < self.len_of[s]:
                own.append(self.free.pop())
            q_start.append(q_start[-1] + len(toks))
            lens.append(self.len_of[s])
            tables.append(own)
            ids += list(toks)
        width = max(map(len, tables))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        batch = vb200.PagedBatch(i32(q_start), i32(lens), i32([t + [0] * (width - len(t)) for t in tables]),
                                 max_new=max(len(t) for t in new.values()), max_len=max(lens), tokens=len(ids))
        eps, T = self.c["rms_norm_eps"], len(ids)
        x = self.w["model.embed_tokens.weight"][torch.tensor(ids, device="cuda")].contiguous()
        q = torch.empty(T, self.H, self.D, device="cuda")
        out = torch.empty_like(q)
        for i, cache in enumerate(self.caches):
            n = vb200.layer_names(i)
            h = self._norm(x, n["input_norm"])
            qkv = [self._mm(h, n[k]).view(T, -1, self.D) for k in ("wq", "wk", "wv")]
            vb200.paged_append(cache, batch, qkv[1], qkv[2], q=qkv[0], q_out=q, cos=self.cos, sin=self.sin,
                               q_norm=self.w[n["q_norm"]], k_norm=self.w[n["k_norm"]], eps=eps)
            vb200.paged_attn(cache, batch, q, out)
            vb200.add(x, self._mm(out.view(T, -1), n["wo"]))
            h = self._norm(x, n["post_norm"])
            gate, up = self._mm(h, n["wg"]), self._mm(h, n["wu"])
            vb200.silu_mul(gate, up)
            vb200.add(x, self._mm(gate, n["wd"]))
        last = torch.tensor(q_start[1:], device="cuda") - 1
        return self._mm(self._norm(x[last].contiguous(), "model.norm.weight"), "model.embed_tokens.weight")

    def drop(self, s):
        self.free += self.pages_of.pop(s)[::-1]
        del self.len_of[s]


def small():
    cfg = vbsynth.qwen3_config(hidden_size=256, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                               intermediate_size=512, vocab_size=1000)
    return cfg, vbsynth.make_weights(cfg, seed=11)


def engine_logits(cfg, w, tokens, steps):
    """Logits behind the last `steps` of the tokens."""
    e = vb200.Engine(cfg, device=0).load(w)
    e.reset_cache(len(tokens) + 1)
    got = [e.step(int(t)) for t in tokens]
    e.close()
    return np.stack(got[-steps:])


@pytest.mark.parametrize("page", [1, 8, 24])
def test_continuous_batching_matches_the_engine(page):
    cfg, w = small()
    rng = np.random.default_rng(5)
    prompts = {s: rng.integers(0, cfg["vocab_size"], n).tolist() for s, n in (("a", 37), ("b", 5), ("c", 70))}
    m = PagedModel(cfg, w, pages=400 // page + 8, page=page)
    said = {s: [] for s in prompts}
    seen = {s: [] for s in prompts}
    todo = {s: list(p) for s, p in prompts.items()}
    arrives = {"a": 0, "b": 2, "c": 3}
    for it in range(12):
        new = {}
        for s in prompts:
            if it < arrives[s]:
                continue
            if todo[s]:  # a chunk of at most 16 tokens of its prompt
                new[s], todo[s] = todo[s][:16], todo[s][16:]
            else:
                new[s] = [said[s][-1]]
        logits = m.step(new)
        pick = torch.empty(len(new), dtype=torch.int32, device="cuda")
        vb200.argmax_rows(logits, pick)
        for i, s in enumerate(new):
            if not todo[s]:
                said[s].append(int(pick[i]))
                seen[s].append(logits[i].cpu().numpy())
    for s, p in prompts.items():
        assert len(said[s]) >= 3
        want = engine_logits(cfg, w, p + said[s][:-1], len(said[s]))
        assert np.abs(np.stack(seen[s]) - want).max() <= 1e-3, s
        assert said[s] == want.argmax(-1).tolist(), s


def test_pages_go_from_one_sequence_to_the_next():
    """A finished sequence's pages, with its old rows in them, serve the next one."""
    cfg, w = small()
    m = PagedModel(cfg, w, pages=4, page=8)
    rng = np.random.default_rng(6)
    for n in (30, 9, 17):
        p = rng.integers(0, cfg["vocab_size"], n).tolist()
        got = m.step({"s": p}).cpu().numpy()
        assert np.abs(got - engine_logits(cfg, w, p, 1)).max() <= 1e-3
        m.drop("s")


def test_generation_under_rules():
    """Chunk, decode, rules, sampler: what is forbidden never comes, what was said comes less often."""
    cfg, w = small()
    V = cfg["vocab_size"]
    m = PagedModel(cfg, w)
    rng = np.random.default_rng(7)
    prompt = rng.integers(0, V, 20).tolist()
    allowed = sorted(rng.choice(V, 12, replace=False).tolist())
    bits = np.zeros((V + 31) // 32, np.uint32)
    for t in allowed:
        bits[t // 32] |= np.uint32(1 << (t % 32))
    mask = torch.from_numpy(bits.view(np.int32)[None].copy()).cuda()
    said, feed = [], prompt
    greedy = vb200.Sampler(temperature=0.0)
    for _ in range(8):
        logits = m.step({"s": feed})
        hist = torch.tensor(prompt + said, dtype=torch.int32, device="cuda")
        rules = vb200.LogitsRules(hist_start=torch.tensor([0, hist.numel()], dtype=torch.int32, device="cuda"), hist_ids=hist,
                                  prompt_len=torch.tensor([len(prompt)], dtype=torch.int32, device="cuda"),
                                  presence=torch.full((1,), 1e4, device="cuda"), mask=mask)
        vb200.logits_process(logits, logits, rules)
        feed = [greedy.sample(logits[0])]
        said += feed
    assert all(t in allowed for t in said)
    assert len(set(said)) == len(said)  # a presence penalty above every difference: nothing is said twice
