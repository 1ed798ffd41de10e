"""vb_logits_process against its definition in 64 bits.

A logit goes through at most one product or division, a product and two
subtractions for the penalties and one sum for the bias, the bias itself a sum
of k terms: each rounds by at most 2^-24 of its result, and no result is larger
than |x| rep + freq n + pres + sum |bias|, so 8 roundings (and one for each
further bias) of that size bound the error; 16-bit logits add their rounding.
"""
import math

import pytest

import vb200

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = {torch.float32: 0.0, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(R, V, dtype=torch.float32, hist=0, bias=0, mask=False, pen=True, seed=0, stride=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    stride = stride or V
    x = (3 * torch.randn(R, stride, device="cuda", generator=g)).to(dtype)[:, :V]
    r = {}
    if hist:
        n = [hist * (i + 1) // R if i != 1 else 0 for i in range(R)]  # the second row has no history
        r["hist_start"] = i32([0] + torch.tensor(n).cumsum(0).tolist())
        r["hist_ids"] = torch.randint(-3, V + 3, (sum(n),), device="cuda", generator=g).to(torch.int32)
        r["prompt_len"] = i32([k // 3 for k in n])
        if pen:
            r["repetition"] = 0.7 + torch.rand(R, device="cuda", generator=g)
            r["frequency"] = torch.randn(R, device="cuda", generator=g)
            r["presence"] = torch.randn(R, device="cuda", generator=g)
    if bias:
        n = [bias if i != R - 1 or R == 1 else 0 for i in range(R)]
        r["bias_start"] = i32([0] + torch.tensor(n).cumsum(0).tolist())
        # few different ids: most stand in the list more than once
        r["bias_ids"] = torch.randint(-2, min(V, 2 * bias // 3 + 1) + 1, (sum(n),), device="cuda", generator=g).to(torch.int32)
        r["bias_vals"] = 3 * torch.randn(sum(n), device="cuda", generator=g)
    if mask:
        r["mask"] = torch.randint(-2**31, 2**31, (R, (V + 31) // 32 + 1), device="cuda", generator=g).to(torch.int32)
    return x, r


def reference(x, r):
    R, V = x.shape
    y = x.double()
    size = y.abs()
    for i in range(R):
        if "hist_ids" in r:
            ids = r["hist_ids"][r["hist_start"][i]:r["hist_start"][i + 1]].long()
            p = int(r["prompt_len"][i]) if "prompt_len" in r else 0
            ok = (ids >= 0) & (ids < V)
            seen = torch.zeros(V, dtype=torch.bool, device="cuda")
            seen[ids[ok]] = True
            n = torch.bincount(ids[p:][ok[p:]], minlength=V).double()
            if "repetition" in r:
                rep = r["repetition"][i].double()
                y[i] = torch.where(seen, torch.where(y[i] > 0, y[i] / rep, y[i] * rep), y[i])
                size[i] = torch.maximum(size[i], y[i].abs())
            for name, k in (("frequency", n), ("presence", (n > 0).double())):
                if name in r:
                    y[i] -= r[name][i].double() * k
                    size[i] += r[name][i].double().abs() * k
        if "bias_ids" in r:
            s = slice(int(r["bias_start"][i]), int(r["bias_start"][i + 1]))
            ids, val = r["bias_ids"][s].long(), r["bias_vals"][s].double()
            ok = (ids >= 0) & (ids < V)
            y[i].index_add_(0, ids[ok], val[ok])
            size[i].index_add_(0, ids[ok], val[ok].abs())
        if "mask" in r:
            t = torch.arange(V, device="cuda")
            y[i][(r["mask"][i].long()[t // 32] >> (t % 32)) & 1 == 0] = -math.inf
    return y, size


def check(x, r, in_place=False, out=None):
    want, size = reference(x, r)
    n = 8 + (r["bias_ids"].numel() if "bias_ids" in r else 0)
    got = x if in_place else torch.empty_like(x) if out is None else out
    vb200.logits_process(x, got, vb200.LogitsRules(**r))
    torch.cuda.synchronize()
    g, inf = got.double(), torch.isinf(want)
    assert torch.equal(g[inf], want[inf])
    tol = n * 2.0**-24 * size + U[x.dtype] * want.abs() + (2.0**-25 if x.dtype == torch.float16 else 0)
    assert ((g - want).abs()[~inf] <= tol[~inf]).all()
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 5, 31, 32, 33, 1000, 4095, 4096, 4097, 8191, 32003, 151936])
def test_sizes(dtype, V):
    check(*make(3, V, dtype, hist=500, bias=40, mask=True, seed=V))


@pytest.mark.parametrize("parts", [dict(), dict(hist=300), dict(bias=33), dict(mask=True), dict(hist=9, pen=False),
                                   dict(hist=20000, bias=1000, mask=True)])
@pytest.mark.parametrize("R", [1, 2, 7])
def test_parts(parts, R):
    check(*make(R, 9001, seed=R, **parts))


@pytest.mark.parametrize("only", ["repetition", "frequency", "presence"])
def test_one_penalty(only):
    x, r = make(3, 5000, hist=2000, seed=1)
    for name in ("repetition", "frequency", "presence"):
        if name != only:
            del r[name]
    check(x, r)
    del r["prompt_len"]  # the whole history counts
    check(x, r)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,stride", [(1001, 1001), (1001, 1003), (4099, 4111), (8000, 8008)])
def test_strides_in_place_and_apart(dtype, V, stride):
    x, r = make(4, V, dtype, hist=100, bias=10, mask=True, seed=stride, stride=stride)
    base = x.clone()
    apart = check(x, r)
    # an output whose rows lie at other offsets, with its neighbours left alone
    big = torch.full((4, V + 7), 5.0, device="cuda", dtype=dtype)
    check(x, r, out=big[:, 3:3 + V])
    assert torch.equal(big[:, 3:3 + V], apart) and (big[:, :3] == 5).all() and (big[:, 3 + V:] == 5).all()
    full = x._base
    rest = full[:, V:].clone()
    check(x, r, in_place=True)
    assert torch.equal(x, apart) and torch.equal(full[:, V:], rest) and not torch.equal(x, base)


def test_values_that_are_not_finite():
    x, r = make(3, 700, hist=300, bias=5, mask=True, seed=2)
    x[:, ::7] = -math.inf
    x[:, 3::11] = math.inf
    x[0, 5] = math.nan
    r["mask"][0, 0] &= ~(1 << 5)  # the NaN is masked: -inf
    got = check(x, r)
    assert got[0, 5] == -math.inf and not torch.isnan(got).any()
    r["mask"].zero_()  # nothing is allowed
    vb200.logits_process(x, got, vb200.LogitsRules(**r))
    assert (got == -math.inf).all()


def test_the_same_bits_every_time():
    # many biases of one token: a sum in another order would round differently
    x, r = make(2, 3000, bias=900, hist=5000, seed=3)
    r["bias_ids"] %= 7
    first = check(x, r)
    for _ in range(5):
        assert torch.equal(check(x, r), first)


def test_lists_out_of_their_array():
    # offsets beyond the lists are cut at their ends
    x, r = make(2, 500, hist=50, bias=8, seed=4)
    want = check(x, r)
    bad = dict(r, hist_start=r["hist_start"].clone(), bias_start=r["bias_start"].clone())
    bad["hist_start"][2] = 10**9
    bad["bias_start"][0] = -5
    got = torch.empty_like(x)
    vb200.logits_process(x, got, vb200.LogitsRules(**bad))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_python_refusals():
    x, r = make(2, 500, hist=50, bias=8, mask=True, seed=5)
    out = torch.empty_like(x)
    ok = vb200.LogitsRules(**r)
    for call in (lambda: vb200.logits_process(x[:1], out[:1], ok), lambda: vb200.logits_process(x, out.half(), ok),
                 lambda: vb200.logits_process(x.T, out.T, vb200.LogitsRules()),
                 lambda: vb200.logits_process(x, out.cpu(), ok),
                 lambda: vb200.LogitsRules(**dict(r, mask=r["mask"].long())),
                 lambda: vb200.LogitsRules(**dict(r, presence=r["presence"][:1])),
                 lambda: vb200.LogitsRules(hist_start=r["hist_start"]),
                 lambda: vb200.LogitsRules(bias_start=r["bias_start"], bias_ids=r["bias_ids"]),
                 lambda: vb200.logits_process(x, out, vb200.LogitsRules(mask=r["mask"][:, :4].contiguous())),
                 lambda: vb200.logits_process(x, out, vb200.LogitsRules(repetition=r["repetition"]))):
        with pytest.raises(vb200.VBError):
            call()


def test_before_the_sampler():
    """Rules, then greedy: the pick is the best allowed token, and a penalised one loses."""
    x, _ = make(1, 2000, seed=6)
    top = torch.topk(x[0], 3).indices.tolist()
    mask = torch.full((1, 63), -1, dtype=torch.int32, device="cuda")
    t = top[0]
    mask[0, t // 32] &= ~(1 << (t % 32)) if t % 32 != 31 else 0x7FFFFFFF
    rules = vb200.LogitsRules(hist_start=i32([0, 1]), hist_ids=i32([top[1]]), presence=torch.full((1,), 50.0, device="cuda"),
                              mask=mask)
    out = torch.empty_like(x)
    vb200.logits_process(x, out, rules)
    greedy = vb200.Sampler(temperature=0.0)
    assert greedy.sample(out[0]) == top[2]
