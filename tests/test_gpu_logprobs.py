"""Token log probabilities (forge_token_logprobs) against float64.

Tolerance: z - m is one rounding (2^-24 of |z - m|, which a probability's
exponent takes over), exp and log one part in 2^21, a sum of vocab terms over
threads and CTAs in trees of at most 64 steps each, 2^-24 a step: with D the
row's largest |z - m| among entries of any weight (below 90, or the term is
0), the LSE is off by at most (90 + 8 + 64) 2^-24 + 2^-24 |log s|, below
2^-16; a log probability by that and 2^-24 |z - m|, the entropy by twice that
times (1 + its size)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
T = 2.0 ** -16


def call(forge, torch, z, tok, top, ld=None, outs=("logprob", "entropy", "rank", "ids", "tops")):
    R, V = z.shape
    f = dict(logprob=torch.full((R,), 7.0), entropy=torch.full((R,), 7.0), rank=torch.full((R,), 7, dtype=torch.int32),
             ids=torch.full((R, top), 7, dtype=torch.int32), tops=torch.full((R, top), 7.0))
    f = {k: v.cuda() for k, v in f.items()}
    p = lambda k: f[k].data_ptr() if k in outs and f[k].numel() else None  # noqa: E731
    t = torch.tensor(tok, dtype=torch.int32, device="cuda") if tok is not None else None
    forge.check(forge.lib().forge_token_logprobs(
        z.data_ptr(), forge.FORGE_LOGITS_F32 if z.dtype == torch.float32 else forge.FORGE_LOGITS_BF16, z.stride(0), R, V,
        t.data_ptr() if t is not None else None, top, p("logprob"), p("entropy"), p("rank"), p("ids"), p("tops"),
        torch.cuda.current_stream().cuda_stream), "logprobs")
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in f.items()}


def check(z, tok, top, got):
    """z float64 numpy [R][V] of finite or -inf values."""
    R, V = z.shape
    for r in range(R):
        m = z[r].max()
        with np.errstate(all="ignore"):
            lp = (z[r] - m) - np.log(np.exp(z[r] - m).sum())  # m first: it may be the type's lowest value
            h = -np.where(np.isneginf(lp), 0, np.exp(lp) * lp).sum()
        order = np.lexsort((np.arange(V), -z[r]))  # larger first, equal ones by index
        y = tok[r]
        if y < 0:
            assert got["logprob"][r] == 0 and got["rank"][r] == -1
        else:
            assert got["rank"][r] == np.flatnonzero(order == y)[0], (r, got["rank"][r])
            if np.isneginf(lp[y]):
                assert np.isneginf(got["logprob"][r])
            else:
                assert abs(got["logprob"][r] - lp[y]) <= T + 2.0 ** -23 * abs(lp[y]), (r, got["logprob"][r], lp[y])
        assert abs(got["entropy"][r] - h) <= 2 * T * (1 + h), (r, got["entropy"][r], h)
        assert np.array_equal(got["ids"][r], order[:top]), (r, got["ids"][r], order[:top])
        want = lp[order[:top]]
        inf = np.isneginf(want)
        assert np.array_equal(np.isneginf(got["tops"][r]), inf)
        with np.errstate(all="ignore"):
            assert (np.abs(got["tops"][r] - want)[~inf] <= (T + 2.0 ** -23 * np.abs(want))[~inf]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,V,top,pad", [(1, 1, 1, 0), (1, 2, 2, 0), (3, 31, 5, 0), (2, 255, 32, 1), (5, 1000, 20, 3),
                                         (1, 32000, 5, 0), (7, 50257, 20, 0), (200, 4097, 7, 5), (1, 262144, 32, 0),
                                         (160, 33001, 0, 1), (400, 129, 32, 0)])
def test_logprobs(forge, cuda, dtype, R, V, top, pad):
    import torch
    g = torch.Generator().manual_seed(R * 7 + V)
    z = (torch.randn(R, V + pad, generator=g) * (1 + 4 * torch.rand(R, 1, generator=g)))
    z = z.to(torch.float32 if dtype == "f32" else torch.bfloat16)
    z[:, V:] = float("nan")  # the padding of a row is not read
    rng = np.random.default_rng(V)
    tok = rng.integers(0, V, R)
    tok[::3] = z[::3, :V].float().argmax(1).numpy()
    tok[R // 2] = -1 if R > 1 else tok[0]
    d = z.cuda()[:, :V]
    got = call(forge, torch, d, tok, top)
    forge.check(forge.lib().forge_ops_check(), "error word")
    check(z[:, :V].double().numpy(), tok, top, got)


@pytest.mark.parametrize("V", [40, 5000, 70001])
def test_ties_and_order(forge, cuda, V):
    """Equal logits by index: all equal, few distinct values, -0 and 0, ascending and descending rows."""
    import torch
    rng = np.random.default_rng(V)
    rows = [np.zeros(V), np.round(rng.standard_normal(V)), np.where(rng.random(V) < 0.5, -0.0, 0.0), np.arange(V) * 1e-3,
            -np.arange(V) * 1e-3, np.where(np.arange(V) >= V - 3, 2.0, 2.0 - 1e-6)]
    z = np.stack(rows).astype(np.float32)
    tok = [V - 1, V // 2, 3, V - 1, V - 1, 0]
    got = call(forge, torch, torch.from_numpy(z).cuda(), tok, 32)
    check(z.astype(np.float64), tok, 32, got)


def test_masked_logits(forge, cuda):
    """-inf and the type's lowest value as masks, few entries left, a single one, a token that is masked."""
    import torch
    V = 9001
    rng = np.random.default_rng(1)
    low = np.finfo(np.float32).min
    z = rng.standard_normal((5, V)).astype(np.float32) * 3
    z[0, rng.random(V) < 0.9] = -np.inf
    z[1, rng.random(V) < 0.9] = low
    z[2, :] = -np.inf
    z[2, 77] = -5.0
    z[3, :] = low
    z[4, :-4] = -np.inf
    tok = [int(np.flatnonzero(np.isneginf(z[0]))[5]), int(np.flatnonzero(z[1] > low)[2]), 77, 8000, 0]
    got = call(forge, torch, torch.from_numpy(z).cuda(), tok, 8)
    keep = [0, 2, 3, 4]
    check(z[keep].astype(np.float64), [tok[i] for i in keep], 8, {k: v[keep] for k, v in got.items()})
    check(np.where(z[1:2] == low, np.float64(low), z[1:2].astype(np.float64)), tok[1:2], 8,
          {k: v[1:2] for k, v in got.items()})


def test_rows_without_a_distribution(forge, cuda):
    """All -inf, a NaN, +inf: NaN log probabilities and entropy, ranked all the same; the rows beside them are right."""
    import torch
    V = 3000
    rng = np.random.default_rng(2)
    z = rng.standard_normal((5, V)).astype(np.float32)
    z[1] = -np.inf
    z[2, 1234] = np.nan
    z[3, 55] = np.inf
    tok = [10, 20, 30, 55, 40]
    got = call(forge, torch, torch.from_numpy(z).cuda(), tok, 4)
    check(z[[0, 4]].astype(np.float64), [10, 40], 4, {k: v[[0, 4]] for k, v in got.items()})
    for r in (1, 2, 3):
        assert np.isnan(got["logprob"][r]) and np.isnan(got["entropy"][r]) and np.isnan(got["tops"][r]).all()
    assert got["ids"][1].tolist() == [0, 1, 2, 3] and got["rank"][1] == 20
    order = np.lexsort((np.arange(V), -np.where(np.isnan(z[2]), -np.inf, z[2])))
    assert got["ids"][2].tolist() == order[:4].tolist() and got["rank"][2] == np.flatnonzero(order == 30)[0]
    assert got["ids"][3][0] == 55 and got["rank"][3] == 0


def test_optional_outputs_and_bad_tokens(forge, cuda):
    """Each output alone; a token outside the vocabulary sets the error word and gives NaN and rank -1."""
    import torch
    R, V = 3, 700
    z = torch.randn(R, V, generator=torch.Generator().manual_seed(1)).cuda()
    every = call(forge, torch, z, [1, 2, 3], 4)
    for k in ("logprob", "entropy", "rank"):
        got = call(forge, torch, z, [1, 2, 3], 0, outs=(k,))
        assert np.array_equal(got[k], every[k])
        assert all((got[o] == 7).all() for o in ("logprob", "entropy", "rank") if o != k)
    for outs in (("ids",), ("tops",), ("entropy", "ids")):
        got = call(forge, torch, z, None, 4, outs=outs)
        assert all(np.array_equal(got[k], every[k]) for k in outs)
        assert (got["logprob"] == 7).all() and (got["rank"] == 7).all()
    forge.check(forge.lib().forge_ops_check(), "error word")
    got = call(forge, torch, z, [1, V, 2147483647], 4)
    with pytest.raises(forge.ForgeError, match="error word"):
        forge.check(forge.lib().forge_ops_check(), "error word")
    assert got["logprob"][0] == every["logprob"][0] and np.isnan(got["logprob"][1:]).all()
    assert got["rank"].tolist() == [every["rank"][0], -1, -1]
    assert np.array_equal(got["ids"], every["ids"]) and np.array_equal(got["entropy"], every["entropy"])


def test_deterministic_streams_and_graph(forge, cuda):
    """The same bits every time, on another stream and from a graph; two calls at once do not disturb each other."""
    import torch
    R, V, top = 9, 32000, 20
    g = torch.Generator(device=cuda).manual_seed(3)
    zs = [torch.randn(R, V, generator=g, device=cuda) * 3 for _ in range(2)]
    tok = torch.arange(R, dtype=torch.int32, device=cuda) * 100
    outs = [[torch.zeros(R, device=cuda), torch.zeros(R, device=cuda), torch.zeros(R, dtype=torch.int32, device=cuda),
             torch.zeros(R, top, dtype=torch.int32, device=cuda), torch.zeros(R, top, device=cuda)] for _ in range(2)]

    def go(i):
        forge.check(forge.lib().forge_token_logprobs(zs[i].data_ptr(), 0, V, R, V, tok.data_ptr(), top,
                                                     *[o.data_ptr() for o in outs[i]],
                                                     torch.cuda.current_stream().cuda_stream), "logprobs")

    go(0)
    go(1)
    torch.cuda.synchronize()
    first = [[o.clone() for o in x] for x in outs]
    check(zs[0].cpu().double().numpy(), tok.tolist(), top,
          dict(zip(("logprob", "entropy", "rank", "ids", "tops"), (o.cpu().numpy() for o in first[0]))))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                go(i)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(0)
        go(1)
    for x, y in zip(outs, first):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
        [a.zero_() for a in x]
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(outs, first):
        assert all(torch.equal(a, b) for a, b in zip(x, y))
