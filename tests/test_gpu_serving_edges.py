"""Edges of the serving operators (4-bit KV cache, packed prefill, token log
probabilities): wide rows, captured graphs, concurrent streams, offsets past
32 bits, unusual values."""
import numpy as np
import pytest

import test_gpu_kv4 as kv4
import test_gpu_logprobs as lp
import test_gpu_prefill_varlen as pv

pytestmark = pytest.mark.gpu


# --------------------------------------------------------------- 4-bit cache
@pytest.mark.parametrize("n", [1, 3])
def test_append_wide_rows_in_a_graph(forge, cuda, n):
    """Rows of 40 heads of 128; a captured append and read whose positions and values change between replays."""
    import torch
    Hkv, hd = 40, 128
    w = Hkv * hd
    cache = kv4.Cache(forge, cuda, 2, Hkv, hd, 32, 16, seed=1, fill=False)
    L = forge.lib()
    dx = [torch.zeros(n, w, dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    ds, dp = (torch.zeros(n, dtype=torch.int32, device=cuda) for _ in range(2))
    out = [torch.zeros(n, w, device=cuda) for _ in range(2)]

    def call():
        forge.check(L.forge_kv4_append(cache.desc, dx[0].data_ptr(), dx[1].data_ptr(), w, ds.data_ptr(), dp.data_ptr(),
                                       n, kv4.stream()), "append")
        forge.check(L.forge_kv4_read(cache.desc, ds.data_ptr(), dp.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(),
                                     w, kv4.stream()), "read")

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = np.random.default_rng(2)
    for i in range(3):
        x = [kv4.bf16(rng.standard_normal((n, Hkv, hd)).astype(np.float32)) for _ in range(2)]
        for d, a in zip(dx, x):
            d.copy_(torch.from_numpy(a.reshape(n, w)))
        ds.copy_(torch.full((n,), i % 2, dtype=torch.int32))
        dp.copy_(torch.arange(i * n, i * n + n, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for kv in range(2):
            want = kv4.values(*kv4.quantise(x[kv])).astype(np.float32)
            assert np.array_equal(out[kv].cpu().numpy().reshape(n, Hkv, hd), want)
    forge.check(forge.lib().forge_ops_check(), "error word")


def test_decode_with_large_query_channels(forge, cuda):
    """A few channels of q far above the rest. q is rounded to 2^-23 of its largest channel, which adds
    2 * 2^-23 max|q| sum|k| / sqrt(hd) to a score's error (twice, for its two sides), and four times that, in
    relative terms, to the output."""
    B, H, Hkv, hd, n = 3, 8, 2, 128, 500
    rng = np.random.default_rng(5)
    cache = kv4.Cache(forge, cuda, B, Hkv, hd, 512, 0, seed=5)
    q = rng.standard_normal((B, H, hd)).astype(np.float32) * np.float32(0.2)
    q[:, :, 17] *= 100
    q[1, :, 100] *= -300
    pos = [n - 1, 63, 200]
    out, tol = kv4.reference(cache, q, pos)
    for b in range(B):
        k, v = (cache.row(kv, b, pos[b] + 1) for kv in range(2))
        for h in range(H):
            kh, vh = k[:, h // 4], v[:, h // 4]
            tol[b, h] += np.abs(vh).max() * 4 * 2 * kv4.U * np.abs(q[b, h]).max() * np.abs(kh).sum(1).max() / np.sqrt(hd)
    kv4.check(kv4.decode(forge, cuda, cache, q, pos), (out, tol))


@pytest.mark.parametrize("hd,H,Hkv", [(64, 4, 4), (64, 6, 3), (128, 8, 4), (128, 2, 1), (64, 1, 1), (64, 9, 3)])
@pytest.mark.parametrize("page", [0, 8, 24])
def test_decode_few_heads(forge, cuda, hd, H, Hkv, page):
    """One, two and three query heads a KV head, at lengths around every boundary and long ones that CTAs share."""
    pos = [0, -1, 1, 6, 7, 8, 15, 16, 31, 32, 47, 62, 63, 64, 65, 127, 128, 500, 1151, 1100]
    cache = kv4.Cache(forge, cuda, len(pos), Hkv, hd, 1152, page, seed=hd + H)
    q = np.random.default_rng(H).standard_normal((len(pos), H, hd)).astype(np.float32) * 2
    got = kv4.decode(forge, cuda, cache, q, pos)
    forge.check(forge.lib().forge_ops_check(), "error word")
    kv4.check(got, kv4.reference(cache, q, pos))
    assert (got[1] == 0).all()


@pytest.mark.parametrize("hd,H,Hkv", [(128, 2, 2), (64, 4, 2)])
def test_decode_few_heads_masked_rows(forge, cuda, hd, H, Hkv):
    """NaN scales behind the last position are not seen; a NaN or an infinity in q is its own head's; a NaN scale of V its
    group's."""
    import torch
    G = H // Hkv
    cache = kv4.Cache(forge, cuda, 2, Hkv, hd, 256, 0, seed=12)
    pos = [77, 200]
    q = np.random.default_rng(7).standard_normal((2, H, hd)).astype(np.float32)
    want = kv4.reference(cache, q, pos)
    for kv in range(2):
        s = cache.scales[kv].copy()
        for b, p in enumerate(pos):
            s[b, :, p + 1:] = np.nan
        cache.d[2 + kv].copy_(torch.from_numpy(kv4.bits16(s).view(np.int16)))
    kv4.check(kv4.decode(forge, cuda, cache, q, pos), want)
    bad = q.copy()
    bad[0, 0, 3], bad[1, H - 1, 9] = np.nan, np.inf
    got = kv4.decode(forge, cuda, cache, bad, pos)
    nan = np.isnan(got)
    assert nan[0, 0].all() and nan[1, H - 1].all() and not nan[0, 1:].any() and not nan[1, :H - 1].any()
    cache.d[3].view(*cache.scales[1].shape)[1, 0, 40, -1] = 0x7FC0
    got = kv4.decode(forge, cuda, cache, q, pos)
    assert np.isnan(got[1, :G, -64:]).all() and np.isfinite(got[1, :G, :-64]).all()
    assert np.isfinite(got[0]).all() and np.isfinite(got[1, G:]).all()


def test_decode_forty_heads_of_one_kv_head(forge, cuda):
    cache = kv4.Cache(forge, cuda, 2, 1, 64, 3000, 8, seed=6)
    q = np.random.default_rng(6).standard_normal((2, 41, 64)).astype(np.float32)
    kv4.check(kv4.decode(forge, cuda, cache, q, [2900, 64]), kv4.reference(cache, q, [2900, 64]))


@pytest.mark.parametrize("H,Hkv", [(64, 16), (32, 32)])
def test_decode_workspace_of_the_largest_batch(forge, cuda, H, Hkv):
    """One workspace, sized for the largest batch, for batches of several sizes in turn."""
    import torch
    hd, most = 64, 40
    cache = kv4.Cache(forge, cuda, 4, Hkv, hd, 640, 0, seed=13)
    q = np.random.default_rng(13).standard_normal((most, H, hd)).astype(np.float32)
    pos, seq = [639 - 7 * b for b in range(most)], [b % 4 for b in range(most)]
    out, tol = kv4.reference(cache, q, pos, seq)
    ws = torch.zeros(forge.lib().forge_flash_decode_kv4_workspace_bytes(most, H, Hkv, hd), dtype=torch.uint8, device=cuda)
    for B in (1, 3, 40, 2, 17, 40):
        kv4.check(kv4.decode(forge, cuda, cache, q[:B], pos[:B], seq[:B], ws), (out[:B], tol[:B]))


def test_decode_on_two_streams_at_once(forge, cuda):
    """Two calls in flight, each with its own workspace, repeated."""
    import torch
    L = forge.lib()
    runs = []
    for seed, (B, H, Hkv, hd, n) in enumerate([(4, 8, 2, 128, 3000), (6, 4, 4, 64, 2000)]):
        cache = kv4.Cache(forge, cuda, B, Hkv, hd, n, 0, seed=seed)
        q = np.random.default_rng(seed).standard_normal((B, H, hd)).astype(np.float32)
        pos = [n - 1 - 37 * b for b in range(B)]
        runs.append(dict(cache=cache, q=q, pos=pos, dims=(B, H), dq=torch.from_numpy(q.reshape(B, -1)).to(cuda),
                         dp=torch.tensor(pos, dtype=torch.int32, device=cuda),
                         out=torch.zeros(B, H * hd, device=cuda), stream=torch.cuda.Stream(),
                         ws=torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd), dtype=torch.uint8,
                                        device=cuda)))
    torch.cuda.synchronize()
    for _ in range(20):
        for r in runs:
            forge.check(L.forge_flash_decode_kv4(r["dq"].data_ptr(), r["cache"].desc, None, r["dp"].data_ptr(),
                                                 *r["dims"], r["out"].data_ptr(), r["ws"].data_ptr(),
                                                 r["stream"].cuda_stream), "decode")
    torch.cuda.synchronize()
    for r in runs:
        kv4.check(r["out"].cpu().numpy().reshape(r["q"].shape), kv4.reference(r["cache"], r["q"], r["pos"]))


@pytest.mark.parametrize("page", [0, 64])
def test_cache_past_32_bits(forge, cuda, page):
    """Sequences whose rows lie more than 2^32 bytes into the arrays: append, read and decode."""
    import torch
    Hkv, hd, lmax, n = 20, 64, 1 << 22, 70
    rows = 2 * Hkv * lmax
    assert (2 * Hkv - 1) * lmax * (hd // 2) > 1 << 32
    d = [torch.empty(rows * w, dtype=torch.uint8, device=cuda) for w in (hd // 2, hd // 2, 2, 2)]
    per = lmax // page if page else 0
    table = None
    if page:  # sequence 1's first pages are the pool's last
        table = torch.arange(2 * per - 1, -1, -1, dtype=torch.int32, device=cuda).view(2, per).flip(0).contiguous()
    cache = forge.ForgeKv4(k=d[0].data_ptr(), v=d[1].data_ptr(), ks=d[2].data_ptr(), vs=d[3].data_ptr(),
                           table=table.data_ptr() if page else None, n_seq=2, n_kv_head=Hkv, head_dim=hd,
                           lmax=0 if page else lmax, page_tokens=page, max_pages=per, num_pages=2 * per)
    rng = np.random.default_rng(9)
    x = [kv4.bf16(rng.standard_normal((n, Hkv, hd)).astype(np.float32)) for _ in range(2)]
    dx = [torch.from_numpy(a.reshape(n, -1)).to(cuda).to(torch.bfloat16) for a in x]
    ds = torch.ones(n, dtype=torch.int32, device=cuda)
    dp = torch.arange(n, dtype=torch.int32, device=cuda)
    L = forge.lib()
    forge.check(L.forge_kv4_append(cache, dx[0].data_ptr(), dx[1].data_ptr(), Hkv * hd, ds.data_ptr(), dp.data_ptr(), n,
                                   kv4.stream()), "append")
    out = [torch.zeros(n, Hkv * hd, device=cuda) for _ in range(2)]
    forge.check(L.forge_kv4_read(cache, ds.data_ptr(), dp.data_ptr(), n, out[0].data_ptr(), out[1].data_ptr(), Hkv * hd,
                                 kv4.stream()), "read")
    host = [kv4.values(*kv4.quantise(a)) for a in x]
    for kv in range(2):
        assert np.array_equal(out[kv].cpu().numpy().reshape(n, Hkv, hd), host[kv].astype(np.float32))

    class Host:  # (what the reference reads)
        pass

    h = Host()
    h.Hkv, h.row = Hkv, lambda kv, seq, m: host[kv][:m]
    q = rng.standard_normal((1, Hkv, hd)).astype(np.float32)
    dq = torch.from_numpy(q.reshape(1, -1)).to(cuda)
    ws = torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(1, Hkv, Hkv, hd), dtype=torch.uint8, device=cuda)
    o = torch.zeros(1, Hkv * hd, device=cuda)
    forge.check(L.forge_flash_decode_kv4(dq.data_ptr(), cache, ds.data_ptr(), dp[n - 1:].data_ptr(), 1, Hkv,
                                         o.data_ptr(), ws.data_ptr(), kv4.stream()), "decode")
    torch.cuda.synchronize()
    forge.check(L.forge_ops_check(), "error word")
    kv4.check(o.cpu().numpy().reshape(1, Hkv, hd), kv4.reference(h, q, [n - 1]))


# ------------------------------------------------------------ packed prefill
def test_prefill_wide_batch(forge, cuda):
    """K and V of all heads larger than half of L2: heads go in groups."""
    import torch
    H, hd, lens = 32, 128, [1025, 900, 2000, 1, 1500, 1024, 2100]
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = pv.make(torch, cuda, cu[-1], H, H, hd, seed=1)
    o = torch.full((cu[-1], H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
    lse = torch.full((H, cu[-1]), float("nan"), device=cuda)
    pv.run(forge, cuda, q, k, v, cu, H, H, hd, o, lse)
    forge.check(forge.lib().forge_ops_check(), "error word")
    pv.check(torch, q, k, v, cu, H, H, hd, o, lse)


def test_prefill_many_sequences_of_all_lengths(forge, cuda):
    import torch
    H, Hkv, hd, lens = 4, 2, 64, [3] * 50 + [900] + [1, 0] * 40 + [700] + [130] * 70 + [2048]
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = pv.make(torch, cuda, cu[-1], H, Hkv, hd, seed=2)
    o = torch.full((cu[-1], H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
    lse = torch.full((H, cu[-1]), float("nan"), device=cuda)
    pv.run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, lse)
    forge.check(forge.lib().forge_ops_check(), "error word")
    pv.check(torch, q, k, v, cu, H, Hkv, hd, o, lse)


def test_prefill_single_nan(forge, cuda):
    """A NaN key makes the rows that see it NaN and no other; a NaN query its own row and head."""
    import torch
    H, Hkv, hd, n, at, row = 4, 2, 128, 400, 150, 300
    q, k, v = pv.make(torch, cuda, n, H, Hkv, hd, seed=3)
    o = torch.zeros(n, H * hd, dtype=torch.bfloat16, device=cuda)
    lse = torch.zeros(H, n, device=cuda)
    clean = [x.clone() for x in (q, k, v)]
    k[at, 5] = float("nan")  # KV head 0: query heads 0 and 1
    q[row, 3 * hd + 7] = float("nan")
    pv.run(forge, cuda, q, k, v, [0, n], H, Hkv, hd, o, lse)
    bad = torch.isnan(o).view(n, H, hd)
    assert torch.isnan(lse[:2, at:]).all() and bad[at:, :2].all()
    assert bad[row, 3].all() and torch.isnan(lse[3, row])
    o2, lse2 = torch.zeros_like(o), torch.zeros_like(lse)
    pv.run(forge, cuda, *clean, [0, n], H, Hkv, hd, o2, lse2)
    good = ~bad
    assert torch.equal(o.view(n, H, hd)[good], o2.view(n, H, hd)[good])
    assert good[:at].all() and good[:, 2].all() and good[:row, 3].all() and good[row + 1:, 3].all()


def test_prefill_rows_past_32_bits(forge, cuda):
    """Row strides that put the last rows more than 2^32 bytes behind the first."""
    import torch
    H, Hkv, hd, lens = 2, 1, 64, [130, 70]
    ld, total = 1 << 24, 200
    buf = torch.empty(total * ld, dtype=torch.bfloat16, device=cuda)
    x = buf.as_strided((total, (H + 2 * Hkv) * hd), (ld, 1))
    x.copy_(torch.randn(total, (H + 2 * Hkv) * hd, generator=torch.Generator().manual_seed(4)))
    q, k, v = x[:, :H * hd], x[:, H * hd:(H + Hkv) * hd], x[:, (H + Hkv) * hd:]
    o = buf.as_strided((total, H * hd), (ld, 1), 1024)
    lse = torch.zeros(H, total, device=cuda)
    cu = [0, 130, 200]
    pv.run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, lse)
    forge.check(forge.lib().forge_ops_check(), "error word")
    pv.check(torch, q, k, v, cu, H, Hkv, hd, o, lse)


# ------------------------------------------------------ token log probabilities
@pytest.mark.parametrize("R", [1, 700])
def test_rising_and_flat_bf16_rows(forge, cuda, R):
    """Rows that overflow the candidate list: rising, with every value many times; a row shared by CTAs and not."""
    import torch
    V = 40003
    z = torch.stack([(torch.arange(V) * 1e-3).to(torch.bfloat16), torch.ones(V, dtype=torch.bfloat16),
                     (-torch.arange(V) * 1e-3).to(torch.bfloat16)])[torch.arange(R) % 3].contiguous()
    tok = [V - 1 - 100 * (r % 7) for r in range(R)]
    got = lp.call(forge, torch, z.cuda(), tok, 32)
    some = list(range(min(R, 9)))
    lp.check(z[some].double().numpy(), [tok[r] for r in some], 32, {k: v[some] for k, v in got.items()})
    for r in range(R):  # every third row the same but for its token and, by alignment, the order of its sums
        assert np.array_equal(got["ids"][r], got["ids"][r % 3])
        assert (np.abs(got["tops"][r] - got["tops"][r % 3]) <= 2 * (lp.T + 2.0 ** -23 * np.abs(got["tops"][r]))).all()
        assert abs(got["entropy"][r] - got["entropy"][r % 3]) <= 4 * lp.T * (1 + got["entropy"][r])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [1, 8, 20, 32])
def test_best_logits_in_one_stretch(forge, cuda, dtype, top):
    """All the best entries in one stretch of 1024 vectors of the row, one or two to a vector, whichever stretch it is:
    where a threshold is taken from them, the last of them equals it."""
    import torch
    per = 4 if dtype == "f32" else 8
    V, R = 1024 * per * 10 + 5, 11
    z = torch.rand(R, V, generator=torch.Generator().manual_seed(6))
    for r in range(R):
        for j in range(top):
            at = min(V - 1, (1024 * r + (j * 37) % 256 + 256 * (j % 4)) * per + (j * 5) % per)
            z[r, at] = 4 + j / 16
    z = z.to(torch.float32 if dtype == "f32" else torch.bfloat16)
    pad = (-V) % 8  # every row starts on 16 bytes
    d = torch.zeros(R, V + pad, dtype=z.dtype, device=cuda)
    d[:, :V] = z
    many = d.repeat(60, 1)[:, :V]  # enough rows for a CTA each
    tok = [(97 * r) % V for r in range(60 * R)]
    got = lp.call(forge, torch, many, tok, top)
    lp.check(z.double().numpy(), tok[:R], top, {k: v[:R] for k, v in got.items()})
    for r in range(R, 60 * R):
        assert np.array_equal(got["ids"][r], got["ids"][r % R])


def test_logits_far_from_zero(forge, cuda):
    """Maxima far from 0, where a logit times log2 e has no room for a fraction, or is no fp32 number."""
    import torch
    V = 3001
    z = np.random.default_rng(3).standard_normal((8, V)).astype(np.float32)
    z[0, 5] = z[0, 2000] = 3.3e38
    z[1] = np.float32(-3.3e38)
    z[1, 9] = np.float32(-3.0e38)
    z[2] *= np.float32(1e37)
    z[3] = -np.float32(2e29) * (1 + np.arange(V) % 7)
    for r, far in ((4, 3e5), (5, -9e5), (6, 5e6), (7, -1e12)):
        z[r] += np.float32(far)
    tok = [2000, 9, int(z[2].argmax()), 0, 5, 6, 7, 8]
    got = lp.call(forge, torch, torch.from_numpy(z).cuda(), tok, 4)
    with np.errstate(all="ignore"):
        z64 = z.astype(np.float64)
        l = z64 - z64.max(1, keepdims=True)
        l -= np.log(np.exp(l).sum(1, keepdims=True))
    for r in range(8):
        order = np.lexsort((np.arange(V), -z64[r]))[:4]
        assert np.array_equal(got["ids"][r], order)
        for a, b in [(got["logprob"][r], l[r, tok[r]])] + list(zip(got["tops"][r], l[r, order])):
            assert abs(a - b) <= lp.T + 2.0 ** -23 * abs(b)
        p = np.exp(l[r])
        h = -(p[p > 0] * l[r][p > 0]).sum()
        assert abs(got["entropy"][r] - h) <= 2 * lp.T * (1 + h)


def test_rows_past_32_bits(forge, cuda):
    """A row stride that puts the last rows more than 2^32 elements behind the first."""
    import torch
    V, ld = 5001, (1 << 30) + (1 << 29) + 3
    buf = torch.empty(3 * ld + V, dtype=torch.bfloat16, device=cuda)
    z = buf.as_strided((4, V), (ld, 1))
    z.copy_(torch.randn(4, V, generator=torch.Generator().manual_seed(5)))
    tok = [1, 5000, 77, 4321]
    got = lp.call(forge, torch, z, tok, 8)
    lp.check(z.double().cpu().numpy(), tok, 8, got)
