"""The 4-bit KV cache on the B200 (forge_kv4_append, forge_kv4_read,
forge_flash_decode_kv4) against plain float64 code.

Codes and scales are exact: they equal forge_q4_quantize_bf16's with group 64
and a restatement of the rule. The attention's tolerance follows from its
arithmetic. With u = 2^-23 (one step of a truncating fp32 sum), a score of hd
products is off by at most ds = (hd + 4) u sum|q k| / sqrt(hd) (hd sums, and q
rounded to 2^-23 of its largest channel, below 4 times the mean); a probability
relative to the largest by 2 ds + 8 u max|s| (the exponent's argument and its
exp2); a sum over n keys in tiles by (64 + n / 64) u; so the output by
vmax (4 ds + (16 smax + 2 (64 + n / 64) + 16) u), vmax the largest |v|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -23


def quantise(x):
    """float32 rows [..., hd] -> (codes [..., hd / 2] uint8, scale [..., hd / 64] float32 of bf16 value)."""
    g = x.reshape(*x.shape[:-1], -1, 64).astype(np.float32)
    amax = np.abs(g).max(-1)
    with np.errstate(all="ignore"):
        s = bf16(amax / np.float32(7))
        s = np.where(s == 0, np.float32(1), s)
        q = g.astype(np.float64) / s[..., None]
        c = np.clip(np.trunc(q + np.where(q < 0, -0.5, 0.5)), -7, 7) + 7
    finite = np.isfinite(g).all(-1)
    s = np.where(finite, s, np.float32("nan"))
    c = np.where(finite[..., None], c, 7).reshape(x.shape).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), s


def bf16(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32)
    return np.where(np.isfinite(x), r, x).astype(np.float32)


def bits16(x):
    return (np.ascontiguousarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)


def values(codes, s):
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(np.float64) - 7
    return (c.reshape(*c.shape[:-1], -1, 64) * s[..., None].astype(np.float64)).reshape(c.shape)


class Cache:
    """A cache on the GPU, its host copy and its descriptor."""

    def __init__(self, forge, cuda, n_seq, Hkv, hd, rows, page=0, seed=0, fill=True, spare=3):
        import torch
        rng = np.random.default_rng(seed)
        self.forge, self.n_seq, self.Hkv, self.hd, self.rows, self.page = forge, n_seq, Hkv, hd, rows, page
        per = -(-rows // page) if page else 0
        self.pages = n_seq * per + spare if page else 0
        shape = (self.pages, Hkv, page) if page else (n_seq, Hkv, rows)
        self.table = rng.permutation(self.pages)[:n_seq * per].reshape(n_seq, per).astype(np.int32) if page else None
        self.codes, self.scales = [], []
        for kv in range(2):
            if fill:
                c, s = quantise(bf16(rng.standard_normal(shape + (hd,)).astype(np.float32)))
            else:
                c, s = np.full(shape + (hd // 2,), 0xEE, np.uint8), np.full(shape + (hd // 64,), np.nan, np.float32)
            self.codes.append(c)
            self.scales.append(s)
        self.d = [torch.from_numpy(c).to(cuda) for c in self.codes] + \
                 [torch.from_numpy(bits16(s).view(np.int16)).to(cuda) for s in self.scales]
        self.dt = torch.from_numpy(self.table).to(cuda) if page else None
        self.desc = forge.ForgeKv4(k=self.d[0].data_ptr(), v=self.d[1].data_ptr(), ks=self.d[2].data_ptr(),
                                   vs=self.d[3].data_ptr(), table=self.dt.data_ptr() if page else None, n_seq=n_seq,
                                   n_kv_head=Hkv, head_dim=hd, lmax=0 if page else rows, page_tokens=page,
                                   max_pages=per, num_pages=self.pages)

    def at(self, seq, pos):
        return (int(self.table[seq, pos // self.page]), pos % self.page) if self.page else (seq, pos)

    def row(self, kv, seq, n):
        """Values [n][Hkv][hd] of the first n rows."""
        return np.stack([values(self.codes[kv][i, :, j], self.scales[kv][i, :, j])
                         for i, j in (self.at(seq, p) for p in range(n))])

    def device(self):
        return [t.cpu().numpy() for t in self.d[:2]], [t.cpu().numpy().view(np.uint16) for t in self.d[2:]]


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def append(forge, cuda, cache, x, seq, pos, ld=None):
    import torch
    n = x[0].shape[0]
    w = cache.Hkv * cache.hd
    ld = ld or w
    dev = []
    for a in x:
        full = np.full((n, ld), 0x7FC0, np.uint16)
        full[:, :w] = bits16(a).reshape(n, w)
        dev.append(torch.from_numpy(full.view(np.int16)).to(cuda))
    ds = torch.tensor(seq, dtype=torch.int32, device=cuda) if seq is not None else None
    dp = torch.tensor(pos, dtype=torch.int32, device=cuda)
    forge.check(forge.lib().forge_kv4_append(cache.desc, dev[0].data_ptr(), dev[1].data_ptr(), ld,
                                             ds.data_ptr() if ds is not None else None, dp.data_ptr(), n, stream()),
                "append")
    torch.cuda.synchronize()


def decode(forge, cuda, cache, q, pos, seq=None, ws=None):
    import torch
    B, H = q.shape[:2]
    L = forge.lib()
    dq = torch.from_numpy(q.reshape(B, -1)).to(cuda)
    dp = torch.tensor(pos, dtype=torch.int32, device=cuda)
    ds = torch.tensor(seq, dtype=torch.int32, device=cuda) if seq is not None else None
    out = torch.full((B, H * cache.hd), 77.0, device=cuda)
    if ws is None:
        ws = torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(B, H, cache.Hkv, cache.hd), dtype=torch.uint8,
                         device=cuda)
    forge.check(L.forge_flash_decode_kv4(dq.data_ptr(), cache.desc, ds.data_ptr() if seq is not None else None,
                                         dp.data_ptr(), B, H, out.data_ptr(), ws.data_ptr(), stream()), "decode")
    torch.cuda.synchronize()
    return out.cpu().numpy().reshape(B, H, cache.hd)


def reference(cache, q, pos, seq=None):
    """(output, tolerance) [B][H][hd] in float64."""
    B, H, hd = q.shape
    G = H // cache.Hkv
    out, tol = np.zeros((B, H, hd)), np.zeros((B, H, 1))
    for b in range(B):
        n = pos[b] + 1
        if n <= 0:
            continue
        k, v = (cache.row(kv, seq[b] if seq is not None else b, n) for kv in range(2))
        for h in range(H):
            qh, kh, vh = q[b, h].astype(np.float64), k[:, h // G], v[:, h // G]
            s = kh @ qh / np.sqrt(hd)
            with np.errstate(all="ignore"):
                p = np.exp(s - s.max())
                out[b, h] = p @ vh / p.sum()
                ds = (hd + 4) * U * (np.abs(kh) @ np.abs(qh)).max() / np.sqrt(hd)
                tol[b, h] = np.abs(vh).max() * (4 * ds + (16 * np.abs(s).max() + 2 * (64 + n / 64) + 16) * U)
    return out, tol


def check(got, want):
    out, tol = want
    assert np.isfinite(got).all()
    err = np.abs(got - out)
    assert (err <= tol).all(), (err.max(), np.unravel_index((err - tol).argmax(), err.shape))


# ------------------------------------------------------------ append and read
@pytest.mark.parametrize("hd,Hkv,page,n,ld", [(128, 2, 0, 5, 0), (64, 3, 8, 37, 0), (128, 1, 16, 1, 136),
                                              (64, 8, 0, 300, 1024), (128, 5, 64, 130, 656)])
def test_append_and_read(forge, cuda, hd, Hkv, page, n, ld):
    import torch
    rng = np.random.default_rng(hd + n)
    cache = Cache(forge, cuda, 4, Hkv, hd, 128, page, seed=n, fill=False)
    x = [bf16((rng.standard_normal((n, Hkv, hd)) * np.exp(rng.uniform(-3, 3, (n, Hkv, 1)))).astype(np.float32))
         for _ in range(2)]
    where = rng.permutation(4 * 128)[:n]
    seq, pos = where // 128, where % 128
    pos[n // 2] = -1 if n > 1 else pos[0]  # a padding row
    append(forge, cuda, cache, x, seq, pos, ld or None)
    for kv in range(2):
        c, s = quantise(x[kv])
        for r in range(n):
            if pos[r] >= 0:
                i, j = cache.at(int(seq[r]), int(pos[r]))
                cache.codes[kv][i, :, j], cache.scales[kv][i, :, j] = c[r], s[r]
    codes, scales = cache.device()
    for kv in range(2):  # every byte: the rows named, and no other
        assert np.array_equal(codes[kv], cache.codes[kv])
        assert np.array_equal(scales[kv], bits16(cache.scales[kv]))
    w = Hkv * hd
    out = [torch.full((n, w + 4), 5.0, device=cuda) for _ in range(2)]
    ds, dp = (torch.tensor(a, dtype=torch.int32, device=cuda) for a in (seq, pos))
    forge.check(forge.lib().forge_kv4_read(cache.desc, ds.data_ptr(), dp.data_ptr(), n, out[0].data_ptr(),
                                           out[1].data_ptr(), w + 4, stream()), "read")
    torch.cuda.synchronize()
    forge.check(forge.lib().forge_ops_check(), "error word")
    for kv in range(2):
        o = out[kv].cpu().numpy()
        assert (o[:, w:] == 5.0).all()
        for r in range(n):
            if pos[r] < 0:
                assert (o[r] == 5.0).all()
            else:
                i, j = cache.at(int(seq[r]), int(pos[r]))
                want = values(cache.codes[kv][i, :, j], cache.scales[kv][i, :, j]).astype(np.float32)
                assert np.array_equal(o[r, :w].reshape(Hkv, hd), want)


def test_append_is_the_int4_weights_rule(forge, cuda):
    """forge_q4_quantize_bf16 with group 64 gives the same codes and scales."""
    import torch
    rng = np.random.default_rng(3)
    n, Hkv, hd = 64, 4, 128
    x = [bf16(rng.standard_normal((n, Hkv, hd)).astype(np.float32)) for _ in range(2)]
    x[0][0] = 0.0
    x[0][1] = np.float32(2.0 ** -133)  # bf16 subnormals: a scale of 0
    x[0][2, :, 0], x[0][2, :, 1:] = 7.0, 0.5  # scale 1: exact halves
    x[0][3, :, 0], x[0][3, :, 1:] = 7.0, -2.5
    cache = Cache(forge, cuda, 1, Hkv, hd, 64, fill=False)
    append(forge, cuda, cache, x, [0] * n, list(range(n)))
    codes, scales = cache.device()
    for kv in range(2):
        w = torch.from_numpy(bits16(x[kv].transpose(1, 0, 2)).reshape(n * Hkv, hd).view(np.int16)).to(cuda)
        c = torch.zeros(n * Hkv, hd // 2, dtype=torch.uint8, device=cuda)
        s = torch.zeros(n * Hkv, hd // 64, dtype=torch.int16, device=cuda)
        forge.check(forge.lib().forge_q4_quantize_bf16(w.data_ptr(), n * Hkv, hd, 64, c.data_ptr(), s.data_ptr(),
                                                       stream()), "quantize")
        torch.cuda.synchronize()
        assert np.array_equal(codes[kv].reshape(n * Hkv, -1), c.cpu().numpy())
        assert np.array_equal(scales[kv].reshape(n * Hkv, -1), s.cpu().numpy().view(np.uint16))


def test_append_extreme_values(forge, cuda):
    """NaN and infinities give a NaN group and spare its neighbours; the largest and smallest bf16 values."""
    hd, Hkv = 128, 1
    x = [np.ones((6, Hkv, hd), np.float32) for _ in range(2)]
    x[0][0, 0, 5] = np.nan
    x[0][1, 0, 70] = np.inf
    x[0][2, 0, 127] = -np.inf
    x[0][3] = bf16(np.float32(3.38e38))
    x[0][4, 0, :] = np.float32(2.0 ** -126) * np.arange(128, dtype=np.float32).clip(0, 127)
    x[0][4] = bf16(x[0][4])
    x[0][5] = -0.0
    cache = Cache(forge, cuda, 1, Hkv, hd, 8, fill=False)
    append(forge, cuda, cache, x, [0] * 6, list(range(6)))
    codes, scales = cache.device()
    c, s = quantise(x[0])
    got = scales[0][0, 0, :6]
    assert np.array_equal(np.isnan(s[:, 0]), (got & 0x7FFF) > 0x7F80)
    ok = ~np.isnan(s[:, 0])
    assert np.array_equal(got[ok], bits16(s[:, 0])[ok])
    assert np.array_equal(codes[0][0, 0, :6], c[:, 0])


@pytest.mark.parametrize("page", [0, 16])
def test_append_and_read_out_of_range(forge, cuda, page):
    import torch
    hd, Hkv = 64, 2
    cache = Cache(forge, cuda, 2, Hkv, hd, 64, page, seed=1, spare=0)
    if page:  # sequence 1's second page is outside the pool
        cache.dt[1, 1] = cache.pages + 100
    x = [np.ones((4, Hkv, hd), np.float32) for _ in range(2)]
    cases = [([0, 1, 2, 0], [64, 1 << 30, 3, 2147483647]), ([-1, 0, 0, 0], [0, -1, -5, -2147483648])]
    if page:
        cases.append(([1, 1, -7, 1], [16, 31, 0, 20]))
    for seq, pos in cases:
        append(forge, cuda, cache, x, seq, pos)
        with pytest.raises(forge.ForgeError, match="error word"):
            forge.check(forge.lib().forge_ops_check(), "error word")
        codes, scales = cache.device()
        for kv in range(2):
            assert np.array_equal(codes[kv], cache.codes[kv]) and np.array_equal(scales[kv], bits16(cache.scales[kv]))
        out = [torch.full((4, Hkv * hd), 5.0, device=cuda) for _ in range(2)]
        ds, dp = (torch.tensor(a, dtype=torch.int32, device=cuda) for a in (seq, pos))
        forge.check(forge.lib().forge_kv4_read(cache.desc, ds.data_ptr(), dp.data_ptr(), 4, out[0].data_ptr(),
                                               out[1].data_ptr(), Hkv * hd, stream()), "read")
        torch.cuda.synchronize()
        with pytest.raises(forge.ForgeError, match="error word"):
            forge.check(forge.lib().forge_ops_check(), "error word")
        for r in range(4):
            assert (out[0][r] == 5.0).all() if pos[r] < 0 else torch.isnan(out[0][r]).all()


# -------------------------------------------------------------------- decode
@pytest.mark.parametrize("hd,H,Hkv", [(128, 4, 4), (64, 4, 1), (128, 8, 2), (64, 6, 2), (128, 14, 2), (64, 8, 1),
                                      (128, 11, 1), (64, 24, 1)])
@pytest.mark.parametrize("page", [0, 8, 48])
def test_decode(forge, cuda, hd, H, Hkv, page):
    """Lengths of zero, one, inside, at and behind every boundary of 16, 32, 64, 128 and 256 keys."""
    pos = [0, -1, 1, 14, 15, 16, 31, 32, 62, 63, 64, 65, 127, 128, 254, 255, 256, 300, 383]
    cache = Cache(forge, cuda, len(pos), Hkv, hd, 384, page, seed=hd + H)
    rng = np.random.default_rng(H)
    q = rng.standard_normal((len(pos), H, hd)).astype(np.float32) * 2
    got = decode(forge, cuda, cache, q, pos)
    forge.check(forge.lib().forge_ops_check(), "error word")
    check(got, reference(cache, q, pos))
    assert (got[1] == 0).all()


@pytest.mark.parametrize("B,H,Hkv,hd,n,page", [(1, 32, 32, 128, 2048, 0), (1, 8, 1, 128, 20000, 16),
                                               (3, 8, 2, 64, 5000, 64), (1, 1, 1, 64, 40000, 0)])
def test_decode_long(forge, cuda, B, H, Hkv, hd, n, page):
    """Long sequences, split over CTAs and joined."""
    pos = [n - 1 - 777 * b for b in range(B)]
    cache = Cache(forge, cuda, B, Hkv, hd, (n + 63) // 64 * 64, page, seed=n)
    q = np.random.default_rng(n).standard_normal((B, H, hd)).astype(np.float32)
    check(decode(forge, cuda, cache, q, pos), reference(cache, q, pos))


def test_decode_many_sequences(forge, cuda):
    """More sequences than a scan's width, most of them short, some empty, named by seq in another order."""
    B, H, Hkv, hd, n_seq = 333, 4, 2, 64, 7
    rng = np.random.default_rng(8)
    cache = Cache(forge, cuda, n_seq, Hkv, hd, 512, 32, seed=9)
    pos = np.where(rng.random(B) < 0.2, -1, np.minimum(511, np.exp(rng.uniform(0, 6.3, B)).astype(int))).tolist()
    seq = rng.integers(0, n_seq, B).tolist()
    q = rng.standard_normal((B, H, hd)).astype(np.float32)
    check(decode(forge, cuda, cache, q, pos, seq), reference(cache, q, pos, seq))


def test_decode_scores_and_values_of_any_size(forge, cuda):
    """One key far above the rest, scores of +-10^4, tiny and huge values, zero queries."""
    B, H, Hkv, hd, n = 4, 8, 2, 128, 200
    rng = np.random.default_rng(4)
    cache = Cache(forge, cuda, B, Hkv, hd, 256, 0, seed=5)
    for b, (sk, sv) in enumerate([(1.0, 1e-30), (300.0, 1e30), (1e-20, 1.0), (30.0, 1.0)]):
        for kv, f in ((0, sk), (1, sv)):
            cache.scales[kv][b] = bf16(cache.scales[kv][b] * np.float32(f))
    cache.scales[1][3, :, ::3] = bf16(cache.scales[1][3, :, ::3] * np.float32(2.0 ** -40))  # values of mixed sizes
    for kv in range(2):
        import torch
        cache.d[2 + kv].copy_(torch.from_numpy(bits16(cache.scales[kv]).view(np.int16)))
    q = rng.standard_normal((B, H, hd)).astype(np.float32)
    q[0, 0] = 0
    q[0, 1] *= np.float32(1e-30)
    q[2] *= np.float32(1e20)
    check(decode(forge, cuda, cache, q, [n - 1] * B), reference(cache, q, [n - 1] * B))


def test_decode_masked_rows_may_hold_anything(forge, cuda):
    """Rows behind the last position, other pages and other sequences hold NaN scales: none of it is seen."""
    import torch
    for page in (0, 16):
        cache = Cache(forge, cuda, 3, 2, 128, 256, page, seed=6)
        pos = [0, 77, 130]
        keep = np.zeros(cache.scales[0].shape[:1] + cache.scales[0].shape[2:3], bool)
        for b, p in enumerate(pos):
            for j in range(p + 1):
                keep[cache.at(b, j)] = True
        q = np.random.default_rng(1).standard_normal((3, 8, 128)).astype(np.float32)
        want = reference(cache, q, pos)
        for kv in range(2):
            s = np.where(keep[:, None, :, None], cache.scales[kv], np.float32("nan"))
            cache.d[2 + kv].copy_(torch.from_numpy(bits16(s).view(np.int16)))
        check(decode(forge, cuda, cache, q, pos), want)
        # a NaN row that is seen makes its head's output NaN and no other
        i, j = cache.at(1, 40)
        cache.d[3].view(*cache.scales[1].shape)[i, 0, j, 1] = 0x7FC0
        got = decode(forge, cuda, cache, q, pos)
        assert np.isnan(got[1, :4, 64:]).all() and np.isfinite(got[1, :4, :64]).all()
        assert np.isfinite(got[[0, 2]]).all() and np.isfinite(got[1, 4:]).all()


@pytest.mark.parametrize("page", [0, 16])
def test_decode_out_of_range(forge, cuda, page):
    """A position, a sequence or a page outside sets the error word, makes that output NaN and spares the others;
    the next call with the same workspace is right."""
    import torch
    B, H, Hkv, hd = 4, 4, 2, 128
    cache = Cache(forge, cuda, B, Hkv, hd, 1024, page, seed=7)
    q = np.random.default_rng(2).standard_normal((B, H, hd)).astype(np.float32)
    good = [100, 1023, 5, 700]
    want = reference(cache, q, good)
    ws = torch.zeros(forge.lib().forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd), dtype=torch.uint8, device=cuda)
    cases = [([100, 1024, 5, 700], None, 1), ([2147483647, 1023, 5, 700], None, 0), (good, [0, 1, 4, 3], 2),
             (good, [0, 1, 2, -1], 3)]
    for pos, seq, bad in cases:
        got = decode(forge, cuda, cache, q, pos, seq, ws)
        with pytest.raises(forge.ForgeError, match="error word"):
            forge.check(forge.lib().forge_ops_check(), "error word")
        rest = [b for b in range(B) if b != bad]
        assert np.isnan(got[bad]).all()
        check(got[rest], (want[0][rest], want[1][rest]))
    if page:
        keep = int(cache.dt[1, 40])
        cache.dt[1, 40] = -1
        got = decode(forge, cuda, cache, q, good, None, ws)
        with pytest.raises(forge.ForgeError, match="error word"):
            forge.check(forge.lib().forge_ops_check(), "error word")
        assert np.isnan(got[1]).all()
        check(got[[0, 2, 3]], (want[0][[0, 2, 3]], want[1][[0, 2, 3]]))
        cache.dt[1, 40] = keep
    check(decode(forge, cuda, cache, q, good, None, ws), want)
    forge.check(forge.lib().forge_ops_check(), "error word")


def test_decode_is_deterministic_and_graph_safe(forge, cuda):
    """The same bits on every call, on another stream, and from a captured graph whose positions change between
    replays."""
    import torch
    B, H, Hkv, hd = 5, 16, 4, 128
    cache = Cache(forge, cuda, B, Hkv, hd, 3000, 0, seed=11)
    rng = np.random.default_rng(3)
    q = rng.standard_normal((B, H, hd)).astype(np.float32)
    L = forge.lib()
    first, later = [2999, 10, 1500, -1, 64], [3, 2500, -1, 999, 2999]
    dq = torch.from_numpy(q.reshape(B, -1)).to(cuda)
    dp = torch.tensor(first, dtype=torch.int32, device=cuda)
    out = torch.zeros(B, H * hd, device=cuda)
    ws = torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd), dtype=torch.uint8, device=cuda)
    call = lambda: forge.check(L.forge_flash_decode_kv4(dq.data_ptr(), cache.desc, None, dp.data_ptr(), B, H,  # noqa
                                                        out.data_ptr(), ws.data_ptr(), stream()), "decode")
    call()
    torch.cuda.synchronize()
    one = out.clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):
            call()
    side.synchronize()
    assert torch.equal(out, one)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for pos in (first, later, first):
        dp.copy_(torch.tensor(pos, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(out.cpu().numpy().reshape(B, H, hd), reference(cache, q, pos))
    assert torch.equal(out, one)


def test_paged_equals_contiguous(forge, cuda):
    """The same rows in pages give the same bits."""
    B, H, Hkv, hd, rows, page = 4, 8, 2, 128, 1024, 16
    a = Cache(forge, cuda, B, Hkv, hd, rows, page, seed=20)
    b = Cache(forge, cuda, B, Hkv, hd, rows, 0, seed=21)
    import torch
    for i in range(4):
        kv = a.d[i][a.dt.long()].transpose(1, 2).reshape(b.d[i].shape)
        b.d[i].copy_(kv)
    torch.cuda.synchronize()
    pos = [1023, 0, 512, 200]
    q = np.random.default_rng(5).standard_normal((B, H, hd)).astype(np.float32)
    assert np.array_equal(decode(forge, cuda, a, q, pos), decode(forge, cuda, b, q, pos))
