"""Decode over the 4-bit KV cache where the rows of V differ in size: attention
sinks, rows of zeros, large rows without weight.

The error is held relative to what the output is made of, not to the largest
row. With u = 2^-23 and, per group g of 64 dims,
A_g = sum_j p_j max_{d in g} |v_jd| / sum p:

- a score (integer sums, exact; 8 fp32 roundings; q rounded to 2^-24 of its
  largest channel) is off by at most
  ds = (8 u sum|q k| + u max|q| sum|k|) / sqrt(hd), a probability relative to
  the largest by 2 ds + 8 u max|s|, so the output by A_g (4 ds + 16 u max|s|);
- the weights p_j s_jg of a tile of 64 keys are rounded to 1.004 2^-24 of the
  largest, times a code of at most 7: 64 1.004 2^-24 (7 max p s) below 33 u of
  the tile's part of A_g, since the largest code of a group that is not zero is
  +-7;
- the joins of tiles, warps and CTAs: (2 (64 + n / 64) + 16) u A_g."""
import numpy as np
import pytest

import test_gpu_kv4 as kv4

pytestmark = pytest.mark.gpu
U = kv4.U


def reference(cache, q, pos):
    """(output, tolerance) [B][H][hd] in float64."""
    B, H, hd = q.shape
    G = H // cache.Hkv
    out, tol = np.zeros((B, H, hd)), np.zeros((B, H, hd))
    for b in range(B):
        n = pos[b] + 1
        k, v = (cache.row(kv, b, n) for kv in range(2))
        for h in range(H):
            qh, kh, vh = q[b, h].astype(np.float64), k[:, h // G], v[:, h // G]
            s = kh @ qh / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h] = p @ vh
            a = p @ np.abs(vh).reshape(n, -1, 64).max(-1)
            ds = U * (8 * (np.abs(kh) @ np.abs(qh)).max() + np.abs(qh).max() * np.abs(kh).sum(1).max()) / np.sqrt(hd)
            rel = 4 * ds + (16 * np.abs(s).max() + 33 + 2 * (64 + n / 64) + 16) * U
            tol[b, h] = np.repeat(a, 64) * rel
    return out, tol


def fill(cache, b, kv, x):
    """Rows x [n][Hkv][hd] as the first of sequence b, on the host."""
    c, s = kv4.quantise(kv4.bf16(x.astype(np.float32)))
    for r in range(x.shape[0]):
        i, j = cache.at(b, r)
        cache.codes[kv][i, :, j], cache.scales[kv][i, :, j] = c[r], s[r]


def upload(cache):
    import torch
    for kv in range(2):
        cache.d[kv].copy_(torch.from_numpy(cache.codes[kv]))
        cache.d[2 + kv].copy_(torch.from_numpy(kv4.bits16(cache.scales[kv]).view(np.int16)))


# (score of key `at`, size of its V, size of the other V, rows of zeros)
CASES = [(14, 1e-3, 1.0, []), (12, 1e-2, 1.0, []), (0, 1.0, 1e-2, [3]), (0, 1e-3, 1e-3, [3, 70, 130]),
         (2, 1e-6, 1e-6, [0, 64, 65, 199]), (-14, 1e2, 1.0, []), (-28, 1e4, 1.0, []), (-28, 1e8, 1.0, []),
         (-200, 1e4, 1.0, []), (-200, 1e8, 1e-3, [5]), (0, 1e-4, 1e-4, list(range(64, 128))),
         (20, 1e-4, 1.0, list(range(1, 64)))]


@pytest.mark.parametrize("hd,H,Hkv", [(128, 2, 2), (128, 4, 2), (64, 2, 2), (64, 4, 2), (128, 8, 2), (64, 4, 1),
                                      (128, 3, 1)])
@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("at", [0, 40])
def test_decode_of_unequal_rows(forge, cuda, hd, H, Hkv, page, at):
    n = 200
    rng = np.random.default_rng(hd + H + at)
    cache = kv4.Cache(forge, cuda, len(CASES), Hkv, hd, 208, page, seed=1, fill=False)
    sign = np.where(rng.random((Hkv, hd)) < 0.5, -0.5, 0.5)
    q = (np.repeat(sign, H // Hkv, 0) + 0.02 * rng.standard_normal((len(CASES), H, hd))).astype(np.float32)
    for b, (score, size, others, zeros) in enumerate(CASES):
        k, v = 0.3 * rng.standard_normal((n, Hkv, hd)), others * rng.standard_normal((n, Hkv, hd))
        k[at] = sign * (score / (0.25 * hd ** 0.5))
        v[at] *= size / others
        v[zeros] = 0
        fill(cache, b, 0, k)
        fill(cache, b, 1, v)
    upload(cache)
    pos = [n - 1] * len(CASES)
    kv4.check(kv4.decode(forge, cuda, cache, q, pos), reference(cache, q, pos))
    forge.check(forge.lib().forge_ops_check(), "error word")


@pytest.mark.parametrize("hd,H,Hkv", [(128, 2, 2), (64, 2, 1), (128, 8, 2), (64, 4, 1)])
def test_decode_of_scales_of_one(forge, cuda, hd, H, Hkv):
    """Rows whose scale is 1 because their largest value is 7 count, beside rows of zeros; V of zeros alone gives zeros;
    a row of zeros in one group of its dims only."""
    n, B = 150, 4
    rng = np.random.default_rng(3)
    cache = kv4.Cache(forge, cuda, B, Hkv, hd, 160, 0, seed=2, fill=False)
    q = rng.standard_normal((B, H, hd)).astype(np.float32)
    for b in range(B):
        v = rng.integers(-7, 8, (n, Hkv, hd)).astype(np.float64)
        v[..., 5], v[..., hd - 1] = 7, -7
        if b == 1:
            v[::3] = 0
        elif b == 2:
            v[:] = 0
        elif b == 3:
            v *= 1e-4
            v[::2, :, :64] = 0
        fill(cache, b, 0, rng.standard_normal((n, Hkv, hd)))
        fill(cache, b, 1, v)
    upload(cache)
    pos = [n - 1, 70, n - 1, 99]
    got = kv4.decode(forge, cuda, cache, q, pos)
    kv4.check(got, reference(cache, q, pos))
    assert (got[2] == 0).all()


def test_decode_of_a_long_sink(forge, cuda):
    """A sink at the start of a long context, which many CTAs share."""
    n, H, Hkv, hd = 9000, 4, 2, 128
    rng = np.random.default_rng(9)
    cache = kv4.Cache(forge, cuda, 1, Hkv, hd, 9024, 0, seed=4)
    sign = np.where(rng.random((Hkv, hd)) < 0.5, -0.5, 0.5)
    q = np.repeat(sign, H // Hkv, 0)[None].astype(np.float32)
    fill(cache, 0, 0, (sign * (13 / (0.25 * hd ** 0.5)))[None])
    fill(cache, 0, 1, 1e-3 * rng.standard_normal((1, Hkv, hd)))
    cache.scales[0][0, :, 1:] *= np.float32(0.25)
    upload(cache)
    kv4.check(kv4.decode(forge, cuda, cache, q, [n - 1]), reference(cache, q, [n - 1]))


def test_decode_of_a_negative_scale(forge, cuda):
    """A scale below zero is not of the format: its group's output is NaN, no other's."""
    for H in (2, 8):
        cache = kv4.Cache(forge, cuda, 2, 2, 128, 128, 0, seed=6)
        q = np.random.default_rng(1).standard_normal((2, H, 128)).astype(np.float32)
        want = kv4.reference(cache, q, [100, 100])
        cache.scales[1][0, 1, 30, 1] *= -1
        upload(cache)
        got = kv4.decode(forge, cuda, cache, q, [100, 100])
        nan = np.zeros_like(got, bool)
        nan[0, H // 2:, 64:] = True
        assert np.array_equal(np.isnan(got), nan)
        assert (np.abs(got - want[0]) <= np.broadcast_to(want[1], got.shape))[~nan].all()


@pytest.mark.parametrize("hd,H,Hkv", [(128, 4, 4), (64, 4, 2), (128, 8, 2), (64, 6, 2), (64, 8, 1), (128, 11, 1)])
@pytest.mark.parametrize("page", [0, 24])
def test_decode_at_every_boundary(forge, cuda, hd, H, Hkv, page):
    """Rows whose sizes are spread over six orders of magnitude, contexts around every boundary and one that CTAs
    share."""
    pos = [0, 1, 14, 15, 16, 31, 32, 62, 63, 64, 65, 127, 128, 255, 256, 300, 383, 2390]
    rng = np.random.default_rng(hd + H)
    cache = kv4.Cache(forge, cuda, len(pos), Hkv, hd, 2400, page, seed=H)
    size = np.exp(rng.uniform(np.log(1e-6), 0, cache.scales[1].shape)).astype(np.float32)
    cache.scales[1] = kv4.bf16(cache.scales[1] * size)
    upload(cache)
    q = rng.standard_normal((len(pos), H, hd)).astype(np.float32) * 2
    got = kv4.decode(forge, cuda, cache, q, pos)
    forge.check(forge.lib().forge_ops_check(), "error word")
    kv4.check(got, reference(cache, q, pos))


@pytest.mark.parametrize("hd,H,Hkv", [(128, 2, 2), (64, 2, 1), (128, 8, 2), (64, 4, 1)])
def test_decode_of_extreme_sizes(forge, cuda, hd, H, Hkv):
    """Scores of ordinary size from tiny queries and huge keys and the other way round, up to the ends of fp32 and bf16;
    V at the ends as well."""
    sizes = [(1e-30, 1e30, 1.0), (1e-37, 1e37, 1.0), (1e37, 1e-37, 1.0), (1e20, 1e-20, 1e37), (1e18, 1e-18, 1e-25),
             (1e-18, 1e20, 1.0), (1e36, 1e-30, 1.0), (1.0, 1.0, 1e37)]
    n = 150
    rng = np.random.default_rng(hd + H)
    cache = kv4.Cache(forge, cuda, len(sizes), Hkv, hd, 152, 0, seed=7)
    q = rng.standard_normal((len(sizes), H, hd)).astype(np.float32)
    for b, (sq, sk, sv) in enumerate(sizes):
        q[b] *= np.float32(sq)
        for kv, f in ((0, sk), (1, sv)):
            cache.scales[kv][b] = kv4.bf16((cache.scales[kv][b].astype(np.float64) * f).astype(np.float32))
    upload(cache)
    pos = [n - 1] * len(sizes)
    kv4.check(kv4.decode(forge, cuda, cache, q, pos), reference(cache, q, pos))


@pytest.mark.parametrize("hd,H,Hkv", [(128, 2, 2), (64, 2, 1), (128, 8, 2), (64, 4, 1)])
def test_decode_of_far_scores(forge, cuda, hd, H, Hkv):
    """Scores from 1e8 to 1e30 of both signs: the key with the largest has all the weight, wherever it lies. (The gap to
    the next is above a score's error, so the others' weights are below 2^-100; what is left is the rounding of one
    weight, one sum and one quotient: 8 u.)"""
    n, sizes = 200, [1e4, 3e4, 1e5, 1e7, 1e15]
    rng = np.random.default_rng(hd + H)
    cache = kv4.Cache(forge, cuda, 2 * len(sizes), Hkv, hd, 200, 0, seed=8)
    sign = np.where(rng.random((Hkv, hd)) < 0.5, -0.5, 0.5)
    q = np.repeat(sign, H // Hkv, 0)[None].repeat(2 * len(sizes), 0)
    top = rng.integers(0, n, 2 * len(sizes))
    for b in range(2 * len(sizes)):
        size, below = sizes[b // 2], b % 2
        k = size * sign * rng.uniform(0.1, 0.8, (n, Hkv, 1))
        k[top[b]] = size * sign * 0.9
        if below:  # all of them negative, the smallest in size on top
            k = size * sign - k
        fill(cache, b, 0, k * (-1 if below else 1))
        q[b] *= size
    upload(cache)
    q = q.astype(np.float32)
    pos = [n - 1] * len(q)
    got = kv4.decode(forge, cuda, cache, q, pos)
    for b in range(len(q)):
        k, v = (cache.row(kv, b, n) for kv in range(2))
        for h in range(H):
            g = h // (H // Hkv)
            s = k[:, g] @ q[b, h].astype(np.float64) / np.sqrt(hd)
            ds = 10 * U * (np.abs(k[:, g]) @ np.abs(q[b, h].astype(np.float64))).max() / np.sqrt(hd)
            assert s[top[b]] - np.delete(s, top[b]).max() > 100 + 2 * ds and (s.max() < 0) == bool(b % 2)
            vmax = np.repeat(np.abs(v[top[b], g]).reshape(-1, 64).max(-1), 64)
            assert (np.abs(got[b, h] - v[top[b], g]) <= 8 * U * vmax).all(), (b, h)
