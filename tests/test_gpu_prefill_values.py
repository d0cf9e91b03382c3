"""The packed prefill's fp32 statistics and its edges, with inputs whose
scores are known exactly."""
import numpy as np
import pytest

import test_gpu_prefill_varlen as pv

pytestmark = pytest.mark.gpu
U = 2.0 ** -23


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(2, 1), (3, 3)])
def test_lse_to_fp32(forge, cuda, hd, H, Hkv):
    """Rows of up to 64 keys whose scores are products of one channel, exact in fp32: key 0 at 0, every eighth of the
    others at -d, the rest at -400 (no weight). With |x| = d log2 e below 3.7, the factor's and the exponent's roundings
    are 2.6 u of a probability and its exp2 is off by 2 u; a sum has 9 terms that are not 0, 4.5 u; the logarithm, its
    factor and their product 2 u |lse|."""
    import torch
    lens, w = 64, hd * (H + 2 * Hkv)
    d = torch.linspace(0, 2.5, 161).mul(hd ** 0.5).to(torch.bfloat16)  # a sequence each
    n = len(d)
    x = torch.zeros(n, lens, w, dtype=torch.bfloat16)
    x[:, :, 0:H * hd:hd] = 1
    keys = torch.full((8, n, lens), -400.0 * hd ** 0.5).to(torch.bfloat16)
    keys[:, :, 0] = 0
    for part in range(8):
        keys[part, :, part::8] = -d[:, None]
        keys[part, :, 0] = 0
    for part in range(8):
        x[:, :, H * hd:(H + Hkv) * hd:hd] = keys[part][:, :, None]
        rows = x.view(n * lens, w).to(cuda)
        q, k, v = rows[:, :H * hd], rows[:, H * hd:(H + Hkv) * hd], rows[:, (H + Hkv) * hd:]
        o = torch.full((n * lens, H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
        lse = torch.full((H, n * lens), float("nan"), device=cuda)
        pv.run(forge, cuda, q, k, v, [lens * i for i in range(n + 1)], H, Hkv, hd, o, lse)
        forge.check(forge.lib().forge_ops_check(), "error word")
        s = keys[part].double() / hd ** 0.5                      # [n][64]
        hide = torch.ones(lens, lens, dtype=torch.bool).triu(1)
        want = torch.logsumexp(s[:, None, :].masked_fill(hide, float("-inf")), -1).flatten()
        err = (lse.double().cpu() - want).abs()
        assert (err <= U * (9.1 + 2 * want.abs())).all(), (part, (err / U).max().item())


@pytest.mark.parametrize("H,Hkv", [(4, 1), (3, 3)])
def test_bounds_that_name_rows_many_times(forge, cuda, H, Hkv):
    """cu_seqlens that goes up and down again: the error word is set, and where the rows would be computed many times
    over nothing is; twice over is answered. Zero lengths and short prompts in number are no overlap."""
    import torch
    total, hd = 600, 64
    q, k, v = pv.make(torch, cuda, total, H, Hkv, hd, seed=1)
    for n, left_out in ((2, False), (40, True), (3000, True)):
        o = torch.full((total, H * hd), 9.0, dtype=torch.bfloat16, device=cuda)
        pv.run(forge, cuda, q, k, v, [0, total] * n, H, Hkv, hd, o, None)
        with pytest.raises(forge.ForgeError, match="error word"):
            forge.check(forge.lib().forge_ops_check(), "error word")
        if left_out:
            assert (o == 9).all()
        else:
            pv.check(torch, q, k, v, [0, total], H, Hkv, hd, o, None)
    for lens in ([1] * 600, [0, 1, 0] * 200 + [0] * 500 + [400], [600] + [0] * 3000):
        cu = [0] + np.cumsum(lens).tolist()
        o = torch.full((total, H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
        pv.run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, None)
        forge.check(forge.lib().forge_ops_check(), "error word")
        pv.check(torch, q, k, v, cu, H, Hkv, hd, o, None)


@pytest.mark.parametrize("hd,H,Hkv", [(64, 4, 2), (128, 2, 1), (128, 3, 3)])
@pytest.mark.parametrize("below", [False, True])
def test_far_scores(forge, cuda, hd, H, Hkv, below):
    """Scores from 1e8 to 1e30 of both signs, the largest so far replaced now and then: its key has all the weight (the
    others' are below 2^-1000), so the output is its row of V and the LSE its score to three roundings. The key's P is
    2^r, r the rounding of its score, not 1: as a bf16 off by 2^-8 of itself, while the sum has it in fp32; the output is
    rounded by 2^-8 as well. Both together 2.01 2^-8 |v|."""
    import torch
    n = 330
    rng = np.random.default_rng(5)
    val = rng.uniform(0.1, 0.4, n)
    for j, r in zip((0, 5, 63, 64, 127, 130, 200, 329), np.linspace(0.5, 0.95, 8)):
        val[j] = r
    best = np.maximum.accumulate(np.where(val >= 0.5, np.arange(n), 0))
    for size in (1e4, 1e5, 1e6, 1e8, 1e15):
        q, k, v = pv.make(torch, cuda, n, H, Hkv, hd, seed=2)
        q.zero_(), k.zero_()
        q[:, ::hd] = size
        k[:, ::hd] = torch.tensor((val - below) * size).to(torch.bfloat16).to(cuda)[:, None]
        o = torch.full((n, H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
        lse = torch.full((H, n), float("nan"), device=cuda)
        pv.run(forge, cuda, q, k, v, [0, n], H, Hkv, hd, o, lse)
        forge.check(forge.lib().forge_ops_check(), "error word")
        want = v.reshape(n, Hkv, hd).repeat_interleave(H // Hkv, 1)[best].flatten(1)
        assert ((o.double() - want.double()).abs() <= 2.01 * 2.0 ** -8 * want.double().abs()).all(), size
        s = k.reshape(n, Hkv, hd)[best, :, 0].double() * float(q[0, 0]) / hd ** 0.5
        s = s.repeat_interleave(H // Hkv, 1).t()
        assert ((lse.double() - s).abs() <= 2 * U * s.abs()).all(), size
