"""Packed causal prefill with grouped heads (forge_flash_prefill_varlen)
against float64.

Tolerance: P is rounded to bf16 for P V and O to bf16 on output, each by at
most 2^-8 of its value, so |dO| <= 2^-8 (P |V| + |O|); the fp32 part (scores
of hd products, 2^-23 a sum, times 4 for their way through exp and both sums)
adds 4 hd 2^-23 max(|q| |k|) / sqrt(hd) + 2^-16 of P |V|. The row's LSE is
held to that fp32 part alone."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, lse, ldo=None, stream=None):
    import torch
    total = q.shape[0]
    dcu = torch.tensor(cu, dtype=torch.int32, device=cuda)
    torch.cuda.synchronize()
    forge.check(forge.lib().forge_flash_prefill_varlen(
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), dcu.data_ptr(), len(cu) - 1,
        total, H, Hkv, hd, o.data_ptr(), o.stride(0), lse.data_ptr() if lse is not None else None,
        stream or torch.cuda.current_stream().cuda_stream), "prefill")
    torch.cuda.synchronize()


def check(torch, q, k, v, cu, H, Hkv, hd, o, lse, seqs=None, rows=(0, 1 << 30)):
    """Every row of the sequences (within `rows`) against float64."""
    for s in range(len(cu) - 1) if seqs is None else seqs:
        a, b = cu[s], cu[s + 1]
        if a == b:
            continue
        qs, ks, vs, os_ = (x[a:b].double().unflatten(1, (-1, hd)).transpose(0, 1) for x in (q, k, v, o))
        ks, vs = (x.repeat_interleave(H // Hkv, 0) for x in (ks, vs))
        x = qs @ ks.transpose(1, 2) / hd ** 0.5
        hide = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device).triu(1)
        x = x.masked_fill(hide, float("-inf"))
        p = torch.softmax(x, -1)
        fine = 4 * hd * 2.0 ** -23 * (qs.abs() @ ks.abs().transpose(1, 2)).amax().item() / hd ** 0.5 + 2.0 ** -16
        pv = p @ vs.abs()
        want = p @ vs
        tol = 2.0 ** -8 * (pv + want.abs()) + fine * pv
        err = (os_ - want).abs()
        mine = slice(max(rows[0] - a, 0), max(min(rows[1], b) - a, 0))
        assert torch.isfinite(os_[:, mine]).all(), s
        assert (err <= tol)[:, mine].all(), (s, b - a, (err - tol).max().item())
        if lse is not None:
            e = (lse[:, a:b].double() - torch.logsumexp(x, -1)).abs()
            assert (e <= fine)[:, mine].all(), (s, e.max().item())


def make(torch, cuda, total, H, Hkv, hd, seed=0, pad=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    w = (H + 2 * Hkv) * hd + pad
    x = torch.randn(max(total, 1), w, generator=g, device=cuda).to(torch.bfloat16)[:total]
    return x[:, :H * hd], x[:, H * hd:(H + Hkv) * hd], x[:, (H + Hkv) * hd:(H + 2 * Hkv) * hd]


@pytest.mark.parametrize("H,Hkv,hd", [(2, 2, 128), (4, 1, 128), (6, 2, 64), (3, 3, 64), (10, 2, 128)])
@pytest.mark.parametrize("lens", [[1], [2], [127], [128], [129], [255, 1, 256, 0, 257], [0, 0, 3], [385, 64, 600],
                                  [5] * 40, [1300]], ids=str)
def test_varlen(forge, cuda, H, Hkv, hd, lens):
    import torch
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = make(torch, cuda, cu[-1], H, Hkv, hd, seed=len(lens) + H)
    o = torch.full((cu[-1], H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
    lse = torch.full((H, cu[-1]), float("nan"), device=cuda)
    run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, lse)
    forge.check(forge.lib().forge_ops_check(), "error word")
    check(torch, q, k, v, cu, H, Hkv, hd, o, lse)


def test_rows_outside_the_sequences_stay(forge, cuda):
    """Rows before the first and behind the last sequence, and the padding between rows of o, are not written; what
    they hold in q, k and v (NaN) is not seen."""
    import torch
    H, Hkv, hd, lens, lead, tail = 4, 2, 128, [70, 200, 1], 13, 300
    cu = [lead] + (lead + np.cumsum(lens)).tolist()
    total = cu[-1] + tail
    q, k, v = make(torch, cuda, total, H, Hkv, hd, seed=3, pad=40)
    for x in (q, k, v):
        x[:lead] = float("nan")
        x[cu[-1]:] = float("inf")
    o = torch.full((total, H * hd + 24), 9.0, dtype=torch.bfloat16, device=cuda)
    lse = torch.full((H, total), 9.0, device=cuda)
    run(forge, cuda, q, k, v, cu, H, Hkv, hd, o[:, :H * hd], lse)
    check(torch, q, k, v, cu, H, Hkv, hd, o[:, :H * hd], lse)
    assert (o[:, H * hd:] == 9).all() and (o[:lead] == 9).all() and (o[cu[-1]:] == 9).all()
    assert (lse[:, :lead] == 9).all() and (lse[:, cu[-1]:] == 9).all()


def test_sequences_are_isolated(forge, cuda):
    """A sequence of NaN and infinities between two others: only its own rows are NaN."""
    import torch
    H, Hkv, hd, lens = 4, 1, 64, [100, 130, 90, 300]
    cu = [0] + np.cumsum(lens).tolist()
    q, k, v = make(torch, cuda, cu[-1], H, Hkv, hd, seed=4)
    k[100:230] = float("nan")
    v[100:230] = float("inf")
    o = torch.zeros(cu[-1], H * hd, dtype=torch.bfloat16, device=cuda)
    lse = torch.zeros(H, cu[-1], device=cuda)
    run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, lse)
    check(torch, q, k, v, cu, H, Hkv, hd, o, lse, seqs=[0, 2, 3])
    assert torch.isnan(o[100:230]).all()


def test_no_lse_and_bad_bounds(forge, cuda):
    """lse may be NULL; a sequence with bad bounds sets the error word and is left out, the others are right."""
    import torch
    H, Hkv, hd = 2, 1, 128
    q, k, v = make(torch, cuda, 500, H, Hkv, hd, seed=5)
    good = [0, 100, 230, 500]
    o = torch.full((500, H * hd), 9.0, dtype=torch.bfloat16, device=cuda)
    run(forge, cuda, q, k, v, good, H, Hkv, hd, o, None)
    forge.check(forge.lib().forge_ops_check(), "error word")
    check(torch, q, k, v, good, H, Hkv, hd, o, None)
    # where bounds decrease, rows 200..299 belong to two sequences and hold either's
    for cu, fine in (([0, 100, 501], [(0, 0, 500)]), ([-5, 100, 300], [(1, 0, 500)]),
                     ([0, 300, 200, 400], [(0, 0, 200), (2, 300, 500)]), ([0, 200, 2147483647], [(0, 0, 500)])):
        o = torch.full((500, H * hd), 9.0, dtype=torch.bfloat16, device=cuda)
        run(forge, cuda, q, k, v, cu, H, Hkv, hd, o, None)
        with pytest.raises(forge.ForgeError, match="error word"):
            forge.check(forge.lib().forge_ops_check(), "error word")
        for s, lo, hi in fine:
            check(torch, q, k, v, cu, H, Hkv, hd, o, None, seqs=[s], rows=(lo, hi))


def test_scores_of_any_size(forge, cuda):
    """Rows whose maximum grows late, scores of +-1000, equal scores."""
    import torch
    H, Hkv, hd, n = 2, 2, 128, 700
    q, k, v = make(torch, cuda, n, H, Hkv, hd, seed=6)
    k[:, :hd] *= torch.linspace(0.01, 12, n, device=cuda)[:, None].to(torch.bfloat16)
    q[:, hd:] = 0
    o = torch.zeros(n, H * hd, dtype=torch.bfloat16, device=cuda)
    lse = torch.zeros(H, n, device=cuda)
    run(forge, cuda, q, k, v, [0, n], H, Hkv, hd, o, lse)
    check(torch, q, k, v, [0, n], H, Hkv, hd, o, lse)


def test_equals_the_padded_prefill(forge, cuda):
    """Against forge_flash_prefill on the same prompts (equal lengths, a multiple of 128, one KV head per query
    head): two roundings of P and O apart at most."""
    import torch
    B, H, S, hd = 2, 3, 256, 128
    q, k, v = make(torch, cuda, B * S, H, H, hd, seed=7)
    o = torch.zeros(B * S, H * hd, dtype=torch.bfloat16, device=cuda)
    run(forge, cuda, q, k, v, [0, S, 2 * S], H, H, hd, o, None)
    dense = [x.reshape(B, S, H, hd).transpose(1, 2).contiguous() for x in (q, k, v)]
    od = torch.zeros_like(dense[0])
    forge.check(forge.lib().forge_flash_prefill(*[x.data_ptr() for x in dense], od.data_ptr(), B, H, S, hd, 1,
                                                torch.cuda.current_stream().cuda_stream), "prefill")
    torch.cuda.synchronize()
    a, b = o.float().view(B, S, H, hd).transpose(1, 2), od.float()
    pv = 4.0  # P |V| of unit normals is below 4 in every column mean; rows of one key reach |v| itself
    assert ((a - b).abs() <= 2.0 ** -7 * (pv + b.abs())).all()


def test_graph_and_stream(forge, cuda):
    """A captured call whose bounds change between replays; the same bits on another stream."""
    import torch
    H, Hkv, hd, total = 4, 2, 64, 900
    q, k, v = make(torch, cuda, total, H, Hkv, hd, seed=8)
    o = torch.zeros(total, H * hd, dtype=torch.bfloat16, device=cuda)
    lse = torch.zeros(H, total, device=cuda)
    cu = torch.tensor([0, 300, 310, 900], dtype=torch.int32, device=cuda)
    call = lambda: forge.check(forge.lib().forge_flash_prefill_varlen(  # noqa: E731
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), cu.data_ptr(), 3, total, H, Hkv,
        hd, o.data_ptr(), o.stride(0), lse.data_ptr(), torch.cuda.current_stream().cuda_stream), "prefill")
    call()
    torch.cuda.synchronize()
    first = o.clone()
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        call()
    torch.cuda.synchronize()
    assert torch.equal(o, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for b in ([0, 300, 310, 900], [0, 1, 899, 900], [0, 900, 900, 900]):
        cu.copy_(torch.tensor(b, dtype=torch.int32))
        o.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(torch, q, k, v, b, H, Hkv, hd, o, lse)
