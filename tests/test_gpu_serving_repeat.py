"""The serving operators called again: on another stream, from captured graphs,
on two streams at once. Every call writes outputs of its own that hold NaN or
-7 before it, so that a call that wrote nothing, or part, would show."""
import numpy as np
import pytest

import test_gpu_kv4 as kv4
import test_gpu_prefill_varlen as pv

pytestmark = pytest.mark.gpu


def clear(outs):
    for o in outs:
        o.fill_(float("nan") if o.is_floating_point() else -7)


def same(torch, a, b):
    kind = {1: torch.int8, 2: torch.int16, 4: torch.int32}
    return all(torch.equal(x.view(kind[x.element_size()]), y.view(kind[y.element_size()])) for x, y in zip(a, b))


def repeat(torch, cuda, call, make, written):
    """call(outs, stream, lane) writes every element of make()'s tensors (lane: which workspace); written checks the
    first's."""
    first = make()
    clear(first)
    torch.cuda.synchronize()
    call(first, torch.cuda.current_stream(), 0)
    torch.cuda.synchronize()
    written(first)
    side = [torch.cuda.Stream() for _ in range(2)]
    outs = [make() for _ in range(12)]
    for o in outs:
        clear(o)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):  # two streams at once
        with torch.cuda.stream(side[i % 2]):
            call(o, side[i % 2], i % 2)
    torch.cuda.synchronize()
    assert all(same(torch, o, first) for o in outs)
    graphs, held = [], []
    for lane in range(2):
        held.append(make())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(held[-1], torch.cuda.current_stream(), lane)
    for _ in range(3):
        for o in held:
            clear(o)
        torch.cuda.synchronize()
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(same(torch, o, first) for o in held)


@pytest.mark.parametrize("H,Hkv,hd", [(4, 2, 64), (8, 2, 128), (3, 3, 128)])
def test_prefill(forge, cuda, H, Hkv, hd):
    import torch
    cu = [0, 300, 310, 310, 900]
    q, k, v = pv.make(torch, cuda, cu[-1], H, Hkv, hd, seed=8)
    dcu = torch.tensor(cu, dtype=torch.int32, device=cuda)

    def call(outs, stream, lane):
        forge.check(forge.lib().forge_flash_prefill_varlen(
            q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), dcu.data_ptr(), len(cu) - 1,
            cu[-1], H, Hkv, hd, outs[0].data_ptr(), H * hd, outs[1].data_ptr(), stream.cuda_stream), "prefill")

    repeat(torch, cuda, call, lambda: [torch.empty(cu[-1], H * hd, dtype=torch.bfloat16, device=cuda),
                                       torch.empty(H, cu[-1], device=cuda)],
           lambda o: pv.check(torch, q, k, v, cu, H, Hkv, hd, *o))


@pytest.mark.parametrize("H,Hkv,hd,page", [(16, 4, 128, 0), (4, 4, 128, 16), (8, 4, 64, 0), (8, 1, 64, 8)])
def test_decode(forge, cuda, H, Hkv, hd, page):
    import torch
    pos = [2999, 10, 1500, -1, 64]
    B = len(pos)
    cache = kv4.Cache(forge, cuda, B, Hkv, hd, 3000, page, seed=11)
    q = np.random.default_rng(3).standard_normal((B, H, hd)).astype(np.float32)
    L = forge.lib()
    dq = torch.from_numpy(q.reshape(B, -1)).to(cuda)
    dp = torch.tensor(pos, dtype=torch.int32, device=cuda)
    ws = [torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd), dtype=torch.uint8, device=cuda)
          for _ in range(2)]

    def call(outs, stream, lane):
        forge.check(L.forge_flash_decode_kv4(dq.data_ptr(), cache.desc, None, dp.data_ptr(), B, H, outs[0].data_ptr(),
                                             ws[lane].data_ptr(), stream.cuda_stream), "decode")

    want = kv4.reference(cache, q, pos)
    repeat(torch, cuda, call, lambda: [torch.empty(B, H * hd, device=cuda)],
           lambda o: kv4.check(o[0].cpu().numpy().reshape(B, H, hd), want))


@pytest.mark.parametrize("R,V,dtype", [(1, 32000, "f32"), (3, 5001, "bf16"), (700, 1003, "bf16"), (5, 7, "f32")])
def test_logprobs(forge, cuda, R, V, dtype):
    import torch
    top = 5
    g = torch.Generator(device=cuda).manual_seed(R)
    z = (torch.randn(R, V, generator=g, device=cuda) * 2).to(torch.float32 if dtype == "f32" else torch.bfloat16)
    tok = torch.randint(0, V, (R,), generator=g, device=cuda).to(torch.int32)
    kind = forge.FORGE_LOGITS_F32 if dtype == "f32" else forge.FORGE_LOGITS_BF16

    def call(outs, stream, lane):
        forge.check(forge.lib().forge_token_logprobs(z.data_ptr(), kind, V, R, V, tok.data_ptr(), top,
                                                     *[o.data_ptr() for o in outs], stream.cuda_stream), "logprobs")

    def make():
        f, i = dict(dtype=torch.float32, device=cuda), dict(dtype=torch.int32, device=cuda)
        return [torch.empty(R, **f), torch.empty(R, **f), torch.empty(R, **i), torch.empty(R, top, **i),
                torch.empty(R, top, **f)]

    def written(o):
        p = torch.log_softmax(z.double(), 1)
        assert ((o[0].double() - p[torch.arange(R, device=cuda), tok.long()]).abs() < 1e-4).all()
        assert ((o[1].double() + (p.exp() * p).sum(1)).abs() < 1e-4).all()
        assert ((o[4].double() - p.sort(1, descending=True).values[:, :top]).abs() < 1e-4).all()
        assert (o[3] >= 0).all() and (o[2] >= 0).all()

    repeat(torch, cuda, call, make, written)


def test_append_and_read(forge, cuda):
    """Into caches of NaN scales, each call's own."""
    import torch
    n, Hkv, hd = 40, 3, 128
    w = Hkv * hd
    x = torch.randn(n, 2 * w, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int32, device=cuda)
    seq = torch.zeros(n, dtype=torch.int32, device=cuda)
    L = forge.lib()

    def make():
        return [torch.empty(1, Hkv, n, hd // 2, dtype=torch.int8, device=cuda) for _ in range(2)] + \
               [torch.empty(1, Hkv, n, hd // 64, dtype=torch.bfloat16, device=cuda) for _ in range(2)] + \
               [torch.empty(n, w, device=cuda) for _ in range(2)]

    def call(o, stream, lane):
        c = forge.ForgeKv4(k=o[0].data_ptr(), v=o[1].data_ptr(), ks=o[2].data_ptr(), vs=o[3].data_ptr(), table=None,
                           n_seq=1, n_kv_head=Hkv, head_dim=hd, lmax=n, page_tokens=0, max_pages=0, num_pages=0)
        forge.check(L.forge_kv4_append(c, x.data_ptr(), x[:, w:].data_ptr(), 2 * w, seq.data_ptr(), pos.data_ptr(), n,
                                       stream.cuda_stream), "append")
        forge.check(L.forge_kv4_read(c, seq.data_ptr(), pos.data_ptr(), n, o[4].data_ptr(), o[5].data_ptr(), w,
                                     stream.cuda_stream), "read")

    def written(o):
        for kv in range(2):
            rows = x[:, kv * w:(kv + 1) * w].float().cpu().numpy().reshape(n, Hkv, hd)
            want = kv4.values(*kv4.quantise(rows)).astype(np.float32)
            assert np.array_equal(o[4 + kv].cpu().numpy().reshape(n, Hkv, hd), want)

    repeat(torch, cuda, call, make, written)


@pytest.mark.parametrize("hd", [64, 128])
def test_prefill_equals_the_padded_one(forge, cuda, hd):
    """forge_flash_prefill on the same prompts: P and O rounded to bf16 on both sides, 2^-8 of P |V| and of |O| each, and
    a score's hd sums (2^-23 of |q| |k| each, on both sides, times 4 for their way through exp and both sums)."""
    import torch
    B, H, S = 2, 3, 384
    q, k, v = pv.make(torch, cuda, B * S, H, H, hd, seed=7)
    o = torch.full((B * S, H * hd), float("nan"), dtype=torch.bfloat16, device=cuda)
    pv.run(forge, cuda, q, k, v, [0, S, 2 * S], H, H, hd, o, None)
    dense = [x.reshape(B, S, H, hd).transpose(1, 2).contiguous() for x in (q, k, v)]
    od = torch.full_like(dense[0], float("nan"))
    forge.check(forge.lib().forge_flash_prefill(*[x.data_ptr() for x in dense], od.data_ptr(), B, H, S, hd, 1,
                                                torch.cuda.current_stream().cuda_stream), "prefill")
    torch.cuda.synchronize()
    a, b = o.double().view(B, S, H, hd).transpose(1, 2), od.double()
    qd, kd, vd = (x.double() for x in dense)
    s = (qd @ kd.transpose(2, 3)) / hd ** 0.5
    p = torch.softmax(s.masked_fill(torch.ones(S, S, dtype=torch.bool, device=cuda).triu(1), float("-inf")), -1)
    fine = 8 * hd * 2.0 ** -23 * (qd.abs() @ kd.abs().transpose(2, 3)).amax().item() / hd ** 0.5 + 2.0 ** -15
    part = p @ vd.abs()
    assert ((a - b).abs() <= 2.0 ** -7 * (part + b.abs()) * (1 + 2.0 ** -7) + fine * part).all()
