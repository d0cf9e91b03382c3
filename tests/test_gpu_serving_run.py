"""The packed prefill, the 4-bit cache and the token log probabilities as a
server uses them together: packed prompts through one attention layer, their
K and V quantised into pages handed out by the page allocator, then decode
steps that append one row a sequence and attend over the cache, and the
logits of each step scored. Float64 code follows along on the same values.

Tolerances: those of the single operators (tests/test_gpu_kv4.py,
test_gpu_prefill_varlen.py, test_gpu_logprobs.py)."""
import numpy as np
import pytest

from test_gpu_kv4 import U, bf16, bits16, quantise, values
from test_gpu_logprobs import check as check_logprobs
from test_gpu_prefill_varlen import check as check_prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,Hkv,hd,lens,page", [(8, 2, 128, [150, 1, 63, 300], 16), (4, 4, 64, [31, 257], 32)])
def test_prompt_cache_decode_score(forge, cuda, H, Hkv, hd, lens, page):
    import torch
    L, rng = forge.lib(), np.random.default_rng(hd)
    st = torch.cuda.current_stream().cuda_stream
    B, V, steps, top = len(lens), 5000, 5, 4
    cu = [0] + np.cumsum(lens).tolist()
    total, w = cu[-1], (H + 2 * Hkv) * hd
    qkv = torch.from_numpy(bits16(bf16(rng.standard_normal((total, w)).astype(np.float32))).view(np.int16)).to(cuda)
    qkv = qkv.view(torch.bfloat16)
    q, k, v = qkv[:, :H * hd], qkv[:, H * hd:(H + Hkv) * hd], qkv[:, (H + Hkv) * hd:]
    o = torch.zeros(total, H * hd, dtype=torch.bfloat16, device=cuda)
    lse = torch.zeros(H, total, device=cuda)
    dcu = torch.tensor(cu, dtype=torch.int32, device=cuda)
    forge.check(L.forge_flash_prefill_varlen(q.data_ptr(), w, k.data_ptr(), w, v.data_ptr(), w, dcu.data_ptr(), B, total,
                                             H, Hkv, hd, o.data_ptr(), H * hd, lse.data_ptr(), st), "prefill")

    # pages from the allocator, as the sequences grow
    most = -(-(max(lens) + steps) // page)
    alloc = forge.PagedKv(B * most + 2, page, hd)
    table = torch.zeros(B, most, dtype=torch.int32, device=cuda)

    def grow(b, n):
        while alloc.seq_pages(b) * page < n:
            i = alloc.seq_pages(b)
            table[b, i] = alloc.alloc_page(b)

    pool = B * most + 2
    d = [torch.full((pool, Hkv, page, hd // 2), 0x33, dtype=torch.uint8, device=cuda) for _ in range(2)] + \
        [torch.full((pool, Hkv, page, hd // 64), 0x7FC0, dtype=torch.int16, device=cuda) for _ in range(2)]
    cache = forge.ForgeKv4(k=d[0].data_ptr(), v=d[1].data_ptr(), ks=d[2].data_ptr(), vs=d[3].data_ptr(),
                           table=table.data_ptr(), n_seq=B, n_kv_head=Hkv, head_dim=hd, lmax=0, page_tokens=page,
                           max_pages=most, num_pages=pool)
    for b in rng.permutation(B):
        grow(int(b), lens[b])
    seq = torch.tensor(np.repeat(np.arange(B), lens), dtype=torch.int32, device=cuda)
    pos = torch.tensor(np.concatenate([np.arange(n) for n in lens]), dtype=torch.int32, device=cuda)
    forge.check(L.forge_kv4_append(cache, k.data_ptr(), v.data_ptr(), w, seq.data_ptr(), pos.data_ptr(), total, st),
                "append the prompts")
    check_prefill(torch, q, k, v, cu, H, Hkv, hd, o, lse)
    kv = [values(*quantise(x.float().cpu().numpy().reshape(total, Hkv, hd))) for x in (k, v)]
    held = [[x[cu[b]:cu[b + 1]] for b in range(B)] for x in kv]

    ws = torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd), dtype=torch.uint8, device=cuda)
    head = torch.randn(H * hd, V, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda) * 0.3
    for step in range(steps):
        now = [n + step for n in lens]
        for b in range(B):
            grow(b, now[b] + 1)
        dq = torch.from_numpy(rng.standard_normal((B, H * hd)).astype(np.float32)).to(cuda)
        row = torch.from_numpy(bits16(bf16(rng.standard_normal((B, 2 * Hkv * hd)).astype(np.float32))).view(np.int16)).to(cuda)
        at = torch.tensor(now, dtype=torch.int32, device=cuda)
        forge.check(L.forge_kv4_append(cache, row.data_ptr(), row.data_ptr() + 2 * Hkv * hd, 2 * Hkv * hd, None,
                                       at.data_ptr(), B, st), "append a step")
        ctx = torch.zeros(B, H * hd, device=cuda)
        forge.check(L.forge_flash_decode_kv4(dq.data_ptr(), cache, None, at.data_ptr(), B, H, ctx.data_ptr(),
                                             ws.data_ptr(), st), "decode")
        z = ctx @ head
        tok = z.argmax(1).to(torch.int32)
        f = [torch.zeros(B, device=cuda), torch.zeros(B, device=cuda), torch.zeros(B, dtype=torch.int32, device=cuda),
             torch.zeros(B, top, dtype=torch.int32, device=cuda), torch.zeros(B, top, device=cuda)]
        forge.check(L.forge_token_logprobs(z.data_ptr(), forge.FORGE_LOGITS_F32, V, B, V, tok.data_ptr(), top,
                                           *[x.data_ptr() for x in f], st), "score")
        torch.cuda.synchronize()
        forge.check(L.forge_ops_check(), "error word")
        new = row.view(torch.bfloat16).float().cpu().numpy().reshape(B, 2, Hkv, hd)
        for i in range(2):
            got = values(*quantise(new[:, i]))
            held[i] = [np.concatenate([x, got[b:b + 1]]) for b, x in enumerate(held[i])]
        qn, cn = (x.cpu().numpy().reshape(B, H, hd).astype(np.float64) for x in (dq, ctx))
        for b in range(B):
            n = now[b] + 1
            for h in range(H):
                kh, vh = held[0][b][:, h // (H // Hkv)], held[1][b][:, h // (H // Hkv)]
                s = kh @ qn[b, h] / np.sqrt(hd)
                p = np.exp(s - s.max())
                ds = (hd + 4) * U * (np.abs(kh) @ np.abs(qn[b, h])).max() / np.sqrt(hd)
                tol = np.abs(vh).max() * (4 * ds + (16 * np.abs(s).max() + 2 * (64 + n / 64) + 16) * U)
                assert np.abs(cn[b, h] - p @ vh / p.sum()).max() <= tol
        check_logprobs(z.cpu().double().numpy(), tok.tolist(), top,
                       dict(zip(("logprob", "entropy", "rank", "ids", "tops"), (x.cpu().numpy() for x in f))))
        assert (f[2] == 0).all() and torch.equal(f[3][:, 0], tok)
