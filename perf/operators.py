"""Workloads of the serving operators on packed prompts and the 4-bit KV cache:

  prefill   forge_flash_prefill_varlen: causal attention of packed prompts of
            different lengths, grouped heads, bf16 in and out, fp32 row LSE
  append    forge_kv4_append + forge_kv4_read: K/V rows quantised into the
            4-bit cache and read back as the values they stand for
  decode    forge_flash_decode_kv4: one query per sequence over the 4-bit
            cache, contiguous or paged
  logprobs  forge_token_logprobs: log probability and rank of given tokens,
            entropy, top alternatives

`own` false computes them with elementary torch operations; true calls the
library. Head shapes: 32 / 8 heads of 64 (the 1B shape), 32 / 32 and 40 / 40
of 128 (7B, 13B), and 32 / 8 of 128.
"""
import math
import os
import sys

import torch

own = False

GROUP = 64  # dims that share one scale of the 4-bit cache
F32, BF16 = 0, 1


def _lib():
    path = os.path.join(os.getcwd(), "hexa-lang_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import forge_b200
    return forge_b200


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one short chat prompt on the 1B shape: launch latency
        dict(name="prefill_1b_one37", op="prefill", H=32, Hkv=8, hd=64, mix="one", n=1, longest=37),
        # a continuous-batching iteration that admits eight ragged prompts
        dict(name="prefill_1b_ragged8x1024", op="prefill", H=32, Hkv=8, hd=64, mix="ragged", n=8, longest=1024),
        # grouped heads of 128, many lengths from 1 to long in one batch
        dict(name="prefill_gqa_ragged16x4096", op="prefill", H=32, Hkv=8, hd=128, mix="ragged", n=16, longest=4096),
        # the repository's prefill workload (8 prompts of 4096, 7B heads), packed
        dict(name="prefill_7b_8x4096", op="prefill", H=32, Hkv=32, hd=128, mix="equal", n=8, longest=4096),
        # the rows of one decode step of 32 sequences
        dict(name="append_step32", op="append", Hkv=8, hd=128, rows=32, n_seq=32, lmax=4096, page=16),
        # a 4096-token prompt of the 7B shape into the cache
        dict(name="append_prompt4096", op="append", Hkv=32, hd=128, rows=4096, n_seq=1, lmax=8192, page=0),
        # 1B shape, eight sequences of about a thousand tokens in pages
        dict(name="decode_1b_bs8_1024", op="decode", H=32, Hkv=8, hd=64, B=8, ctx=1024, mix="ragged", page=16),
        # 7B shape, one sequence at 2048: the latency of interactive use
        dict(name="decode_7b_bs1_2048", op="decode", H=32, Hkv=32, hd=128, B=1, ctx=2048, mix="equal", page=0),
        # a served batch of very different lengths, grouped heads, pages
        dict(name="decode_gqa_bs32_16384", op="decode", H=32, Hkv=8, hd=128, B=32, ctx=16384, mix="ragged", page=32),
        # 13B shape, batch 64 at 4096: the throughput end
        dict(name="decode_13b_bs64_4096", op="decode", H=40, Hkv=40, hd=128, B=64, ctx=4096, mix="equal", page=0),
        # the token just sampled, with five alternatives, an API's answer
        dict(name="logprobs_1x32000", op="logprobs", rows=1, vocab=32000, dtype="f32", top=5),
        # a scored prompt batch: every position's token, bf16 logits of an odd vocabulary
        dict(name="logprobs_2048x50257", op="logprobs", rows=2048, vocab=50257, dtype="bf16", top=20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prefill", "append", "decode", "decode", "logprobs"])
    if op == "prefill":
        H, Hkv, hd = rng.choice([(32, 8, 64), (32, 8, 128), (32, 32, 128), (40, 40, 128), (12, 4, 64), (6, 1, 128)])
        return dict(op=op, H=H, Hkv=Hkv, hd=hd, mix=rng.choice(["ragged", "equal"]), n=_log(rng, 1, 16),
                    longest=_log(rng, 1, 2500))
    if op == "append":
        n_seq = _log(rng, 1, 64)
        page = rng.choice([0, 8, 16, 64])
        return dict(op=op, Hkv=rng.choice([1, 4, 8, 32, 40]), hd=rng.choice([64, 128]), rows=_log(rng, 1, 4096),
                    n_seq=n_seq, lmax=4096 if n_seq > 8 else 8192, page=page)
    if op == "decode":
        H, Hkv, hd = rng.choice([(32, 8, 64), (32, 8, 128), (32, 32, 128), (40, 40, 128), (12, 4, 64), (24, 1, 128)])
        B = _log(rng, 1, 64)
        return dict(op=op, H=H, Hkv=Hkv, hd=hd, B=B, ctx=_log(rng, 1, 131072 // B if Hkv <= 8 else 65536 // B),
                    mix=rng.choice(["ragged", "equal"]), page=rng.choice([0, 8, 16, 64]))
    vocab = _log(rng, 1000, 262144)
    return dict(op=op, rows=_log(rng, 1, min(2048, 100_000_000 // vocab)), vocab=vocab,
                dtype=rng.choice(["f32", "bf16"]), top=rng.choice([0, 1, 5, 20, 32]))


def _lengths(case, n, longest):
    """Lengths of a batch, the same for every seed: equal, or spread over the
    logarithm from 1 to the longest."""
    if case["mix"] == "equal" or n == 1:
        return [longest] * n
    if case["mix"] == "ragged":
        return [max(1, int(round(longest ** ((i * 7 % n + 1) / n)))) for i in range(n)]
    return [longest] * n


def _pages(case, g, n_seq, rows):
    """(page table [n_seq][max_pages] in a scattered order, pages) or None."""
    if not case["page"]:
        return None, 0
    per = -(-rows // case["page"])
    table = torch.randperm(n_seq * per, generator=g, device="cuda").to(torch.int32).view(n_seq, per)
    return table.contiguous(), n_seq * per


def _cache_shape(case, n_seq, rows, n_pages):
    return (n_pages, case["Hkv"], case["page"]) if case["page"] else (n_seq, case["Hkv"], rows)


# --------------------------------------------------------------- 4-bit rows
def _quantise(x):
    """bf16 values [..., hd] to (codes [..., hd / 2] uint8, scales [..., hd / 64] bf16), the rule of the int4 weights:
    per group of 64, scale = amax / 7 rounded to bf16 (1 where that is 0), code = x / scale to the nearest integer,
    halves away from zero, in -7..7, plus 7; low nibble first."""
    v = x.float().unflatten(-1, (-1, GROUP))
    scale = (v.abs().amax(-1) / 7.0).to(torch.bfloat16)
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    r = v / scale.float().unsqueeze(-1)
    c = torch.trunc(r + torch.where(r < 0, -0.5, 0.5)).clamp(-7, 7) + 7
    c = c.flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), scale


def _values(codes, scales, kind=torch.float32):
    """The values that codes and scales stand for."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).to(kind) - 7
    return (c.unflatten(-1, (-1, GROUP)) * scales.to(kind).unsqueeze(-1)).flatten(-2)


def _normal(shape, g, outliers=False):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    if outliers:  # keys have a few channels of larger size
        x = x * (1 + 3 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.05)).to(torch.bfloat16)
    return x


# ------------------------------------------------------------------ prepare
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"prefill": _prepare_prefill, "append": _prepare_append, "decode": _prepare_decode,
            "logprobs": _prepare_logprobs}[case["op"]](case, g)


def _prepare_prefill(case, g):
    H, Hkv, hd = case["H"], case["Hkv"], case["hd"]
    lens = _lengths(case, case["n"], case["longest"])
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    total = sum(lens)
    # one projection's output: Q, K and V side by side in a row
    qkv = _normal((total, (H + 2 * Hkv) * hd), g)
    q, k, v = qkv[:, :H * hd], qkv[:, H * hd:(H + Hkv) * hd], qkv[:, (H + Hkv) * hd:]
    o = torch.empty(total, H * hd, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(H, total, dtype=torch.float32, device="cuda")
    return dict(case, q=q, k=k, v=v, cu=cu, total=total, most=max(lens), o=o, lse=lse)


def _prepare_append(case, g):
    Hkv, hd, rows, n_seq = case["Hkv"], case["hd"], case["rows"], case["n_seq"]
    table, pages = _pages(case, g, n_seq, case["lmax"])
    shape = _cache_shape(case, n_seq, case["lmax"], pages)
    # row r is the next token of sequence r % n_seq, from a start of its own
    r = torch.arange(rows, device="cuda")
    seq = (r % n_seq).to(torch.int32)
    start = torch.randint(0, case["lmax"] - rows // n_seq, (n_seq,), generator=g, device="cuda")
    pos = (start[seq.long()] + r // n_seq).to(torch.int32)
    kv = _normal((rows, 2 * Hkv * hd), g, outliers=True)
    k, v = kv[:, :Hkv * hd], kv[:, Hkv * hd:]
    code = lambda: torch.full(shape + (hd // 2,), 0x77, dtype=torch.uint8, device="cuda")  # noqa: E731
    scale = lambda: torch.zeros(shape + (hd // GROUP,), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    out = [torch.empty(rows, Hkv * hd, dtype=torch.float32, device="cuda") for _ in range(2)]
    return dict(case, k=k, v=v, seq=seq, pos=pos, kc=code(), vc=code(), ks=scale(), vs=scale(), table=table,
                pages=pages, out=out)


def _prepare_decode(case, g):
    H, Hkv, hd, B = case["H"], case["Hkv"], case["hd"], case["B"]
    lens = _lengths(case, B, case["ctx"])
    page = case["page"]
    rows = -(-case["ctx"] // (page or 8)) * (page or 8)
    table, pages = _pages(case, g, B, rows)
    shape = _cache_shape(case, B, rows, pages)
    part = max(1, (64 << 20) // (shape[1] * shape[2] * hd))

    def cache(outliers):
        codes = torch.empty(shape + (hd // 2,), dtype=torch.uint8, device="cuda")
        scales = torch.empty(shape + (hd // GROUP,), dtype=torch.bfloat16, device="cuda")
        for i in range(0, shape[0], part):
            c, s = _quantise(_normal((min(part, shape[0] - i),) + shape[1:] + (hd,), g, outliers))
            codes[i:i + part], scales[i:i + part] = c, s
        return codes, scales

    kc, ks = cache(True)
    vc, vs = cache(False)
    q = torch.randn(B, H * hd, generator=g, device="cuda")
    pos = torch.tensor(lens, dtype=torch.int32, device="cuda") - 1
    out = torch.empty(B, H * hd, dtype=torch.float32, device="cuda")
    return dict(case, q=q, kc=kc, ks=ks, vc=vc, vs=vs, pos=pos, table=table, pages=pages, rows=rows, out=out)


def _prepare_logprobs(case, g):
    R, V, top = case["rows"], case["vocab"], case["top"]
    kind = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
    # confident and unsure rows: the spread of the logits differs by row
    z = torch.randn(R, V, generator=g, device="cuda") * (1 + 3 * torch.rand(R, 1, generator=g, device="cuda"))
    # a token that the model gives some weight: the largest of a few hundred
    pick = torch.randint(0, V, (R, 256), generator=g, device="cuda")
    tok = pick.gather(1, z.gather(1, pick).argmax(1, keepdim=True)).view(R).to(torch.int32)
    f = lambda *s: torch.empty(*s, dtype=torch.float32, device="cuda")  # noqa: E731
    i = lambda *s: torch.empty(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    return dict(case, z=z.to(kind), tok=tok, logprob=f(R), entropy=f(R), rank=i(R), ids=i(R, top), tops=f(R, top))


# ---------------------------------------------------------------------- run
def run(state):
    if own:
        return {"prefill": _own_prefill, "append": _own_append, "decode": _own_decode,
                "logprobs": _own_logprobs}[state["op"]](state)
    return {"prefill": _plain_prefill, "append": _plain_append, "decode": _plain_decode,
            "logprobs": _plain_logprobs}[state["op"]](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_prefill(s):
    fb = _lib()
    q, k, v, o = s["q"], s["k"], s["v"], s["o"]
    fb.check(fb.lib().forge_flash_prefill_varlen(
        q.data_ptr(), q.stride(0), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), s["cu"].data_ptr(), s["n"],
        s["total"], s["H"], s["Hkv"], s["hd"], o.data_ptr(), o.stride(0), s["lse"].data_ptr(), _stream()), "prefill")
    return {"o": o, "lse": s["lse"]}


def _own_cache(fb, s, n_seq, rows):
    if "cache" not in s:  # the descriptor that a program keeps beside its buffers
        page = s["page"]
        s["cache"] = fb.ForgeKv4(k=s["kc"].data_ptr(), v=s["vc"].data_ptr(), ks=s["ks"].data_ptr(),
                                 vs=s["vs"].data_ptr(), table=s["table"].data_ptr() if page else None, n_seq=n_seq,
                                 n_kv_head=s["Hkv"], head_dim=s["hd"], lmax=0 if page else rows, page_tokens=page,
                                 max_pages=s["table"].shape[1] if page else 0, num_pages=s["pages"])
    return s["cache"]


def _own_append(s):
    fb = _lib()
    c, k, v, out = _own_cache(fb, s, s["n_seq"], s["lmax"]), s["k"], s["v"], s["out"]
    fb.check(fb.lib().forge_kv4_append(c, k.data_ptr(), v.data_ptr(), k.stride(0), s["seq"].data_ptr(),
                                       s["pos"].data_ptr(), s["rows"], _stream()), "append")
    fb.check(fb.lib().forge_kv4_read(c, s["seq"].data_ptr(), s["pos"].data_ptr(), s["rows"], out[0].data_ptr(),
                                     out[1].data_ptr(), out[0].stride(0), _stream()), "read")
    return {"k": out[0], "v": out[1]}


def _own_decode(s):
    fb = _lib()
    c = _own_cache(fb, s, s["B"], s["rows"])
    if "ws" not in s:  # the workspace that a program keeps; zeroed once
        s["ws"] = torch.zeros(fb.lib().forge_flash_decode_kv4_workspace_bytes(s["B"], s["H"], s["Hkv"], s["hd"]),
                              dtype=torch.uint8, device="cuda")
    fb.check(fb.lib().forge_flash_decode_kv4(s["q"].data_ptr(), c, None, s["pos"].data_ptr(), s["B"], s["H"],
                                             s["out"].data_ptr(), s["ws"].data_ptr(), _stream()), "decode")
    return s["out"]


def _own_logprobs(s):
    fb = _lib()
    z, top = s["z"], s["top"]
    fb.check(fb.lib().forge_token_logprobs(
        z.data_ptr(), F32 if s["dtype"] == "f32" else BF16, z.stride(0), s["rows"], s["vocab"], s["tok"].data_ptr(), top,
        s["logprob"].data_ptr(), s["entropy"].data_ptr(), s["rank"].data_ptr(), s["ids"].data_ptr() if top else None,
        s["tops"].data_ptr() if top else None, _stream()), "logprobs")
    return _logprob_outputs(s["logprob"], s["entropy"], s["rank"], s["ids"], s["tops"], top)


def _logprob_outputs(logprob, entropy, rank, ids, tops, top):
    d = {"logprob": logprob, "entropy": entropy, "rank": rank}
    return dict(d, ids=ids, tops=tops) if top else d


# -------------------------------------------------------------- plain forms
def _plain_prefill(s):
    H, Hkv, hd, n, most, total, cu = s["H"], s["Hkv"], s["hd"], s["n"], s["most"], s["total"], s["cu"].long()
    at = torch.arange(most, device="cuda")
    inside = at < (cu[1:] - cu[:-1])[:, None]                       # [n][most]
    row = (cu[:-1, None] + at).clamp(max=total - 1)
    pad = lambda x, h: x[row].view(n, most, h, hd).transpose(1, 2).float()  # noqa: E731
    q = pad(s["q"], H).unflatten(1, (Hkv, H // Hkv)).flatten(2, 3)  # the group's queries over one KV head
    k, v = pad(s["k"], Hkv), pad(s["v"], Hkv)
    x = torch.matmul(q, k.transpose(2, 3)).unflatten(2, (H // Hkv, most))
    x = x.mul_(1.0 / math.sqrt(hd)).masked_fill_(at[None, :] > at[:, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = x.sub_(m).exp_()
    l = x.sum(-1, keepdim=True)
    o = torch.matmul(x.div_(l).flatten(2, 3), v).unflatten(2, (H // Hkv, most)).flatten(1, 2)  # [n][H][most][hd]
    lse = (m + l.log()).squeeze(-1).flatten(1, 2)                   # [n][H][most]
    o = o.transpose(1, 2)[inside].flatten(1).to(torch.bfloat16)
    return {"o": o, "lse": lse.transpose(1, 2)[inside].t().contiguous()}


def _rows_at(s, seq, pos):
    """Index of (sequence, position) into the cache's first and third axis."""
    if s["page"]:
        return s["table"][seq, pos // s["page"]].long(), pos % s["page"]
    return seq, pos


def _plain_append(s):
    Hkv, hd = s["Hkv"], s["hd"]
    i, j = _rows_at(s, s["seq"].long(), s["pos"].long())
    out = {}
    for name, codes, scales in (("k", "kc", "ks"), ("v", "vc", "vs")):
        c, sc = _quantise(s[name].unflatten(1, (Hkv, hd)))
        s[codes][i, :, j], s[scales][i, :, j] = c, sc
        out[name] = _values(s[codes][i, :, j], s[scales][i, :, j]).flatten(1)
    return out


def _plain_decode(s):
    H, Hkv, hd, B, rows = s["H"], s["Hkv"], s["hd"], s["B"], s["rows"]

    def whole(codes, scales):  # [B][Hkv][rows][hd]
        if s["page"]:
            t = s["table"].long()
            codes, scales = (x[t].transpose(1, 2).flatten(2, 3) for x in (codes, scales))
        return _values(codes, scales)

    q = s["q"].view(B, Hkv, H // Hkv, hd)
    x = torch.matmul(q, whole(s["kc"], s["ks"]).transpose(2, 3)) * (1.0 / math.sqrt(hd))
    hidden = torch.arange(rows, device="cuda") > s["pos"][:, None]
    x = x.masked_fill(hidden[:, None, None], -math.inf)
    p = (x - x.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    return torch.matmul(p, whole(s["vc"], s["vs"])).view(B, H * hd)


def _plain_logprobs(s):
    z, tok, V, top = s["z"].float(), s["tok"].long()[:, None], s["vocab"], s["top"]
    d = z - z.amax(1, keepdim=True)
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    entropy = (log_total - (e * d).sum(1, keepdim=True) / total).view(-1)
    at = torch.arange(V, device="cuda")
    mine = z.gather(1, tok)
    rank = ((z > mine) | ((z == mine) & (at < tok))).sum(1).to(torch.int32)
    logprob = (d.gather(1, tok) - log_total).view(-1)
    if not top:
        return _logprob_outputs(logprob, entropy, rank, None, None, 0)
    # order by value, ties to the lowest index: both in one whole number
    bits = s["z"].float().add(0.0).view(torch.int32).long()
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32) + (V - 1 - at)
    ids = V - 1 - (key.topk(top, dim=1).values & 0xFFFFFFFF)
    return _logprob_outputs(logprob, entropy, rank, ids.to(torch.int32), d.gather(1, ids) - log_total, top)


# ------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"prefill": _exact_prefill, "append": _exact_append, "decode": _exact_decode,
            "logprobs": _exact_logprobs}[case["op"]](s)


def _exact_prefill(s):
    """Sequence by sequence and head by head."""
    H, Hkv, hd, cu = s["H"], s["Hkv"], s["hd"], s["cu"].tolist()
    o = torch.empty(s["total"], H * hd, dtype=torch.float64, device="cuda")
    lse = torch.empty(H, s["total"], dtype=torch.float64, device="cuda")
    for a, b in zip(cu[:-1], cu[1:]):
        causal = torch.ones(b - a, b - a, dtype=torch.bool, device="cuda").tril()
        for h in range(H):
            g = h // (H // Hkv)
            q, k, v = s["q"][a:b, h * hd:(h + 1) * hd], s["k"][a:b, g * hd:(g + 1) * hd], s["v"][a:b, g * hd:(g + 1) * hd]
            x = (q.double() @ k.double().T) / hd ** 0.5
            x = torch.where(causal, x, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
            lse[h, a:b] = torch.logsumexp(x, 1)
            o[a:b, h * hd:(h + 1) * hd] = torch.softmax(x, 1) @ v.double()
    return {"o": o, "lse": lse}


def _exact_append(s):
    """The nearest of the 15 values of each group, by the definition."""
    out = {}
    for name in ("k", "v"):
        x = s[name].double().reshape(s["rows"], -1, GROUP)
        scale = (x.abs().max(2, keepdim=True).values / 7).to(torch.bfloat16).double()
        scale = torch.where(scale == 0, 1.0, scale)
        q = torch.sign(x) * torch.floor(x.abs() / scale + 0.5).clamp(max=7)
        out[name] = (q * scale).reshape(s["rows"], -1)
    return out


def _exact_decode(s):
    """Sequence by sequence, over its own rows alone."""
    H, Hkv, hd, page = s["H"], s["Hkv"], s["hd"], s["page"]
    out = torch.empty(s["B"], H, hd, dtype=torch.float64, device="cuda")
    weight = torch.tensor([1, 16], device="cuda")
    for b, last in enumerate(s["pos"].tolist()):
        L = last + 1
        kv = []
        for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
            if page:
                ids = s["table"][b, :-(-L // page)].long()
                c, f = codes[ids].permute(1, 0, 2, 3).reshape(Hkv, -1, hd // 2), scales[ids].permute(1, 0, 2, 3).reshape(Hkv, -1, hd // GROUP)
            else:
                c, f = codes[b], scales[b]
            c = (c[:, :L, :, None] // weight) % 16
            kv.append((c.reshape(Hkv, L, hd).double() - 7) * f[:, :L].double().repeat_interleave(GROUP, 2))
        q = s["q"][b].double().view(Hkv, H // Hkv, hd)
        p = torch.softmax(torch.einsum("hgd,htd->hgt", q, kv[0]) / hd ** 0.5, -1)
        out[b] = torch.einsum("hgt,htd->hgd", p, kv[1]).reshape(H, hd)
    return out.view(s["B"], H * hd)


def _exact_logprobs(s):
    """Row blocks of the log softmax; the alternatives' order is a whole number
    and has no value here."""
    R, V, top = s["rows"], s["vocab"], s["top"]
    logprob, entropy, tops = [], [], []
    for i in range(0, R, 128):
        lp = torch.log_softmax(s["z"][i:i + 128].double(), 1)
        logprob.append(lp[torch.arange(lp.shape[0], device="cuda"), s["tok"][i:i + 128].long()])
        entropy.append(-(lp.exp() * lp).sum(1))
        tops.append(lp.sort(1, descending=True).values[:, :top])
    return _logprob_outputs(torch.cat(logprob), torch.cat(entropy), None, None, torch.cat(tops), top)


# --------------------------------------------------------------------- work
def work(case):
    if case["op"] == "prefill":
        H, Hkv, hd = case["H"], case["Hkv"], case["hd"]
        lens = _lengths(case, case["n"], case["longest"])
        return {"bytes": sum(lens) * ((2 * H + 2 * Hkv) * hd * 2 + 4 * H),
                "flops": 4 * hd * H * sum(n * (n + 1) // 2 for n in lens)}
    if case["op"] == "append":
        n = 2 * case["rows"] * case["Hkv"] * case["hd"]
        held = n // 2 + n // GROUP * 2
        return {"bytes": 2 * n + 2 * held + 4 * n, "flops": 4 * n}  # rows in; cache out and in; values out
    if case["op"] == "decode":
        H, Hkv, hd = case["H"], case["Hkv"], case["hd"]
        keys = sum(_lengths(case, case["B"], case["ctx"]))
        return {"bytes": keys * Hkv * 2 * (hd // 2 + hd // GROUP * 2) + 8 * case["B"] * H * hd,
                "flops": 4 * keys * H * hd}
    R, V = case["rows"], case["vocab"]
    return {"bytes": R * V * (4 if case["dtype"] == "f32" else 2) + R * (16 + 8 * case["top"]), "flops": 5 * R * V}
