"""Refusals of the packed prefill, the 4-bit cache and the token log
probabilities, checked before anything touches a GPU; every call here names
addresses that are never read."""
import ctypes as C

import pytest

A = 1 << 20  # an aligned address


def cache(forge, **kw):
    d = dict(k=A, v=A, ks=A, vs=A, table=None, n_seq=4, n_kv_head=2, head_dim=128, lmax=64, page_tokens=0, max_pages=0,
             num_pages=0)
    d.update(kw)
    return forge.ForgeKv4(**d)


def paged(**kw):
    return dict(dict(table=A, lmax=0, page_tokens=16, max_pages=4, num_pages=16), **kw)


BAD_CACHE = [dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(k=A + 8), dict(vs=A + 2), dict(n_seq=0),
             dict(n_kv_head=0), dict(n_kv_head=-1), dict(head_dim=96), dict(head_dim=256), dict(lmax=0), dict(lmax=-8),
             dict(lmax=60), dict(lmax=(1 << 30) + 8), paged(page_tokens=0), paged(page_tokens=12), paged(max_pages=0),
             paged(num_pages=0), paged(page_tokens=1 << 16, max_pages=1 << 16)]


def refused(forge, rc, code=None):
    assert rc == (forge.FORGE_INVALID_ARGS if code is None else code)
    assert forge.lib().forge_b200_last_error()


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_cache(forge, bad):
    L, c = forge.lib(), cache(forge, **bad)
    refused(forge, L.forge_kv4_append(c, A, A, 256, A, A, 3, None))
    refused(forge, L.forge_kv4_read(c, A, A, 3, A, A, 256, None))
    refused(forge, L.forge_flash_decode_kv4(A, c, A, A, 3, 4, A, A, None))


def test_null_cache(forge):
    L = forge.lib()
    refused(forge, L.forge_kv4_append(None, A, A, 256, A, A, 3, None))
    refused(forge, L.forge_kv4_read(None, A, A, 3, A, A, 256, None))
    refused(forge, L.forge_flash_decode_kv4(A, None, A, A, 3, 4, A, A, None))


def test_append_and_read_args(forge):
    L, c = forge.lib(), cache(forge)
    for k, v, ld, seq, pos, n in [(None, A, 256, A, A, 3), (A, None, 256, A, A, 3), (A, A, 256, A, None, 3),
                                  (A, A, 256, A, A, -1), (A, A, 248, A, A, 3), (A, A, 260, A, A, 3),
                                  (A + 2, A, 256, A, A, 3), (A, A + 8, 256, A, A, 3), (A, A, 256, None, A, 5)]:
        refused(forge, L.forge_kv4_append(c, k, v, ld, seq, pos, n, None))
    for seq, pos, n, k, v, ld in [(A, None, 3, A, A, 256), (A, A, -1, A, A, 256), (A, A, 3, None, A, 256),
                                  (A, A, 3, A, None, 256), (A, A, 3, A, A, 252), (A, A, 3, A, A, 258),
                                  (A, A, 3, A + 4, A, 256), (None, A, 5, A, A, 256)]:
        refused(forge, L.forge_kv4_read(c, seq, pos, n, k, v, ld, None))


def test_no_rows_is_nothing(forge):
    """Zero rows, sequences or tokens: 0 without a GPU."""
    L, c = forge.lib(), cache(forge)
    assert L.forge_kv4_append(c, A, A, 256, A, A, 0, None) == 0
    assert L.forge_kv4_read(c, A, A, 0, A, A, 256, None) == 0
    assert L.forge_flash_prefill_varlen(A, 256, A, 256, A, 256, A, 0, 10, 2, 2, 128, A, 256, None, None) == 0
    assert L.forge_flash_prefill_varlen(A, 256, A, 256, A, 256, A, 3, 0, 2, 2, 128, A, 256, None, None) == 0
    assert L.forge_token_logprobs(A, 0, 100, 0, 100, A, 5, A, A, A, A, A, None) == 0


def test_decode_args(forge):
    L, c = forge.lib(), cache(forge)
    for q, seq, pos, B, H, out, ws in [(None, A, A, 3, 4, A, A), (A, A, None, 3, 4, A, A), (A, A, A, 3, 4, None, A),
                                       (A, A, A, 3, 4, A, None), (A, A, A, 0, 4, A, A), (A, A, A, 3, 0, A, A),
                                       (A, A, A, 3, 3, A, A), (A, None, A, 5, 4, A, A), (A + 4, A, A, 3, 4, A, A),
                                       (A, A, A, 3, 4, A + 8, A), (A, A, A, 3, 4, A, A + 8), (A, A, A, 65536, 4, A, A)]:
        refused(forge, L.forge_flash_decode_kv4(q, c, seq, pos, B, H, out, ws, None))
    for B, H, Hkv, hd in [(0, 4, 2, 128), (1, 0, 2, 128), (1, 4, 0, 128), (1, 4, 3, 128), (1, 4, 2, 80)]:
        assert L.forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd) == -1
    assert L.forge_flash_decode_kv4_workspace_bytes(3, 32, 8, 128) > 0


def test_prefill_args(forge):
    L = forge.lib()
    good = dict(q=A, ldq=512, k=A, ldk=256, v=A, ldv=256, cu=A, n=3, total=50, H=4, Hkv=2, hd=128, o=A, ldo=512)

    def call(**kw):
        a = dict(good, **kw)
        return L.forge_flash_prefill_varlen(*a.values(), A, None)

    for kw in [dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(cu=None), dict(n=-1), dict(total=-1),
               dict(H=0), dict(Hkv=0), dict(H=3), dict(ldq=504), dict(ldk=248), dict(ldv=248), dict(ldo=504),
               dict(ldq=516), dict(ldk=260), dict(ldv=257), dict(ldo=514), dict(q=A + 8), dict(k=A + 2), dict(v=A + 4),
               dict(o=A + 8), dict(n=65536), dict(H=1 << 17, ldq=1 << 24, ldo=1 << 24)]:
        refused(forge, call(**kw))
    for hd in (32, 96, 256):
        refused(forge, call(hd=hd), forge.FORGE_KERNEL_UNSUPPORTED)


def test_logprobs_args(forge):
    L = forge.lib()
    good = dict(z=A, dtype=0, ld=100, rows=4, vocab=100, tok=A, top=5, lp=A, ent=A, rank=A, ids=A, tops=A)

    def call(**kw):
        return L.forge_token_logprobs(*dict(good, **kw).values(), None)

    for kw in [dict(z=None), dict(dtype=2), dict(dtype=-1), dict(ld=99), dict(rows=-1), dict(vocab=0), dict(top=-1),
               dict(top=33), dict(vocab=4, top=5), dict(tok=None), dict(tok=None, rank=None), dict(tok=None, lp=None),
               dict(ids=None, tops=None), dict(z=A + 2), dict(z=A + 1, dtype=1)]:
        refused(forge, call(**kw))


def test_cache_descriptor_layout(forge):
    """The struct a hexa caller packs by hand (include/forge_kv4.h)."""
    f = forge.ForgeKv4
    assert C.sizeof(f) == 72
    assert [getattr(f, n).offset for n in ("k", "v", "ks", "vs", "table", "n_seq", "n_kv_head", "head_dim", "lmax",
                                           "page_tokens", "max_pages", "num_pages")] == \
        [0, 8, 16, 24, 32, 40, 44, 48, 52, 56, 60, 64]
