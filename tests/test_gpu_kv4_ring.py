"""The rings of copies of the 4-bit decode: a warp's first tiles, in calls so
short that they are all it has."""
import numpy as np
import pytest

import test_gpu_kv4 as kv4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,H,Hkv", [(64, 4, 4), (128, 4, 2), (64, 8, 2), (128, 8, 1)])
@pytest.mark.parametrize("page", [0, 16])
def test_first_tiles_of_short_calls(forge, cuda, hd, H, Hkv, page):
    """One to eight tiles a sequence, call after call into outputs that are cleared between them: the same bits each
    time, and no wait runs out."""
    import torch
    pos = [0, 63, 64, 127, 200, 300, 511, 5]
    B, L = len(pos), forge.lib()
    cache = kv4.Cache(forge, cuda, B, Hkv, hd, 512, page, seed=hd)
    q = np.random.default_rng(hd).standard_normal((B, H, hd)).astype(np.float32)
    want = kv4.reference(cache, q, pos)
    dq = torch.from_numpy(q.reshape(B, -1)).to(cuda)
    dp = torch.tensor(pos, dtype=torch.int32, device=cuda)
    out = torch.zeros(64, B, H * hd, device=cuda)
    ws = torch.zeros(L.forge_flash_decode_kv4_workspace_bytes(B, H, Hkv, hd), dtype=torch.uint8, device=cuda)
    out.fill_(float("nan"))
    for o in out:
        forge.check(L.forge_flash_decode_kv4(dq.data_ptr(), cache.desc, None, dp.data_ptr(), B, H, o.data_ptr(),
                                             ws.data_ptr(), kv4.stream()), "decode")
    torch.cuda.synchronize()
    forge.check(L.forge_ops_check(), "error word")
    kv4.check(out[0].cpu().numpy().reshape(B, H, hd), want)
    assert (out == out[0]).all()
