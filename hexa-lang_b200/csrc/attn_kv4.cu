// attn_kv4.cu — flash-decode over the 4-bit KV cache (forge_kv4.h).
#include <cmath>
#include "common.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"
#include "../../include/forge_kv4.h"

namespace {
struct Kv4Args {
    ForgeKv4 c;
    const float* q;
    const int32_t *seq, *pos;
    int B, H;
    float* out;
    uint32_t* err;
};

// One CTA of head_dim threads per (query head, sequence), one key at a time:
// thread d holds dim d.
__global__ void k_kv4_decode(const Kv4Args a) {
    const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x, hd = a.c.head_dim, ng = hd / FORGE_KV4_GROUP;
    const int kvh = h / (a.H / a.c.n_kv_head);
    const int sq = a.seq ? a.seq[b] : b, P = a.pos[b];
    const int cap = a.c.table ? a.c.max_pages * a.c.page_tokens : a.c.lmax;
    __shared__ float red[4];
    float m = -INFINITY, l = 0.f, o = 0.f;
    bool bad = P >= cap || sq < 0 || sq >= a.c.n_seq;
    const float q = a.q[((size_t)b * a.H + h) * hd + d] / sqrtf((float)hd);
    for (int j = 0; !bad && j <= P; ++j) {
        size_t row = ((size_t)sq * a.c.n_kv_head + kvh) * a.c.lmax + j;
        if (a.c.table) {
            const int pg = a.c.table[(size_t)sq * a.c.max_pages + j / a.c.page_tokens];
            if ((unsigned)pg >= (unsigned)a.c.num_pages) { bad = true; break; }
            row = ((size_t)pg * a.c.n_kv_head + kvh) * a.c.page_tokens + j % a.c.page_tokens;
        }
        auto value = [&](const uint8_t* codes, const uint16_t* scales) {
            const int c = (codes[row * (hd / 2) + d / 2] >> (4 * (d & 1))) & 15;
            return (float)(c - 7) * bf16_bits_to_f32(scales[row * ng + d / FORGE_KV4_GROUP]);
        };
        float s = q * value(a.c.k, a.c.ks);
        for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
        __syncthreads();
        if ((d & 31) == 0) red[d >> 5] = s;
        __syncthreads();
        s = 0.f;
        for (int i = 0; i < hd / 32; ++i) s += red[i];
        const float mn = fmaxf(m, s), al = expf(m - mn), p = expf(s - mn);
        l = l * al + p;
        o = o * al + p * value(a.c.v, a.c.vs);
        m = mn;
    }
    if (bad && d == 0) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
    a.out[((size_t)b * a.H + h) * hd + d] = bad ? NAN : P < 0 ? 0.f : o / l;
}
}  // namespace

extern "C" FORGE_API int64_t forge_flash_decode_kv4_workspace_bytes(int B, int H, int n_kv_head, int head_dim) {
    if (B <= 0 || H <= 0 || n_kv_head <= 0 || H % n_kv_head || (head_dim != 64 && head_dim != 128)) return -1;
    return 256;
}

extern "C" FORGE_API int forge_flash_decode_kv4(const float* q, const ForgeKv4* cache, const int32_t* seq,
                                                const int32_t* pos, int B, int H, float* out, void* workspace,
                                                void* stream) {
    if (int rc = forge_kv4_check(cache, "forge_flash_decode_kv4")) return rc;
    if (!q || !pos || !out || !workspace || B <= 0 || B > 65535 || H <= 0 || H % cache->n_kv_head ||
        (!seq && B > cache->n_seq) || (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15))
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_decode_kv4: bad args (arrays 16-byte aligned, H a multiple of the KV heads)");
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_flash_decode_kv4: no device");
    Kv4Args a{*cache, q, seq, pos, B, H, out, err};
    k_kv4_decode<<<dim3(H, B), cache->head_dim, 0, (cudaStream_t)stream>>>(a);
    return forge_check_launch("forge_flash_decode_kv4");
}
