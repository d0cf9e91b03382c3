// prefill_varlen.cu — causal attention of packed prompts (grouped heads,
// sequences of any length back to back), bf16 in / bf16 out.
#include <cmath>
#include "common.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"

namespace {
struct VarlenArgs {
    const uint16_t *q, *k, *v;
    int64_t ldq, ldk, ldv, ldo;
    const int32_t* cu;
    int n_seq, total, H, Hkv, hd;
    uint16_t* o;
    float* lse;
    uint32_t* err;
};

// One warp per (row, head), one key at a time: lane l holds dims l, l + 32, ...
__global__ void __launch_bounds__(128) k_prefill_varlen(const VarlenArgs a) {
    const int s = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, E = a.hd / 32;
    const int r0 = a.cu[s], r1 = a.cu[s + 1];
    if (r0 < 0 || r1 < r0 || r1 > a.total) {
        if (threadIdx.x == 0) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
        return;
    }
    const int kvh = h / (a.H / a.Hkv);
    for (int r = r0 + blockIdx.x * 4 + (threadIdx.x >> 5); r < r1; r += gridDim.x * 4) {
        float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
        for (int e = 0; e < E; ++e) q[e] = bf16_bits_to_f32(a.q[r * a.ldq + h * a.hd + lane + 32 * e]) / sqrtf((float)a.hd);
        for (int j = r0; j <= r; ++j) {
            float x = 0.f;
            for (int e = 0; e < E; ++e) x = fmaf(q[e], bf16_bits_to_f32(a.k[j * a.ldk + kvh * a.hd + lane + 32 * e]), x);
            for (int i = 16; i; i >>= 1) x += __shfl_xor_sync(0xffffffffu, x, i);
            const float mn = fmaxf(m, x), al = expf(m - mn), p = expf(x - mn);
            for (int e = 0; e < E; ++e) o[e] = o[e] * al + p * bf16_bits_to_f32(a.v[j * a.ldv + kvh * a.hd + lane + 32 * e]);
            l = l * al + p;
            m = mn;
        }
        for (int e = 0; e < E; ++e) a.o[r * a.ldo + h * a.hd + lane + 32 * e] = f32_to_bf16_bits(o[e] / l);
        if (a.lse && lane == 0) a.lse[(int64_t)h * a.total + r] = m + logf(l);
    }
}
}  // namespace

extern "C" FORGE_API int forge_flash_prefill_varlen(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk,
                                                    const uint16_t* v, int64_t ldv, const int32_t* cu_seqlens, int n_seq,
                                                    int total, int H, int Hkv, int hd, uint16_t* o, int64_t ldo,
                                                    float* lse, void* stream) {
    if (!q || !k || !v || !o || !cu_seqlens || n_seq < 0 || total < 0 || H <= 0 || Hkv <= 0 || H % Hkv || n_seq > 65535 || H > 65535)
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_prefill_varlen: bad args");
    if (hd != 128 && hd != 64)
        return forge_fail(FORGE_KERNEL_UNSUPPORTED, "forge_flash_prefill_varlen: head_dim %d (128 or 64)", hd);
    if (ldq < (int64_t)H * hd || ldo < (int64_t)H * hd || ldk < (int64_t)Hkv * hd || ldv < (int64_t)Hkv * hd ||
        (ldq | ldk | ldv | ldo) % 8 || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) & 15))
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_prefill_varlen: rows must be 16-byte aligned and at least their heads long");
    if (n_seq == 0 || total == 0) return 0;
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_flash_prefill_varlen: no device");
    VarlenArgs a{q, k, v, ldq, ldk, ldv, ldo, cu_seqlens, n_seq, total, H, Hkv, hd, o, lse, err};
    k_prefill_varlen<<<dim3(64, H, n_seq), 128, 0, (cudaStream_t)stream>>>(a);
    return forge_check_launch("forge_flash_prefill_varlen");
}
