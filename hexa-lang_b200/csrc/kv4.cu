// kv4.cu — the 4-bit KV cache: rows quantised into it (append) and read back.
//
// Per group of 64 dims: s = bf16_rn(amax / 7), 1 where that is 0; code =
// x / s to the nearest integer, halves away from zero, clamped to -7..7, plus
// 7 (the rule of k_q4_quantize, weights.cu). A group with a value that is not
// finite gets a NaN scale.
#include "common.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"
#include "../../include/forge_kv4.h"

namespace {
constexpr int kGroup = FORGE_KV4_GROUP;

struct RowArgs {
    ForgeKv4 c;
    const uint16_t *k, *v;   // append: bf16 rows
    float *ko, *vo;          // read: fp32 rows
    int64_t ld;
    const int32_t *seq, *pos;
    int n_rows;
    uint32_t* err;
};

// Index of the cache row (slab * Hkv + head) * rows + row, or -1 (error word).
__device__ int64_t cache_row(const ForgeKv4& c, int s, int p, int head, uint32_t* err) {
    const int cap = c.table ? c.max_pages * c.page_tokens : c.lmax;
    if (s < 0 || s >= c.n_seq || p >= cap) {
        atomicOr(err, FORGE_DEVERR_BAD_INDEX);
        return -1;
    }
    if (!c.table) return ((int64_t)s * c.n_kv_head + head) * c.lmax + p;
    const int pg = c.table[(int64_t)s * c.max_pages + p / c.page_tokens];
    if ((unsigned)pg >= (unsigned)c.num_pages) {
        atomicOr(err, FORGE_DEVERR_BAD_INDEX);
        return -1;
    }
    return ((int64_t)pg * c.n_kv_head + head) * c.page_tokens + p % c.page_tokens;
}

// One warp per (row, head, K or V, group): lane l holds dims 2l, 2l + 1.
__global__ void __launch_bounds__(256) k_kv4_append(const RowArgs a) {
    const int lane = threadIdx.x & 31;
    const int ng = a.c.head_dim / kGroup;
    const int64_t n = (int64_t)a.n_rows * a.c.n_kv_head * 2 * ng;
    for (int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; w < n; w += (int64_t)gridDim.x * 8) {
        const int g = (int)(w % ng), kv = (int)(w / ng % 2), h = (int)(w / ng / 2 % a.c.n_kv_head);
        const int64_t r = w / ng / 2 / a.c.n_kv_head;
        const int p = a.pos[r];
        if (p < 0) continue;
        const int64_t row = cache_row(a.c, a.seq ? a.seq[r] : (int)r, p, h, a.err);
        if (row < 0) continue;
        const uint32_t x2 = *reinterpret_cast<const uint32_t*>((kv ? a.v : a.k) + r * a.ld + h * a.c.head_dim + g * kGroup + 2 * lane);
        const float x[2] = {bf16_lo_f32(x2), bf16_hi_f32(x2)};
        float m = fmaxf(fabsf(x[0]), fabsf(x[1]));
        if (!(fabsf(x[0]) <= 3.4e38f) || !(fabsf(x[1]) <= 3.4e38f)) m = INFINITY;
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        uint16_t sb = m == INFINITY ? 0x7FC0 : f32_to_bf16_bits(m / 7.0f);
        if (sb == 0) sb = 0x3F80;
        const float s = bf16_bits_to_f32(sb);
        uint32_t byte = 0;
        for (int i = 0; i < 2; ++i) {
            const float q = m == INFINITY ? 0.f : x[i] / s;
            const int c = max(-7, min(7, (int)(q + (q < 0.f ? -0.5f : 0.5f)))) + 7;
            byte |= (uint32_t)c << (4 * i);
        }
        (kv ? a.c.v : a.c.k)[row * (a.c.head_dim / 2) + g * (kGroup / 2) + lane] = (uint8_t)byte;
        if (lane == 0) (kv ? a.c.vs : a.c.ks)[row * ng + g] = sb;
    }
}

// One warp per (row, head, K or V, group): lane l writes dims 2l, 2l + 1.
__global__ void __launch_bounds__(256) k_kv4_read(const RowArgs a) {
    const int lane = threadIdx.x & 31;
    const int ng = a.c.head_dim / kGroup;
    const int64_t n = (int64_t)a.n_rows * a.c.n_kv_head * 2 * ng;
    for (int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5; w < n; w += (int64_t)gridDim.x * 8) {
        const int g = (int)(w % ng), kv = (int)(w / ng % 2), h = (int)(w / ng / 2 % a.c.n_kv_head);
        const int64_t r = w / ng / 2 / a.c.n_kv_head;
        const int p = a.pos[r];
        if (p < 0) continue;
        const int64_t row = cache_row(a.c, a.seq ? a.seq[r] : (int)r, p, h, a.err);
        float2 o = make_float2(NAN, NAN);
        if (row >= 0) {
            const uint32_t byte = (kv ? a.c.v : a.c.k)[row * (a.c.head_dim / 2) + g * (kGroup / 2) + lane];
            const float s = bf16_bits_to_f32((kv ? a.c.vs : a.c.ks)[row * ng + g]);
            o = make_float2((float)((int)(byte & 15) - 7) * s, (float)((int)(byte >> 4) - 7) * s);
        }
        *reinterpret_cast<float2*>((kv ? a.vo : a.ko) + r * a.ld + h * a.c.head_dim + g * kGroup + 2 * lane) = o;
    }
}

int rows_entry(const char* what, const RowArgs& a, void (*kern)(RowArgs), cudaStream_t stream) {
    const int64_t warps = (int64_t)a.n_rows * a.c.n_kv_head * 2 * (a.c.head_dim / kGroup);
    const int64_t blocks = (warps + 7) / 8, most = 16ll * forge_sm_count();
    kern<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(a);
    return forge_check_launch(what);
}
}  // namespace

// Shape, pointers and alignment of a cache descriptor; 0 or FORGE_INVALID_ARGS.
int forge_kv4_check(const ForgeKv4* c, const char* what) {
    if (!c || !c->k || !c->v || !c->ks || !c->vs || c->n_seq <= 0 || c->n_kv_head <= 0 ||
        (c->head_dim != 64 && c->head_dim != 128))
        return forge_fail(FORGE_INVALID_ARGS, "%s: bad cache (null array, no sequence or head, or head_dim not 64 or 128)", what);
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->ks | (uintptr_t)c->vs) & 15)
        return forge_fail(FORGE_INVALID_ARGS, "%s: the cache's arrays must be 16-byte aligned", what);
    if (!c->table) {
        if (c->lmax <= 0 || c->lmax % 8 || c->lmax > (1 << 30))
            return forge_fail(FORGE_INVALID_ARGS, "%s: lmax %d must be a positive multiple of 8", what, c->lmax);
    } else if (c->page_tokens <= 0 || c->page_tokens % 8 || c->max_pages <= 0 || c->num_pages <= 0 ||
               (int64_t)c->max_pages * c->page_tokens > (1 << 30)) {
        return forge_fail(FORGE_INVALID_ARGS, "%s: bad pages (page_tokens %d must be a multiple of 8, max_pages %d, num_pages %d)",
                          what, c->page_tokens, c->max_pages, c->num_pages);
    }
    return 0;
}

extern "C" FORGE_API int forge_kv4_append(const ForgeKv4* cache, const uint16_t* k, const uint16_t* v, int64_t ld,
                                          const int32_t* seq, const int32_t* pos, int n_rows, void* stream) {
    if (int rc = forge_kv4_check(cache, "forge_kv4_append")) return rc;
    if (!k || !v || !pos || n_rows < 0 || ld < (int64_t)cache->n_kv_head * cache->head_dim || ld % 8 ||
        (((uintptr_t)k | (uintptr_t)v) & 15) || (!seq && n_rows > cache->n_seq))
        return forge_fail(FORGE_INVALID_ARGS, "forge_kv4_append: bad args (rows 16-byte aligned, ld a multiple of 8 and at least a row)");
    if (n_rows == 0) return 0;
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_kv4_append: no device");
    RowArgs a{*cache, k, v, nullptr, nullptr, ld, seq, pos, n_rows, err};
    return rows_entry("forge_kv4_append", a, k_kv4_append, (cudaStream_t)stream);
}

extern "C" FORGE_API int forge_kv4_read(const ForgeKv4* cache, const int32_t* seq, const int32_t* pos, int n_rows,
                                        float* k_out, float* v_out, int64_t ld, void* stream) {
    if (int rc = forge_kv4_check(cache, "forge_kv4_read")) return rc;
    if (!k_out || !v_out || !pos || n_rows < 0 || ld < (int64_t)cache->n_kv_head * cache->head_dim || ld % 4 ||
        (((uintptr_t)k_out | (uintptr_t)v_out) & 15) || (!seq && n_rows > cache->n_seq))
        return forge_fail(FORGE_INVALID_ARGS, "forge_kv4_read: bad args (rows 16-byte aligned, ld a multiple of 4 and at least a row)");
    if (n_rows == 0) return 0;
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_kv4_read: no device");
    RowArgs a{*cache, nullptr, nullptr, k_out, v_out, ld, seq, pos, n_rows, err};
    return rows_entry("forge_kv4_read", a, k_kv4_read, (cudaStream_t)stream);
}
