// kv4.cu — the 4-bit KV cache: rows quantised into it (append) and read back.
//
// Per group of 64 dims: s = bf16_rn(amax / 7), 1 where that is 0; code =
// x / s to the nearest integer, halves away from zero, clamped to -7..7, plus
// 7 (the rule of k_q4_quantize, weights.cu). A group with a value that is not
// finite gets a NaN scale.
//
// Bound by HBM for prompts (appending and reading 4096 rows of 32 heads of 128:
// 39 us, 6.1 TB/s, two launches), by latency for a decode step's rows (32 rows:
// 4.4 us for both). A CTA takes
// the K or the V of one row, so the row's place in the cache is looked up once;
// a thread takes 8 dims (16 bytes of bf16, 4 bytes of codes, 32 bytes of fp32),
// 8 neighbouring threads a group, and a row's loads are issued before its
// place is known.
#include "common.cuh"
#include "f32x2.cuh"
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

// Index of the cache row (slab * Hkv) * rows + row of head 0, or -1 (error word).
__device__ int64_t cache_row(const ForgeKv4& c, int s, int p, uint32_t* err) {
    const int cap = c.table ? c.max_pages * c.page_tokens : c.lmax;
    if (s >= 0 && s < c.n_seq && p < cap) {
        if (!c.table) return (int64_t)s * c.n_kv_head * c.lmax + p;
        const int pg = c.table[(int64_t)s * c.max_pages + p / c.page_tokens];
        if ((unsigned)pg < (unsigned)c.num_pages) return (int64_t)pg * c.n_kv_head * c.page_tokens + p % c.page_tokens;
    }
    if (threadIdx.x == 0) atomicOr(err, FORGE_DEVERR_BAD_INDEX);
    return -1;
}

constexpr int kThreads = 128;
constexpr int kAhead = 4;  // chunks of 8 dims a thread has in flight

// Codes of 8 dims (even dim in a byte's low nibble) of a group shared by 8
// neighbouring lanes, and the group's scale.
//
// Rounding x / s (halves away from zero) without a division: x and s are bf16
// values, so x / s is a half exactly or at least 2^-10 away from one (a
// difference of products of 8-bit integers over 2 s). x inv with inv = 1 / s
// to 2^-22, made larger by 2^-14, lies beyond a half that x / s meets and,
// below 7.5, not beyond one that it does not; an fma onto 1.5 2^23 + 7 then
// rounds it to the integer and leaves the code in the low bits. amax / 7 in
// the same way: the nearest bf16 of amax (1 / 7) is that of amax / 7, which
// is a bf16 value or at least 2^-13 of itself from a half between two.
__device__ __forceinline__ uint32_t quantise8(const uint4& x, uint16_t& scale) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t amax = max(m & 0xffffu, m >> 16);  // bf16 bits; infinity and NaN from 0x7F80 on
    scale = f32_to_bf16_bits(bf16_bits_to_f32((uint16_t)amax) * (1.0f / 7.0f));
    if (scale == 0) scale = 0x3F80;
    const float s = bf16_bits_to_f32(scale);
    const bool tiny = s < 0x1p-100f;  // (1 / s may be no fp32 number, and amax / s above 7.5)
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(tiny ? s * 0x1p64f : s));
    inv *= 1.0f + 0x1p-14f;
    uint32_t codes = 0;
    if (!__any_sync(0xffffffffu, tiny)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float y = fmaf(i & 1 ? bf16_hi_f32(w[i / 2]) : bf16_lo_f32(w[i / 2]), inv, 12582919.0f);
            codes += (__float_as_uint(y) - 0x4B400000u) << (4 * i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = (i & 1 ? bf16_hi_f32(w[i / 2]) : bf16_lo_f32(w[i / 2])) * (tiny ? 0x1p64f : 1.0f);
            const float y = fminf(fmaxf(fmaf(v, inv, 12582919.0f), 12582912.0f), 12582926.0f);
            codes += (__float_as_uint(y) - 0x4B400000u) << (4 * i);
        }
    }
    if (amax >= 0x7F80u) {
        scale = 0x7FC0;
        codes = 0x77777777u;
    }
    return codes;
}

template <int HD>
__global__ void __launch_bounds__(kThreads) k_kv4_append(const RowArgs a) {
    constexpr int kPer = HD / 8;  // chunks a head
    const int64_t r = blockIdx.x;
    const bool v = blockIdx.y;
    const int chunks = a.c.n_kv_head * kPer;
    const uint4* x = reinterpret_cast<const uint4*>((v ? a.v : a.k) + r * a.ld);
    uint4 in[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
        if (i * kThreads + (int)threadIdx.x < chunks) in[i] = __ldcs(x + i * kThreads + threadIdx.x);
    const int p = a.pos[r];
    if (p < 0) return;
    const int64_t row = cache_row(a.c, a.seq ? a.seq[r] : (int)r, p, a.err);
    if (row < 0) return;
    const int64_t head_rows = a.c.table ? a.c.page_tokens : a.c.lmax;  // from a head to the next
    uint32_t* codes = reinterpret_cast<uint32_t*>(v ? a.c.v : a.c.k) + row * kPer;
    uint16_t* scales = (v ? a.c.vs : a.c.ks) + row * (HD / kGroup);
    for (int base = 0; base < chunks; base += kAhead * kThreads) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (base + i * kThreads >= chunks) break;  // (the whole CTA: a group's lanes shuffle)
            const int c = base + i * kThreads + (int)threadIdx.x;
            uint16_t s;
            const uint32_t q = quantise8(in[i], s);
            if (c < chunks) {
                const int64_t at = (c / kPer) * head_rows;
                const int d = c % kPer;
                codes[at * kPer + d] = q;
                if (d % 8 == 0) scales[at * (HD / kGroup) + d / 8] = s;
            }
            const int next = c + kAhead * kThreads;
            if (next < chunks) in[i] = __ldcs(x + next);
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kThreads) k_kv4_read(const RowArgs a) {
    constexpr int kPer = HD / 8;
    const int64_t r = blockIdx.x;
    const bool v = blockIdx.y;
    const int chunks = a.c.n_kv_head * kPer;
    const int p = a.pos[r];
    if (p < 0) return;
    const int64_t row = cache_row(a.c, a.seq ? a.seq[r] : (int)r, p, a.err);
    const int64_t head_rows = a.c.table ? a.c.page_tokens : a.c.lmax;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(v ? a.c.v : a.c.k) + row * kPer;
    const uint16_t* scales = (v ? a.c.vs : a.c.ks) + row * (HD / kGroup);
    float4* out = reinterpret_cast<float4*>((v ? a.vo : a.ko) + r * a.ld);
    for (int base = 0; base < chunks; base += kAhead * kThreads) {
        uint32_t q[kAhead];
        uint16_t s[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int c = base + i * kThreads + (int)threadIdx.x;
            q[i] = 0;
            s[i] = 0x7FC0;  // a row out of range reads as NaN
            if (c < chunks && row >= 0) {
                const int64_t at = (c / kPer) * head_rows;
                q[i] = codes[at * kPer + c % kPer];
                s[i] = scales[at * (HD / kGroup) + c % kPer / 8];
            }
        }
        // a warp's 32 chunks in two stores of 512 contiguous bytes: lane l writes half l % 2 of chunk 16 j + l / 2
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (base + i * kThreads >= chunks) break;
            const int lane = threadIdx.x & 31, first = base + i * kThreads + ((int)threadIdx.x & ~31);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int from = 16 * j + lane / 2;
                const uint32_t w = __shfl_sync(0xffffffffu, q[i], from) >> (16 * (lane & 1));
                const float f = bf16_bits_to_f32((uint16_t)__shfl_sync(0xffffffffu, (uint32_t)s[i], from));
                F2 o[2];
#pragma unroll
                for (int k = 0; k < 2; ++k)  // code in the low bits of 2^23, exact less 2^23 + 7
                    o[k] = (F2(__uint_as_float((w >> (8 * k) & 15u) | 0x4B000000u), __uint_as_float((w >> (8 * k + 4) & 15u) | 0x4B000000u)) +
                            F2(-8388615.0f, -8388615.0f)) * F2(f, f);
                if (first + from < chunks) __stcs(out + 2 * first + 32 * j + lane, make_float4(o[0].x(), o[0].y(), o[1].x(), o[1].y()));
            }
        }
    }
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
    (cache->head_dim == 128 ? k_kv4_append<128> : k_kv4_append<64>)<<<dim3(n_rows, 2), kThreads, 0, (cudaStream_t)stream>>>(a);
    return forge_check_launch("forge_kv4_append");
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
    (cache->head_dim == 128 ? k_kv4_read<128> : k_kv4_read<64>)<<<dim3(n_rows, 2), kThreads, 0, (cudaStream_t)stream>>>(a);
    return forge_check_launch("forge_kv4_read");
}
