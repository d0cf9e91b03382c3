// attn_kv4.cu — flash-decode over the 4-bit KV cache (forge_kv4.h).
//
// out[h] = sum_j p_j v_j / sum_j p_j, p_j = exp(q_h . k_j / sqrt(hd)), with
// k_jd = sk_jg (n_jd - 7) and v alike (n the 4-bit code, g the group of 64
// dims). A KV head's keys are read once for up to 8 of its query heads, on
// m16n8k16 fp16 tensor-core products with fp32 sums:
//
//   S: A = q of 8 heads, rows 0-7 their fp16 heads and rows 8-15 what fp16
//      left over (q is first scaled by a power of two so that its largest
//      entry is near 2^15: the pair holds 22 bits), B = the codes of 8 keys.
//      (word >> 8k) & 0x000F000F is the fp16 pair (n, n') 2^-24, a
//      subnormal, & 0x00F000F0 sixteen times that, and one fp16 fma makes
//      either (n - 7) 2^-9 (exact). Subnormals fed to the tensor cores as
//      they are cost no fma, but a product is aligned by the exponent field,
//      not by its leading bit, and cut off 2^-25 below that: scores came out
//      8e-6 off. The key's scale multiplies each group's sum in fp32.
//   O: A = the weights p_j sv_jg of 8 heads as fp16 and remainder, times a
//      power of two that follows the largest scale seen, B = the codes of
//      two keys per register (one byte permute per four dims), less 7 in
//      the same way. A tile's product is added to O in fp32
//      registers: no chain of tensor-core sums is longer than 4.
//
// Work: the tiles of 64 keys of all (sequence, KV head, 8 query heads) form
// one line, cut into one range per CTA, so a batch of very different lengths
// is as even as one of equal ones. In a CTA each warp takes every fourth tile
// with a ring of bulk copies and a softmax of its own; a sequence's end in the
// range joins the four warps, and where a range ends inside a sequence the
// last CTA to arrive joins the CTAs that shared it, in the order of the keys.
#include <cmath>
#include <cuda_fp16.h>
#include "common.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"
#include "../../include/forge_kv4.h"

namespace {
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 64;          // keys per tile
constexpr int kStages = 2;         // tiles a warp has in flight
constexpr int kCtasPerSm = 3;
constexpr int kMinTiles = kWarps;  // a range gives every warp a tile
constexpr int kHeads = 8;          // query heads that share a pass over the keys

template <int HD>
struct Geo {
    static constexpr int kNG = HD / FORGE_KV4_GROUP;
    static constexpr int kCodes = kKeys * HD / 2, kScales = kKeys * kNG * 2;  // bytes of a tile, K or V
    static constexpr int kSlot = 2 * (kCodes + kScales);                      // K codes, V codes, K scales, V scales
    static constexpr int kRedHeads = 256 / HD;                                // heads joined at a time
    static constexpr int kOffRed = kWarps * kStages * kSlot;
    static constexpr int kOffMl = kOffRed + kWarps * 256 * 4;                 // [warp][8] m, then l
    static constexpr int kOffBar = kOffMl + 2 * kWarps * kHeads * 4;
    static constexpr int kSmem = kOffBar + kWarps * kStages * 8;
};

struct Kv4Args {
    ForgeKv4 c;
    const float* q;
    const int32_t *seq, *pos;
    int B, H, G, nhb, ph;   // query heads, heads per KV head, blocks of 8 of them, (KV head, block) pairs
    int cap;                // rows a sequence can hold
    float scale_log2;       // log2(e) / sqrt(hd)
    float* out;
    uint32_t* counters;     // [B][ph]
    float* partial;         // [CTA][2][8][hd + 2]
    uint32_t* err;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// x as fp16 and what that leaves, two values at once
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x0, x1);
    const float2 f = __half22float2(h);
    hi = h2bits(h);
    lo = h2bits(__floats2half2_rn(x0 - f.x, x1 - f.y));
}
// The codes in bits 0-3 (lo) or 4-7 (hi) of both halves, less 7 and times
// 2^-9, as an fp16 pair (exact).
__device__ __forceinline__ uint32_t fma2_bits(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}
__device__ __forceinline__ uint32_t code_lo(uint32_t w) { return fma2_bits(w & 0x000F000Fu, 0x78007800u, 0xA300A300u); }
__device__ __forceinline__ uint32_t code_hi(uint32_t w) { return fma2_bits(w & 0x00F000F0u, 0x68006800u, 0xA300A300u); }

// Tiles of sequence slot b; -1 when its position or sequence is out of range.
__device__ __forceinline__ int tiles_of(const Kv4Args& a, int b) {
    const int p = a.pos[b];
    if (p < 0) return 0;
    const int s = a.seq ? a.seq[b] : b;
    return (p >= a.cap || s < 0 || s >= a.c.n_seq) ? -1 : p / kKeys + 1;
}

// A place on the line of tiles: tile j of n of pair `pair` of sequence slot b.
struct Place {
    int b, pair, j, n;
    __device__ void settle(const Kv4Args& a) {  // after j grew; the place is on the line
        while (j >= n) {
            j -= n;
            if (++pair == a.ph) {
                pair = 0;
                do n = ++b < a.B ? max(0, tiles_of(a, b)) : 1 << 30;
                while (n == 0);
            }
        }
    }
};

template <int HD>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) k_kv4_decode(const Kv4Args a) {
    using X = Geo<HD>;
    constexpr int NG = X::kNG;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    uint8_t* ring = smem + warp * kStages * X::kSlot;
    float* red = reinterpret_cast<float*>(smem + X::kOffRed);
    float* sm_m = reinterpret_cast<float*>(smem + X::kOffMl);
    float* sm_l = sm_m + kWarps * kHeads;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + X::kOffBar) + warp * kStages;
    __shared__ int s_last;

    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }

    // ---- the line's length; sequences without tiles are answered here
    long long total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + lane;
        int n = b < a.B ? tiles_of(a, b) : 0;
        if (warp == 0) {
            unsigned none = __ballot_sync(0xffffffffu, b < a.B && n <= 0 && b % (int)gridDim.x == (int)blockIdx.x);
            for (; none; none &= none - 1) {
                const int w = __ffs(none) - 1;
                const bool bad = __shfl_sync(0xffffffffu, n, w) < 0;
                if (bad && lane == 0) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
                float* o = a.out + (size_t)(b0 + w) * a.H * HD;
                for (int i = lane; i < a.H * HD; i += 32) o[i] = bad ? NAN : 0.f;
            }
        }
        n = max(n, 0);
        total += __reduce_add_sync(0xffffffffu, n);
    }
    total *= a.ph;
    const long long per = max((long long)kMinTiles, (total + gridDim.x - 1) / gridDim.x);
    const long long start = (long long)blockIdx.x * per, end = min(total, start + per);
    if (start >= end) return;

    // ---- the place where this CTA's range starts
    Place at{0, 0, 0, 0};
    long long base = 0;  // line index of the first tile of slot at.b
    for (int b0 = 0;; b0 += 32) {
        const int b = b0 + lane;
        const int n = b < a.B ? max(0, tiles_of(a, b)) : 0;
        int inc = n;
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + (long long)inc * a.ph > start);
        if (past) {
            const int w = __ffs(past) - 1;
            at.n = __shfl_sync(0xffffffffu, n, w);
            base += (long long)(__shfl_sync(0xffffffffu, inc, w) - at.n) * a.ph;
            at.b = b0 + w;
            at.pair = (int)((start - base) / at.n);
            at.j = (int)(start - base - (long long)at.pair * at.n);
            break;
        }
        base += (long long)__shfl_sync(0xffffffffu, inc, 31) * a.ph;
    }
    __syncwarp();

    // ---- copies of this warp's tiles start + warp, + 4, ...
    Place in = at;
    in.j += warp;
    long long f_in = start + warp;
    int n_in = 0;
    uint32_t poison = 0;  // slots whose tile names a page outside the pool
    if (f_in < end) in.settle(a);
    auto issue = [&]() {
        if (f_in >= end) return;
        const int s = n_in % kStages;
        const int L = a.pos[in.b] + 1, sq = a.seq ? a.seq[in.b] : in.b, kvh = in.pair / a.nhb;
        const int key0 = in.j * kKeys;
        const int rows = min(kKeys, (L - key0 + 7) & ~7);
        uint8_t* dst = ring + s * X::kSlot;
        if (lane == 0) mbar_arrive_expect_tx(&full[s], rows * (HD + 4 * NG));
        __syncwarp();
        // lane 4i + k copies array k (K codes, V codes, K scales, V scales) of segment i
        const int seg = lane >> 2, arr = lane & 3;
        int r0 = 0, r1 = rows;
        int64_t row = 0;
        bool bad = false;
        if (!a.c.table) {
            if (seg) r1 = 0;
            row = ((int64_t)sq * a.c.n_kv_head + kvh) * a.c.lmax + key0;
        } else {
            const int pt = a.c.page_tokens, pg0 = key0 / pt;
            r0 = max(0, (pg0 + seg) * pt - key0);
            r1 = min(rows, (pg0 + seg + 1) * pt - key0);
            if (r0 < r1) {
                int pg = a.c.table[(int64_t)sq * a.c.max_pages + pg0 + seg];
                bad = (unsigned)pg >= (unsigned)a.c.num_pages;
                if (bad) {
                    atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
                    pg = 0;
                }
                row = ((int64_t)pg * a.c.n_kv_head + kvh) * pt + (key0 + r0) % pt;
            }
        }
        if (r0 < r1) {
            const int unit = arr < 2 ? HD / 2 : NG * 2;  // bytes a row
            const uint8_t* src = arr == 0 ? a.c.k : arr == 1 ? a.c.v : (const uint8_t*)(arr == 2 ? a.c.ks : a.c.vs);
            const int off = arr == 0 ? 0 : arr == 1 ? X::kCodes : 2 * X::kCodes + (arr - 2) * X::kScales;
            bulk_g2s_stream(dst + off + r0 * unit, src + row * unit, (r1 - r0) * unit, &full[s], l2_evict_first());
        }
        poison &= ~(1u << s);
        if (__any_sync(0xffffffffu, bad)) poison |= 1u << s;
        f_in += kWarps;
        ++n_in;
        in.j += kWarps;
        if (f_in < end) in.settle(a);
    };
    for (int s = 0; s < kStages; ++s) issue();

    int n_out = 0;
    bool dead = false;  // a wait ran out: nothing more is read
    for (long long f = start; f < end;) {
        // ---- one sequence's pair: tiles [f, f1) of the line
        const long long pair0 = f - at.j, pair1 = pair0 + at.n, f1 = min(end, pair1);
        const int kvh = at.pair / a.nhb, h0 = (at.pair % a.nhb) * kHeads, nh = min(kHeads, a.G - h0);
        const int L = a.pos[at.b] + 1;
        const size_t qrow = (size_t)at.b * a.H + kvh * a.G + h0;

        // q as A operands: head g, dims 64 gr + 16 t + 8 w + {0..7}; fp16 pairs (d, d + 4) and (d + 1, d + 5)
        // (in shared memory, one quarter from each warp: registers are short while the codes of V are unpacked)
        float fac;
        uint4* qs = reinterpret_cast<uint4*>(red);  // [4 NG][32 lanes]
        {
            float4 v[NG][4];
            float mx = 0.f;
#pragma unroll
            for (int i = 0; i < NG; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[i][j] = g < nh ? *reinterpret_cast<const float4*>(a.q + (qrow + g) * HD + 64 * i + 16 * t + 4 * j)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v[i][j].x), fabsf(v[i][j].y)), fmaxf(fabsf(v[i][j].z), fabsf(v[i][j].w))));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // 2^e <= mx < 2^(e + 1); q 2^(14 - e) fits fp16
            const int e = max(-110, min(120, (int)(__float_as_uint(mx) >> 23) - 127));
            const float up = pow2i(14 - e);
            fac = a.scale_log2 * 0x1p-5f * pow2i(e);  // 2^9 of the codes, 2^(e - 14) of q
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                // word warp / 2 of the 16 dims, dims 2 k, 2 k + 4 and 2 k + 1, 2 k + 5 of it, k = warp % 2
                const float4 lo4 = warp & 2 ? v[i][2] : v[i][0], hi4 = warp & 2 ? v[i][3] : v[i][1];
                const bool k = warp & 1;
                uint4 r;
                split_f16((k ? lo4.z : lo4.x) * up, (k ? hi4.z : hi4.x) * up, r.x, r.y);
                split_f16((k ? lo4.w : lo4.y) * up, (k ? hi4.w : hi4.y) * up, r.z, r.w);
                qs[(4 * i + warp) * 32 + lane] = r;
            }
        }
        __syncthreads();

        float m = -INFINITY, l = 0.f;
        float o[NG][8][2];  // [group][nibble][column pair]: dims 64 i + 16 t + n and + 8, times 2^(-9 + 14 - e_run)
        int e_run = -100;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 8; ++n) o[i][n][0] = o[i][n][1] = 0.f;

        for (long long ft = f + ((warp - (int)(f - start)) & (kWarps - 1)); ft < f1; ft += kWarps) {
            if (dead) break;
            const int s = n_out % kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (n_out / kStages) & 1, a.err))) {
                dead = true;  // the copies in flight land before the CTA exits
                while (++n_out < n_in) mbar_wait(&full[n_out % kStages], (n_out / kStages) & 1, a.err);
                break;
            }
            const uint8_t* kc = ring + s * X::kSlot;
            const uint8_t* vc = kc + X::kCodes;
            const uint8_t* ks = vc + X::kCodes;
            const uint8_t* vs = ks + X::kScales;
            const int left = L - (int)(ft - pair0) * kKeys;  // valid keys of the tile (may be more than 64)

            // ---- scores of keys 8 u + t and 8 u + 4 + t, head g (log2 units)
            uint32_t qa[NG][4][4];
#pragma unroll
            for (int i = 0; i < 4 * NG; ++i) {
                const uint4 r = qs[i * 32 + lane];
                qa[i / 4][i % 4][0] = r.x; qa[i / 4][i % 4][1] = r.y; qa[i / 4][i % 4][2] = r.z; qa[i / 4][i % 4][3] = r.w;
            }
            float x[8][2];
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint8_t* row = kc + (8 * u + (g >> 1) + 4 * (g & 1)) * (HD / 2) + t * 8;
                float x0 = 0.f, x1 = 0.f;
                uint32_t s0, s1;
                if (NG == 2) {
                    s0 = *reinterpret_cast<const uint32_t*>(ks + (8 * u + t) * 4);
                    s1 = *reinterpret_cast<const uint32_t*>(ks + (8 * u + 4 + t) * 4);
                } else {
                    s0 = *reinterpret_cast<const uint16_t*>(ks + (8 * u + t) * 2);
                    s1 = *reinterpret_cast<const uint16_t*>(ks + (8 * u + 4 + t) * 2);
                }
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const uint2 w = *reinterpret_cast<const uint2*>(row + 32 * i);
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16(c, qa[i][0], code_lo(w.x), code_hi(w.x));
                    mma_f16(c, qa[i][1], code_lo(w.x >> 8), code_hi(w.x >> 8));
                    mma_f16(c, qa[i][2], code_lo(w.y), code_hi(w.y));
                    mma_f16(c, qa[i][3], code_lo(w.y >> 8), code_hi(w.y >> 8));
                    x0 = fmaf(c[0] + c[2], i ? bf16_hi_f32(s0) : bf16_lo_f32(s0), x0);
                    x1 = fmaf(c[1] + c[3], i ? bf16_hi_f32(s1) : bf16_lo_f32(s1), x1);
                }
                x[u][0] = x0 * fac;
                x[u][1] = x1 * fac;
            }
            // ---- scales of V; keys behind the last one count for nothing
            uint32_t sv[8][2];
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    sv[u][k] = NG == 2 ? *reinterpret_cast<const uint32_t*>(vs + (8 * u + 4 * k + t) * 4)
                                       : *reinterpret_cast<const uint16_t*>(vs + (8 * u + 4 * k + t) * 2);
            if (left < kKeys) {
#pragma unroll
                for (int u = 0; u < 8; ++u)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (8 * u + 4 * k + t >= left) {
                            x[u][k] = -INFINITY;
                            sv[u][k] = 0;
                        }
            }
            __nv_bfloat162 smx = __floats2bfloat162_rn(0.f, 0.f);
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    mx = fmaxf(mx, x[u][k]);
                    smx = __hmax2(smx, *reinterpret_cast<const __nv_bfloat162*>(&sv[u][k]));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            float sm = fmaxf(__low2float(smx), __high2float(smx));
            sm = fmaxf(sm, __shfl_xor_sync(0xffffffffu, sm, 1));
            sm = fmaxf(sm, __shfl_xor_sync(0xffffffffu, sm, 2));
            const float m_new = fmaxf(m, mx);
            float alpha = ex2(m - m_new);  // 0 at the first tile
            if (m_new == -INFINITY) alpha = 1.f;
            m = m_new;
            const float m_ref = m_new == -INFINITY ? 0.f : m_new;
            // weights p sv 2^(14 - e) stay below 2^15; e follows the largest scale (the same in all lanes)
            const int e = max(e_run, min(129, (int)(__float_as_uint(sm) >> 23) - 126));
            const float up = pow2i(14 - e);
            const float alpha_o = e_run - e < -126 ? 0.f : alpha * pow2i(e_run - e);
            e_run = e;
            float ls = 0.f;
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float p = ex2(x[u][k] - m_ref);
                    ls += p;
                    x[u][k] = p * up;
                }
            l = fmaf(l, alpha, ls);

            // ---- O += P V, group by group
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                float c[8][4];
#pragma unroll
                for (int n = 0; n < 8; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    uint32_t pa[4];
                    float w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t s2 = sv[2 * kk + (j >> 1)][j & 1];
                        w[j] = x[2 * kk + (j >> 1)][j & 1] * (i ? bf16_hi_f32(s2) : bf16_lo_f32(s2));
                    }
                    split_f16(w[0], w[1], pa[0], pa[1]);
                    split_f16(w[2], w[3], pa[2], pa[3]);
                    uint32_t r[4];  // word g of group i of keys 16 kk + t + {0, 4, 8, 12}
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        r[j] = *reinterpret_cast<const uint32_t*>(vc + (16 * kk + 4 * j + t) * (HD / 2) + 32 * i + 4 * g);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        // nibbles 4 hf .. 4 hf + 3 of two keys side by side
                        const uint32_t p0 = __byte_perm(r[0], r[1], hf ? 0x7632 : 0x5410);
                        const uint32_t p1 = __byte_perm(r[2], r[3], hf ? 0x7632 : 0x5410);
                        mma_f16(c[4 * hf + 0], pa, code_lo(p0), code_lo(p1));
                        mma_f16(c[4 * hf + 1], pa, code_hi(p0), code_hi(p1));
                        mma_f16(c[4 * hf + 2], pa, code_lo(p0 >> 8), code_lo(p1 >> 8));
                        mma_f16(c[4 * hf + 3], pa, code_hi(p0 >> 8), code_hi(p1 >> 8));
                    }
                }
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    o[i][n][0] = fmaf(o[i][n][0], alpha_o, c[n][0] + c[n][2]);
                    o[i][n][1] = fmaf(o[i][n][1], alpha_o, c[n][1] + c[n][3]);
                }
            }
            if (poison >> s & 1) l = NAN;
            ++n_out;
            __syncwarp();
            issue();
        }
        if (dead) l = NAN;

        // ---- join the warps: O / l of the CTA's keys, with their (m, l)
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
            sm_m[warp * kHeads + g] = m;
            sm_l[warp * kHeads + g] = l;
        }
        __syncthreads();
        float mj = -INFINITY, lj = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mj = fmaxf(mj, sm_m[w * kHeads + g]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float mw = sm_m[w * kHeads + g];
            lj = fmaf(sm_l[w * kHeads + g], mw == -INFINITY ? 0.f : ex2(mw - mj), lj);
            if (isnan(sm_l[w * kHeads + g])) lj = NAN;
        }
        // o 2^(e_run - 5) ex2(m - mj) / lj
        const float fo = (m == -INFINITY ? 0.f : ex2(m - mj)) / lj * 0x1p15f;
        const float up0 = pow2i(e_run - 20);
        const bool whole = f == pair0 && f1 == pair1;  // no other CTA shares the pair
        const long long cfirst = pair0 / per, clast = (pair1 - 1) / per;
        float* part = a.partial + ((size_t)blockIdx.x * 2 + (blockIdx.x == cfirst)) * kHeads * (HD + 2);
        constexpr int RH = X::kRedHeads;
        for (int hr = 0; hr < nh; hr += RH) {
            if (g >= hr && g < hr + RH) {
                float* dst = red + (warp * RH + g - hr) * HD;
#pragma unroll
                for (int i = 0; i < NG; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int n = 0; n < 8; ++n)
                            dst[64 * i + 16 * t + 8 * k + n] = o[i][n][k] * fo * up0;
            }
            __syncthreads();
            for (int idx = threadIdx.x; idx < RH * HD; idx += kThreads) {
                const int h = hr + idx / HD, d = idx % HD;
                if (h < nh) {
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) v += red[w * RH * HD + idx];
                    if (whole) a.out[(qrow + h) * HD + d] = v;
                    else part[h * (HD + 2) + d] = v;
                }
            }
            __syncthreads();
        }
        if (!whole) {
            if (warp == 0 && t == 0 && g < nh) {
                part[g * (HD + 2) + HD] = mj;
                part[g * (HD + 2) + HD + 1] = lj;
            }
            // the last of the pair's CTAs joins them: the block barrier orders
            // the partial's stores before thread 0's release
            __syncthreads();
            if (threadIdx.x == 0) {
                uint32_t old;
                const uint32_t top = (uint32_t)(clast - cfirst);  // the counter returns to 0 after the last
                asm volatile("fence.acq_rel.gpu;" ::: "memory");
                asm volatile("atom.inc.acq_rel.gpu.global.u32 %0, [%1], %2;"
                             : "=r"(old) : "l"(a.counters + (size_t)at.b * a.ph + at.pair), "r"(top) : "memory");
                s_last = old == top;
            }
            __syncthreads();
            if (s_last) {
                const int nc = (int)(clast - cfirst) + 1;
                for (int h = warp; h < nh; h += kWarps) {
                    // slot of contribution c: the pair starts in the first CTA's range and before every other's
                    auto slot = [&](int c) {
                        return a.partial + (((size_t)cfirst + c) * 2 + (c == 0)) * kHeads * (HD + 2) + h * (HD + 2);
                    };
                    float mm = -INFINITY;
                    for (int c = lane; c < nc; c += 32) mm = fmaxf(mm, __ldcg(slot(c) + HD));
                    for (int d = 16; d; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
                    constexpr int E = HD / 32;
                    float acc[E] = {}, sum = 0.f;
                    for (int c0 = 0; c0 < nc; c0 += 32) {
                        float wl = 0.f;
                        if (c0 + lane < nc) {
                            const float mc = __ldcg(slot(c0 + lane) + HD), lc = __ldcg(slot(c0 + lane) + HD + 1);
                            wl = mc == -INFINITY && !isnan(lc) ? 0.f : lc * ex2(mc - mm);
                        }
                        const int cn = min(32, nc - c0);
                        for (int c = 0; c < cn; c += 8) {
                            float2 v[8][E / 2];
#pragma unroll
                            for (int j = 0; j < 8; ++j)
#pragma unroll
                                for (int k = 0; k < E / 2; ++k)
                                    if (c + j < cn) v[j][k] = __ldcg(reinterpret_cast<const float2*>(slot(c0 + c + j)) + 32 * k + lane);
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                const float w = __shfl_sync(0xffffffffu, wl, (c + j) & 31);
                                if (c + j < cn) {
                                    sum += w;
#pragma unroll
                                    for (int k = 0; k < E / 2; ++k) {
                                        acc[2 * k] = w == 0.f ? acc[2 * k] : fmaf(w, v[j][k].x, acc[2 * k]);
                                        acc[2 * k + 1] = w == 0.f ? acc[2 * k + 1] : fmaf(w, v[j][k].y, acc[2 * k + 1]);
                                    }
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < E / 2; ++k)
                        reinterpret_cast<float2*>(a.out + (qrow + h) * HD)[32 * k + lane] =
                            make_float2(acc[2 * k] / sum, acc[2 * k + 1] / sum);
                }
            }
        }
        f = f1;
        at.j = (int)(f1 - pair0);
        if (f < end) at.settle(a);
    }
}

int configure() {
    static bool done[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return forge_fail(-1, "forge_flash_decode_kv4: no device");
    if (done[dev]) return 0;
    cudaError_t e = cudaFuncSetAttribute(k_kv4_decode<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<64>::kSmem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_kv4_decode<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<128>::kSmem);
    for (auto k : {k_kv4_decode<64>, k_kv4_decode<128>})
        if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e != cudaSuccess) return forge_fail(-1, "forge_flash_decode_kv4: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
    return 0;
}

int64_t counter_bytes(int B, int H, int Hkv) {
    const int64_t pairs = (int64_t)B * Hkv * ((H / Hkv + kHeads - 1) / kHeads);
    return (pairs * 4 + 255) / 256 * 256;
}
constexpr int kMaxCtas = 148 * kCtasPerSm;  // a B200's; fixed so that workspace sizes do not depend on the device
}  // namespace

extern "C" FORGE_API int64_t forge_flash_decode_kv4_workspace_bytes(int B, int H, int n_kv_head, int head_dim) {
    if (B <= 0 || H <= 0 || n_kv_head <= 0 || H % n_kv_head || (head_dim != 64 && head_dim != 128)) return -1;
    return counter_bytes(B, H, n_kv_head) + (int64_t)kMaxCtas * 2 * kHeads * (head_dim + 2) * 4;
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
    if (configure()) return -1;
    const int hd = cache->head_dim;
    Kv4Args a{};
    a.c = *cache; a.q = q; a.seq = seq; a.pos = pos; a.B = B; a.H = H;
    a.G = H / cache->n_kv_head;
    a.nhb = (a.G + kHeads - 1) / kHeads;
    a.ph = cache->n_kv_head * a.nhb;
    a.cap = cache->table ? cache->max_pages * cache->page_tokens : cache->lmax;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)hd));
    a.out = out; a.err = err;
    a.counters = (uint32_t*)workspace;
    a.partial = (float*)((char*)workspace + counter_bytes(B, H, cache->n_kv_head));
    // no more CTAs than the longest sequences could feed
    const int64_t most = ((int64_t)B * a.ph * ((a.cap + kKeys - 1) / kKeys) + kMinTiles - 1) / kMinTiles;
    const int grid = (int)(most < kMaxCtas ? most : kMaxCtas);
    if (hd == 128) k_kv4_decode<128><<<grid, kThreads, Geo<128>::kSmem, (cudaStream_t)stream>>>(a);
    else k_kv4_decode<64><<<grid, kThreads, Geo<64>::kSmem, (cudaStream_t)stream>>>(a);
    return forge_check_launch("forge_flash_decode_kv4");
}
