// attn_kv4.cu — flash-decode over the 4-bit KV cache (forge_kv4.h).
//
// out[h] = sum_j p_j v_j / sum_j p_j, p_j = exp(q_h . k_j / sqrt(hd)), with
// k_jd = sk_jg (n_jd - 7) and v alike (n the 4-bit code, g the group of 64
// dims). The products are m16n8k32 ones of 8-bit integers with 32-bit sums,
// which are exact. The codes are bytes after a mask (and a shift for odd dims of
// K); a factor in fp32 becomes three base-256 digits.
//
//   S: q times a power of two as 24-bit integers, signed digits; -7 sum q is
//      in the initial sum. A group's sum is multiplied by the key's scale in
//      fp32.
//   O: the weights p_j sv_jg of a tile as integers below 2^23, relative to the
//      largest of them (of a head and group): added to 2^23 their digits are the
//      fp32's low bytes. A unit of p's and sv's own maxima would lose the bits
//      of a sink, a key that has the weight but not the scale. Groups of zeros,
//      whose scale is 1 by the format, are left out of it. ldmatrix transposes
//      V's bytes, so that a register holds a byte of four keys; odd dims stay
//      times 16 in theirs.
//      One more product, with a constant 7, gives 7 times the sum of the
//      weights, taken off exactly before the tile joins O in fp32.
//
// A sum starts at 1.5 2^23 as an integer's bits, so its bits are the fp32
// 12582912 + sum and need no conversion.
//
// Two forms, for how many query heads read a KV head. Up to 2: keys and dims
// are the 16 rows of A and the digits of both heads 6 of the 8 columns, so a lane
// has half of a tile's scores, exponentials and sums of the other form: 800
// instructions for 64 keys of 128 dims (pairs' starts and joins among them), and
// 168 registers let 3 CTAs share an SM. 3 and more: 4 heads' digits are 12 of
// the 16 rows, keys and dims the 8 columns: 980 instructions (pages of 32), fewer
// than two passes of the first form, and the keys are read once for the 4.
// Measured, 64 sequences of 4096 with 40 heads of 128, each reading its own KV head
// (1.43 GB; 218 us at the rate of a copy): 222 us in the first form, 6.4 TB/s,
// bound by HBM, next by shared-memory banks (0.74 of the wavefronts: ldmatrix's
// rows 64 bytes apart share them), 259 with 2 CTAs an SM; 280 in the second, bound by
// issue and latencies (0.41 of the issue slots with 2 warps a scheduler; 3 would
// have 168 registers and spill). 32 ragged sequences up to 16384, 4 heads a KV head:
// 29.7 us in the second form, 37.5 in the first. The same products in fp16, q and
// weights as pairs of fp16, took 379 for the former. Short contexts are a chain of
// latencies: 10 us for one sequence of 2048. The unit of the weights costs 2 to 4%:
// without it (see O) 217 and 28.2 us.
//
// Work: the tiles of 64 keys of all (sequence, KV head, heads of a pass) form
// one line, every pair's tiles behind a few units for what a pair costs by
// itself, cut into one range per CTA, so a batch of very different lengths is
// as even as one of equal ones. In a CTA each warp takes every fourth tile
// with a ring of bulk copies and a softmax of its own; a pair's end in the
// range joins the four warps, and where a range ends inside a pair the last
// CTA to arrive joins the CTAs that shared it, in the order of the keys.
#include <algorithm>
#include <cmath>
#include "common.cuh"
#include "f32x2.cuh"
#include "forge_internal.h"
#include "ring.cuh"
#include "../../include/forge_b200.h"
#include "../../include/forge_kv4.h"

namespace {
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kKeys = 64;          // keys per tile
constexpr int kStages = 2;         // tiles a warp has in flight
constexpr int kCtasMany = 2, kCtasFew = 3;  // CTAs per SM
constexpr int kPairUnits = 6;      // what a pair costs beside its tiles, in tiles (4: 30.5 us for 32 ragged sequences, 6: 29.7)
constexpr int kMinUnits = 2 * kWarps;  // least range of a CTA
constexpr int kJoin = kWarps / 2;  // sums of warps that shared memory holds at the end of a pair
constexpr int kHeadsMany = 4, kHeadsFew = 2;  // query heads that share a pass over the keys
constexpr int kMagic = 0x4B400000; // 1.5 2^23 as fp32

template <int HD>
struct Geo {
    static constexpr int kNG = HD / FORGE_KV4_GROUP;
    static constexpr int kCodes = kKeys * HD / 2, kScales = kKeys * kNG * 2;  // bytes of a tile, K or V
    static constexpr int kSlot = 2 * (kCodes + kScales);                      // K codes, V codes, K scales, V scales
};

struct Kv4Args {
    ForgeKv4 c;
    const float* q;
    const int32_t *seq, *pos;
    int B, H, G, nhb, ph;   // query heads, heads per KV head, blocks of them that share a pass, (KV head, block) pairs
    int cap;                // rows a sequence can hold
    float scale_log2;       // log2(e) / sqrt(hd)
    float* out;
    uint32_t* counters;     // [B][ph]
    float* partial;         // [CTA][2][heads of a pass][hd + 2]
    uint32_t* err;
};

// d = A B + c: m16n8k32, 8-bit integers, 32-bit integer sums.
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, const int4& c) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w));
}
__device__ __forceinline__ void mma_u8u8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, const int4& c) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], const uint4& a, uint32_t b0, uint32_t b1, const int4& c) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w));
}
__device__ __forceinline__ int4 quad(const int (&d)[4]) { return make_int4(d[0], d[1], d[2], d[3]); }
// The codes of even dims of a word (or of a byte of four keys), of odd ones times 16.
__device__ __forceinline__ uint32_t even(uint32_t w) { return w & 0x0F0F0F0Fu; }
__device__ __forceinline__ uint32_t odd16(uint32_t w) { return w & 0xF0F0F0F0u; }
// Bytes of two words; a selector of 8 + b gives 0 where byte b is not negative.
__device__ __forceinline__ uint32_t prmt(uint32_t x, uint32_t y, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(sel));
    return r;
}
__device__ __forceinline__ uint32_t low_bytes(const uint32_t* w) { return prmt(prmt(w[0], w[1], 0x40), prmt(w[2], w[3], 0x40), 0x5410); }
// Bytes of 32 rows of 16, transposed: r[k] has bytes g (k 0, 2) or 8 + g (k 1, 3) of rows 4 t .. 4 t + 3 (k 0, 1) or 16
// more (k 2, 3). Lane l gives row l's address.
__device__ __forceinline__ void load_transposed(uint32_t (&r)[4], const uint8_t* row) {
    asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(row)));
}
// The scales of keys 4 r .. 4 r + 3, and those of keys 2 f, 2 f + 1 of them for a group.
template <int NG>
struct Scales {
    uint32_t w[2 * NG];
    __device__ __forceinline__ Scales(const uint8_t* base, int r) {
        if constexpr (NG == 2) {
            const uint4 v = reinterpret_cast<const uint4*>(base)[r];
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
            const uint2 v = reinterpret_cast<const uint2*>(base)[r];
            w[0] = v.x; w[1] = v.y;
        }
    }
    __device__ __forceinline__ F2 of(int f, int group) const {
        if constexpr (NG == 1) return F2(bf16_lo_f32(w[f]), bf16_hi_f32(w[f]));
        else return group ? F2(bf16_hi_f32(w[2 * f]), bf16_hi_f32(w[2 * f + 1])) : F2(bf16_lo_f32(w[2 * f]), bf16_lo_f32(w[2 * f + 1]));
    }
};
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p = 0;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\t@e mov.s32 %0, 1;\n\t}" : "+r"(p));
    return p;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127
// The scores' integer sums (below 2^32 for q's below 2^e) are taken down by this power of two, so that no scale of K takes
// them out of fp32's range; not for q's so large that a large scale would take the score itself out.
__device__ __forceinline__ int sum_down(int e) { return e <= 64 ? 32 : 0; }
// Factors of a lane's two sums that start at 1.5 2^23, and what takes that off.
__device__ __forceinline__ int4 factors(float a, float b) {
    return make_int4(__float_as_int(a), __float_as_int(b), __float_as_int(-12582912.f * (a + b)), 0);
}
__device__ __forceinline__ F2 float_bits(int x, int y) { return F2(__int_as_float(x), __int_as_float(y)); }

// Tiles of sequence slot b; -1 when its position or sequence is out of range.
__device__ __forceinline__ int tiles_of(const Kv4Args& a, int b) {
    const int p = a.pos[b];
    if (p < 0) return 0;
    const int s = a.seq ? a.seq[b] : b;
    return (p >= a.cap || s < 0 || s >= a.c.n_seq) ? -1 : p / kKeys + 1;
}

// A pair on the line: pair `pair` of sequence slot b, n tiles, units base ..
// base + kPairUnits + n - 1.
struct Place {
    int b, pair, n, base;
    __device__ void next(const Kv4Args& a) {  // (behind the last pair: a place past every range)
        base += kPairUnits + n;
        if (++pair == a.ph) {
            pair = 0;
            do n = ++b < a.B ? max(0, tiles_of(a, b)) : 1 << 29;
            while (n == 0);
        }
    }
    // tiles of the pair inside units [start, end)
    __device__ int lo(int start) const { return max(0, start - base - kPairUnits); }
    __device__ int hi(int end) const { return min(n, end - base - kPairUnits); }
    // first tile at or behind j that is warp w's
    __device__ int mine(int j, int w) const { return j + ((w - j - pair) & (kWarps - 1)); }
};

// Zeroes the scales of a tile behind its `left` keys.
template <int HD>
__device__ __forceinline__ void clear_scales(uint8_t* vs, int left, int lane) {
    constexpr int NG = HD / FORGE_KV4_GROUP;
#pragma unroll
    for (int k = 0; k < kKeys * NG; k += 32)
        if (k + lane >= left * NG) reinterpret_cast<uint16_t*>(vs)[k + lane] = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before the copies that come into the slot)
    __syncwarp();
}
// Whether a scale of the tile may be exactly 1.
template <int HD>
__device__ __forceinline__ bool has_one(const uint8_t* vs, int lane) {
    constexpr int NG = HD / FORGE_KV4_GROUP;
    uint32_t w = 0xFFFFFFFFu;
#pragma unroll
    for (int k = 0; k < kKeys * NG / 2; k += 32) w = __vminu2(w, reinterpret_cast<const uint32_t*>(vs)[k + lane] ^ 0x3F803F80u);
    return !(w & 0xffffu) || !(w >> 16);
}
// Makes the scales of a tile's groups of zeros 0: the format gives them 1, which would be the unit of the weights where
// the other values are small. (Only a scale of exactly 1 has its codes looked at; other groups have a code of 0 or 14.)
template <int HD>
__device__ __forceinline__ void drop_zeros(bool one, uint8_t* vs, const uint8_t* vc, int lane) {
    constexpr int NG = HD / FORGE_KV4_GROUP;
    if (!__any_sync(0xffffffffu, one)) return;
#pragma unroll 1
    for (int e = lane; e < kKeys * NG; e += 32) {
        uint16_t* s = reinterpret_cast<uint16_t*>(vs) + e;
        if (*s != 0x3F80u) continue;
        const uint4* c = reinterpret_cast<const uint4*>(vc + e / NG * (HD / 2) + e % NG * 32);
        const uint4 a = c[0], b = c[1];
        if ((a.x & a.y & a.z & a.w & b.x & b.y & b.z & b.w) == 0x77777777u && (a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w) == 0x77777777u) *s = 0;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // (before the copies that come into the slot)
    __syncwarp();
}
// Scores (times log2 e) beyond this are taken relative to the tile's largest before they are multiplied: rounded, that is
// steps of 2 and more off, and the largest p would be as far below 1, or 0.
constexpr float kFar = 0x1p24f;
// The bits of a weight, for the largest of a tile: negative or no number (a scale that is) above all others.
__device__ __forceinline__ uint32_t larger(uint32_t m, F2 y) { return __vimax3_u32(m, __float_as_uint(y.x()), __float_as_uint(y.y())); }
constexpr uint32_t kNoWeight = 0x7F800000u;  // from here on
constexpr float kLeastUnit = 0x1p-100f;      // of a tile's largest weight (its inverse times 2^23 is an fp32 number)
// A key's scales, both groups' or one's.
template <int NG>
__device__ __forceinline__ uint32_t scale_word(const uint8_t* base, int key) {
    if constexpr (NG == 2) return reinterpret_cast<const uint32_t*>(base)[key];
    else return reinterpret_cast<const uint16_t*>(base)[key];
}

// ---- up to 4 query heads: keys in the columns of B, digits in the rows of A
// (rows r: digit 2, 1, 0 of head r % 4 for r < 4, r < 8, 8 <= r < 12)
template <int HD>
struct Many {
    static constexpr int kHeads = kHeadsMany, kCtas = kCtasMany, NG = HD / FORGE_KV4_GROUP, U = kKeys / 8;
    static constexpr int kSmem = 2 * NG * 512 + NG * 128 + 16 + 128;  // A operands of q [2 groups][32 lanes], sums to start from [groups][8], kMagic, factors [8]
    const int warp, lane, g, t, h;
    const float da, db;       // this lane's rows: digit a (2 or 1) and digit b (0, or none) of head h
    const uint32_t sel;       // digits a of two words, then digits b
    uint4* qs;
    int4* from;
    float fac, m;
    F2 l, o[NG][8];  // o[group][2 k + b]: dims 64 i + 16 k + 4 t + b and + 2, this lane's digits' part

    __device__ Many(uint8_t* smem, int warp, int lane)
        : warp(warp), lane(lane), g(lane >> 2), t(lane & 3), h(g & 3), da(g < 4 ? 65536.f : 256.f), db(g < 4 ? 1.f : 0.f),
          sel(g < 4 ? 0x4062 : 0xBB51), qs(reinterpret_cast<uint4*>(smem)),
          from(reinterpret_cast<int4*>(smem + 2 * NG * 512)) {
        if (threadIdx.x == 0) from[8 * NG] = make_int4(kMagic, kMagic, kMagic, kMagic);
    }
    __device__ int q_head() const { return h; }
    __device__ bool holds() const { return g < 4; }      // the sums of head h, after sum_lanes()
    __device__ bool first() const { return lane < 16 && t == 0; }  // of those that hold it

    // q (dims 64 i + 16 t .. + 15 of head h) as A operands, dims 64 i + 16 t + 8 w + {0, 2, 4, 6} and {1, 3, 5, 7} (in
    // shared memory, word w of group i from warp 2 i + w), and the sums that they start from
    __device__ __forceinline__ void stage(const float4 (&v)[NG][4], float scale_log2) {
        uint32_t mx = 0;  // largest |q| as bits
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mx = max(max(mx, __float_as_uint(fabsf(v[i][j].x))), __float_as_uint(fabsf(v[i][j].y)));
                mx = max(max(mx, __float_as_uint(fabsf(v[i][j].z))), __float_as_uint(fabsf(v[i][j].w)));
            }
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^e > 1.004 |q|: |q| 2^(23 - e) is at most 127 (1 + 2^8 + 2^16), the largest three signed digits
        const int e = (int)(__float_as_uint(1.004f * __uint_as_float(mx)) >> 23) - 126, sd = sum_down(e);
        const float up = pow2i(min(23 - e, 127)), up2 = pow2i(max(23 - e, 127) - 127);  // (for the smallest q, two factors)
        const float down = pow2i(-sd);
        if (warp == 0 && t == 0) from[8 * NG + 1 + g] = factors(da * down, db * down);
        fac = mx >= 0x7F800000u ? NAN : scale_log2 * pow2i(e - 23 + sd);  // (an infinite or NaN q: all NaN)
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            int sa = 0, sb = 0;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float4 lo4 = v[i][2 * w], hi4 = v[i][2 * w + 1];
                const float x[8] = {lo4.x, lo4.z, hi4.x, hi4.z, lo4.y, lo4.w, hi4.y, hi4.w};  // even dims, odd dims
                uint32_t da[8], db[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int n = __float2int_rn(x[k] * up * up2), d0 = (int)(int8_t)n, n1 = (n - d0) >> 8, d1 = (int)(int8_t)n1;
                    da[k] = g < 4 ? (n1 - d1) >> 8 : d1;
                    db[k] = g < 4 ? d0 : 0;
                }
                const uint4 r = make_uint4(low_bytes(da), low_bytes(db), low_bytes(da + 4), low_bytes(db + 4));
                if (warp == 2 * i + w) qs[(2 * i + w) * 32 + lane] = r;
                sa = __dp4a((int)r.z, 0x01010101, __dp4a((int)r.x, 0x01010101, sa));
                sb = __dp4a((int)r.w, 0x01010101, __dp4a((int)r.y, 0x01010101, sb));
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                sa += __shfl_xor_sync(0xffffffffu, sa, o);
                sb += __shfl_xor_sync(0xffffffffu, sb, o);
            }
            if (warp == 0 && t == 0) from[8 * i + g] = make_int4(kMagic - 7 * sa, kMagic - 7 * sa, kMagic - 7 * sb, kMagic - 7 * sb);
        }
        m = -INFINITY;
        l = F2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 8; ++n) o[i][n] = F2(0.f, 0.f);
    }

    __device__ __forceinline__ void tile(uint8_t* slot, int left) {
        const uint8_t *kc = slot, *ks = slot + 2 * Geo<HD>::kCodes;
        uint8_t* vs = slot + 2 * Geo<HD>::kCodes + Geo<HD>::kScales;
        const uint8_t* krow = kc + (4 * (g >> 1) + (g & 1)) * (HD / 2) + 8 * t;  // this lane's keys of B, and of V's transposition
        const uint8_t* vrow = kc + Geo<HD>::kCodes + lane * (HD / 2);
        const bool one = has_one<HD>(vs, lane);
        const int4 fs = from[8 * NG + 1 + g];
        const float sa = __int_as_float(fs.x), sb = __int_as_float(fs.y), off = __int_as_float(fs.z);
        // ---- scores of keys 16 (u / 2) + 4 t + 2 (u % 2) + {0, 1}, head h, over fac
        F2 x[U];
#pragma unroll
        for (int u0 = 0; u0 < U; u0 += 2) {
            const Scales<NG> sk(ks, 2 * u0 + t);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint4 q0 = qs[2 * i * 32 + lane], q1 = qs[(2 * i + 1) * 32 + lane];
                const int4 c0 = from[8 * i + g];
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                    const uint2 w = *reinterpret_cast<const uint2*>(krow + (8 * u0 + 2 * f) * (HD / 2) + 32 * i);
                    int c[4];
                    mma_s8u8(c, q0, even(w.x), even(w.x >> 4), c0);
                    mma_s8u8(c, q1, even(w.y), even(w.y >> 4), quad(c));
                    // digit a times sa + digit b times sb; both offsets of 12582912 come off exactly with the first
                    const F2 sum = fma2(float_bits(c[2], c[3]), F2(sb, sb), fma2(float_bits(c[0], c[1]), F2(sa, sa), F2(off, off)));
                    x[u0 + f] = i ? fma2(sum, sk.of(f, i), x[u0 + f]) : sum * sk.of(f, i);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)  // the other digits
            x[u] = x[u] + F2(__shfl_xor_sync(0xffffffffu, x[u].x(), 16), __shfl_xor_sync(0xffffffffu, x[u].y(), 16));
        // ---- the tile's largest score; keys behind the last one count for nothing
        if (left < kKeys) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                {
                const int key = 8 * (u & ~1) + 2 * (u & 1) + 4 * t;
                x[u] = F2(key < left ? x[u].x() : -INFINITY, key + 1 < left ? x[u].y() : -INFINITY);
            }
            clear_scales<HD>(vs, left, lane);
        }
        drop_zeros<HD>(one, vs, kc + Geo<HD>::kCodes, lane);
        float mx = fmaxf(x[0].x(), x[0].y());
#pragma unroll
        for (int u = 1; u < U; ++u) mx = max3(mx, x[u].x(), x[u].y());
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float top = mx;
        mx = __fmul_ru(mx, fac);  // (up, so that no difference to it comes out above 0)
        // p = 2^(x - mx) <= 1
        float nmx = mx == -INFINITY ? 0.f : -mx;
        if (fabsf(mx) > kFar && fabsf(mx) < INFINITY) {
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = x[u] + F2(-top, -top);
            nmx = 0.f;
        }
        F2 ls;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const F2 y = fma2(x[u], F2(fac, fac), F2(nmx, nmx));
            x[u] = F2(ex2(y.x()), ex2(y.y()));
            ls = u ? ls + x[u] : x[u];
        }
        // the tile's part of the sums, relative to the largest score so far
        const float m_new = fmaxf(m, mx), alpha = m == -INFINITY ? 0.f : ex2(m - m_new);
        const float beta = mx == -INFINITY ? 0.f : ex2(mx - m_new);
        m = m_new;
        l = fma2(l, F2(alpha, alpha), ls * F2(beta, beta));

        // ---- O += P V, group by group
        const Scales<NG> sv[U / 2] = {{vs, t}, {vs, 4 + t}, {vs, 8 + t}, {vs, 12 + t}};
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            // weights p sv unit < 2^23: 2^23 + weight has them in its low bits. (rcp is off by an ulp, the same for the tile)
            F2 y[U];
            uint32_t big = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                y[u] = x[u] * sv[u / 2].of(u & 1, i);
                big = larger(big, y[u]);
            }
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const float ymx = fmaxf(__uint_as_float(big), kLeastUnit), unit = rcp(ymx) * (8388608.f * 255.f / 256.f);
            const float back = big ? beta * ymx * (256.f / 255.f / 8388608.f) : 0.f;  // (rows of zeros give zeros)
            const float wa = back * da, wb = back * db;
            const int4 magic = from[8 * NG];
            uint4 pa[U / 4];
            int c7[4];
#pragma unroll
            for (int kb = 0; kb < U / 4; ++kb) {
                uint32_t w[4];  // two digits of keys 32 kb + 16 (k / 2) + 4 t + 2 (k % 2) + {0, 1}
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const F2 n = fma2(y[4 * kb + k], F2(unit, unit), F2(8388608.f, 8388608.f));
                    w[k] = prmt(__float_as_uint(n.x()), __float_as_uint(n.y()), sel);
                }
                pa[kb] = make_uint4(prmt(w[0], w[1], 0x5410), prmt(w[0], w[1], 0x7632), prmt(w[2], w[3], 0x5410), prmt(w[2], w[3], 0x7632));
                mma_u8u8(c7, pa[kb], 0x07070707u, 0x07070707u, kb ? quad(c7) : magic);
            }
            // odd dims are 16 times; digit a's 7s and offset come off exactly, digit b's to below a unit of the weights
            const float a7 = __int_as_float(c7[0]), b7 = __int_as_float(c7[2]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {  // 16 bytes of the group's 32
                int c[4][4];
#pragma unroll
                for (int kb = 0; kb < U / 4; ++kb) {
                    uint32_t r[4];
                    load_transposed(r, vrow + 32 * kb * (HD / 2) + 32 * i + 16 * j);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        mma_u8u8(c[2 * k], pa[kb], even(r[k]), even(r[k + 2]), kb ? quad(c[2 * k]) : magic);
                        mma_u8u8(c[2 * k + 1], pa[kb], odd16(r[k]), odd16(r[k + 2]), kb ? quad(c[2 * k + 1]) : magic);
                    }
                }
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float ua = n & 1 ? wa * 0.0625f : wa, ub = n & 1 ? wb * 0.0625f : wb;
                    const float ma = n & 1 ? fmaf(a7, -16.f, 15.f * 12582912.f) : -a7, mb = n & 1 ? fmaf(b7, -16.f, 15.f * 12582912.f) : -b7;
                    const F2 na = float_bits(c[n][0], c[n][1]) + F2(ma, ma);
                    const F2 join = fma2(o[i][4 * j + n], F2(alpha, alpha), F2(mb * ub, mb * ub));
                    o[i][4 * j + n] = fma2(na, F2(ua, ua), fma2(float_bits(c[n][2], c[n][3]), F2(ub, ub), join));
                }
            }
            // (a scale that is negative or no number has no digits)
            if (big >= kNoWeight)
#pragma unroll
                for (int n = 0; n < 8; ++n) o[i][n] = F2(NAN, NAN);
        }
    }

    __device__ __forceinline__ float sum_lanes() {  // returns the sum of the probabilities
        float lw = l.x() + l.y();
        lw += __shfl_xor_sync(0xffffffffu, lw, 1);
        lw += __shfl_xor_sync(0xffffffffu, lw, 2);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 8; ++n)
                o[i][n] = o[i][n] + F2(__shfl_xor_sync(0xffffffffu, o[i][n].x(), 16), __shfl_xor_sync(0xffffffffu, o[i][n].y(), 16));
        return lw;
    }
    __device__ __forceinline__ void put(float* row) const {
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 8; n += 2)
                *reinterpret_cast<float4*>(row + 64 * i + 8 * n + 4 * t) = make_float4(o[i][n].x(), o[i][n + 1].x(), o[i][n].y(), o[i][n + 1].y());
    }
    __device__ __forceinline__ void add(float* row, float f, float fo) const {  // fo row + f o
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 8; n += 2) {
                float4* at = reinterpret_cast<float4*>(row + 64 * i + 8 * n + 4 * t);
                float4 v = *at;
                v.x = fmaf(o[i][n].x(), f, v.x * fo); v.y = fmaf(o[i][n + 1].x(), f, v.y * fo);
                v.z = fmaf(o[i][n].y(), f, v.z * fo); v.w = fmaf(o[i][n + 1].y(), f, v.w * fo);
                *at = v;
            }
    }
};

// ---- one or two query heads: keys (of S) and dims (of O) in the rows of A,
// digits in the columns of B (columns 4 h + 0, 1, 2: digits 2, 1, 0 of head h)
template <int HD>
struct Few {
    static constexpr int kHeads = kHeadsFew, kCtas = kCtasFew, NG = HD / FORGE_KV4_GROUP, kBlocks = kKeys / 16;
    static constexpr int kRowY = kKeys + 8;                              // words of a (head, group)'s weights, no bank twice
    static constexpr int kY = kHeads * NG * kRowY * 4;                   // a warp's weights
    static constexpr int kSmem = NG * 64 + 16 + 64 + kWarps * kY;        // sums to start from [groups][t], kMagic, factors [t], weights
    const int warp, lane, g, t, h, hq;
    const float da, db;       // this lane's columns 2 t, 2 t + 1: digits 2 and 1 of head h, or digit 0 and nothing
    const uint32_t sel;       // the digit of column g, of two words
    int4* from;
    uint32_t* ys;
    uint2 qb[NG][2];
    float fac, m;
    F2 l, o[NG][4];  // o[group][2 k + b]: dims 64 i + 32 k + 2 g + b and + 16, this lane's digits' part

    __device__ Few(uint8_t* smem, int warp, int lane)
        : warp(warp), lane(lane), g(lane >> 2), t(lane & 3), h(t >> 1), hq(g >> 2), da(t & 1 ? 1.f : 65536.f),
          db(t & 1 ? 0.f : 256.f),
          sel((g & 3) == 0 ? 0x62 : (g & 3) == 1 ? 0x51 : (g & 3) == 2 ? 0x40 : 0xFB), from(reinterpret_cast<int4*>(smem)),
          ys(reinterpret_cast<uint32_t*>(smem + NG * 64 + 16 + 64 + warp * kY)) {
        if (threadIdx.x == 0) from[4 * NG] = make_int4(kMagic, kMagic, kMagic, kMagic);
    }
    __device__ int q_head() const { return hq; }
    __device__ bool holds() const { return !(t & 1); }
    __device__ bool first() const { return g == 0 && !(t & 1); }

    // q (dims 64 i + 16 t .. + 15 of head g / 4) as B operands, dims 64 i + 16 t + 8 w + {0, 2, 4, 6} and {1, 3, 5, 7}, and
    // the sums that the scores start from
    __device__ __forceinline__ void stage(const float4 (&v)[NG][4], float scale_log2) {
        uint32_t mx = 0;  // largest |q| as bits
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mx = max(max(mx, __float_as_uint(fabsf(v[i][j].x))), __float_as_uint(fabsf(v[i][j].y)));
                mx = max(max(mx, __float_as_uint(fabsf(v[i][j].z))), __float_as_uint(fabsf(v[i][j].w)));
            }
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // 2^e > 1.004 |q|: |q| 2^(23 - e) is at most 127 (1 + 2^8 + 2^16), the largest three signed digits
        const int e = (int)(__float_as_uint(1.004f * __uint_as_float(mx)) >> 23) - 126, sd = sum_down(e);
        const float up = pow2i(min(23 - e, 127)), up2 = pow2i(max(23 - e, 127) - 127);  // (for the smallest q, two factors)
        const float down = pow2i(-__shfl_sync(0xffffffffu, sd, 16 * h));
        if (warp == 0 && g == 0) from[4 * NG + 1 + t] = factors(da * down, db * down);
        fac = mx >= 0x7F800000u ? NAN : scale_log2 * pow2i(e - 23 + sd);  // (an infinite or NaN q: all NaN)
        fac = __shfl_sync(0xffffffffu, fac, 16 * h);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            int sum = 0;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const float4 lo4 = v[i][2 * w], hi4 = v[i][2 * w + 1];
                const float x[8] = {lo4.x, lo4.z, hi4.x, hi4.z, lo4.y, lo4.w, hi4.y, hi4.w};  // even dims, odd dims
                uint32_t d[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int n = __float2int_rn(x[k] * up * up2), d0 = (int)(int8_t)n, n1 = (n - d0) >> 8, d1 = (int)(int8_t)n1;
                    d[k] = (g & 3) == 0 ? (n1 - d1) >> 8 : (g & 3) == 1 ? d1 : (g & 3) == 2 ? d0 : 0;
                }
                qb[i][w] = make_uint2(low_bytes(d), low_bytes(d + 4));
                sum = __dp4a((int)qb[i][w].x, 0x01010101, __dp4a((int)qb[i][w].y, 0x01010101, sum));
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int fa = kMagic - 7 * __shfl_sync(0xffffffffu, sum, 8 * t), fb = kMagic - 7 * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            if (warp == 0 && g == 0) from[4 * i + t] = make_int4(fa, fb, fa, fb);
        }
        m = -INFINITY;
        l = F2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n) o[i][n] = F2(0.f, 0.f);
    }

    __device__ __forceinline__ void tile(uint8_t* slot, int left) {
        const uint8_t *kc = slot, *ks = slot + 2 * Geo<HD>::kCodes;
        uint8_t* vs = slot + 2 * Geo<HD>::kCodes + Geo<HD>::kScales;
        const uint8_t *krow = kc + g * (HD / 2) + 8 * t, *vrow = kc + Geo<HD>::kCodes + lane * (HD / 2);
        const int4 magic = from[4 * NG];
        const bool one = has_one<HD>(vs, lane);
        const int4 fs = from[4 * NG + 1 + t];
        const float sa = __int_as_float(fs.x), sb = __int_as_float(fs.y), off = __int_as_float(fs.z);
        // ---- scores of keys 16 b + g and + 8, head h, over fac
        F2 x[kBlocks];
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const uint32_t s0 = scale_word<NG>(ks, 16 * b + g), s1 = scale_word<NG>(ks, 16 * b + 8 + g);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint2 w = *reinterpret_cast<const uint2*>(krow + 16 * b * (HD / 2) + 32 * i);
                const uint2 z = *reinterpret_cast<const uint2*>(krow + (16 * b + 8) * (HD / 2) + 32 * i);
                int c[4];
                mma_u8s8(c, make_uint4(even(w.x), even(z.x), even(w.x >> 4), even(z.x >> 4)), qb[i][0].x, qb[i][0].y, from[4 * i + t]);
                mma_u8s8(c, make_uint4(even(w.y), even(z.y), even(w.y >> 4), even(z.y >> 4)), qb[i][1].x, qb[i][1].y, quad(c));
                // digits times sa and sb; both offsets of 12582912 come off exactly with the first
                const F2 sum = fma2(float_bits(c[1], c[3]), F2(sb, sb), fma2(float_bits(c[0], c[2]), F2(sa, sa), F2(off, off)));
                const F2 sp = i ? F2(bf16_hi_f32(s0), bf16_hi_f32(s1)) : F2(bf16_lo_f32(s0), bf16_lo_f32(s1));
                x[b] = i ? fma2(sum, sp, x[b]) : sum * sp;
            }
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)  // the other digits
            x[b] = x[b] + F2(__shfl_xor_sync(0xffffffffu, x[b].x(), 1), __shfl_xor_sync(0xffffffffu, x[b].y(), 1));
        // ---- the tile's largest score; keys behind the last one count for nothing
        if (left < kKeys) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                x[b] = F2(16 * b + g < left ? x[b].x() : -INFINITY, 16 * b + 8 + g < left ? x[b].y() : -INFINITY);
            clear_scales<HD>(vs, left, lane);
        }
        drop_zeros<HD>(one, vs, kc + Geo<HD>::kCodes, lane);
        float mx = fmaxf(x[0].x(), x[0].y());
#pragma unroll
        for (int b = 1; b < kBlocks; ++b) mx = max3(mx, x[b].x(), x[b].y());
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float top = mx;
        mx = __fmul_ru(mx, fac);  // (up, so that no difference to it comes out above 0)
        // p = 2^(x - mx) <= 1
        float nmx = mx == -INFINITY ? 0.f : -mx;
        if (fabsf(mx) > kFar && fabsf(mx) < INFINITY) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) x[b] = x[b] + F2(-top, -top);
            nmx = 0.f;
        }
        F2 ls;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) {
            const F2 y = fma2(x[b], F2(fac, fac), F2(nmx, nmx));
            x[b] = F2(ex2(y.x()), ex2(y.y()));
            ls = b ? ls + x[b] : x[b];
        }
        // the tile's part of the sums, relative to the largest score so far
        const float m_new = fmaxf(m, mx), alpha = m == -INFINITY ? 0.f : ex2(m - m_new);
        const float beta = mx == -INFINITY ? 0.f : ex2(mx - m_new);
        m = m_new;
        l = fma2(l, F2(alpha, alpha), ls * F2(beta, beta));

        // ---- weights p sv unit < 2^23, added to 2^23, of head h: lane t of the two for group t % 2 (both the same where there
        // is one); through shared memory to the lanes whose column needs their keys
        uint32_t mine = 0;  // the largest of this lane's group
        {
            const int i = NG == 2 ? t & 1 : 0;
            const uint16_t* sv = reinterpret_cast<const uint16_t*>(vs) + g * NG + i;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                x[b] = x[b] * F2(bf16_bits_to_f32(sv[16 * b * NG]), bf16_bits_to_f32(sv[(16 * b + 8) * NG]));
                mine = larger(mine, x[b]);
            }
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 4));
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 8));
            mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, 16));
            const float unit = rcp(fmaxf(__uint_as_float(mine), kLeastUnit)) * (8388608.f * 255.f / 256.f);  // (off by an ulp, the same for the tile)
            uint32_t* y = ys + (h * NG + i) * kRowY + g;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const F2 n = fma2(x[b], F2(unit, unit), F2(8388608.f, 8388608.f));
                y[16 * b] = __float_as_uint(n.x());
                y[16 * b + 8] = __float_as_uint(n.y());
            }
        }
        __syncwarp();

        // ---- O += P V, group by group
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const uint32_t big = __shfl_sync(0xffffffffu, mine, (lane & ~1) | i);
            const float back = big ? beta * fmaxf(__uint_as_float(big), kLeastUnit) * (256.f / 255.f / 8388608.f) : 0.f;  // (rows of zeros give zeros)
            const float wa = back * da, wb = back * db;
            uint2 pb[kKeys / 32];
            int c7[4];
#pragma unroll
            for (int kb = 0; kb < kKeys / 32; ++kb) {
                const uint32_t* y = ys + (hq * NG + i) * kRowY + 32 * kb + 4 * t;
                const uint4 ya = *reinterpret_cast<const uint4*>(y), yb = *reinterpret_cast<const uint4*>(y + 16);
                pb[kb].x = prmt(prmt(ya.x, ya.y, sel), prmt(ya.z, ya.w, sel), 0x5410);
                pb[kb].y = prmt(prmt(yb.x, yb.y, sel), prmt(yb.z, yb.w, sel), 0x5410);
                mma_u8u8(c7, make_uint4(0x07070707u, 0x07070707u, 0x07070707u, 0x07070707u), pb[kb].x, pb[kb].y, kb ? quad(c7) : magic);
            }
            const float a7 = __int_as_float(c7[0]), b7 = __int_as_float(c7[1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {  // 16 bytes of the group's 32
                int c[2][4];               // even dims; odd ones, times 16
#pragma unroll
                for (int kb = 0; kb < kKeys / 32; ++kb) {
                    uint32_t r[4];
                    load_transposed(r, vrow + 32 * kb * (HD / 2) + 32 * i + 16 * j);
                    mma_u8u8(c[0], make_uint4(even(r[0]), even(r[1]), even(r[2]), even(r[3])), pb[kb].x, pb[kb].y, kb ? quad(c[0]) : magic);
                    mma_u8u8(c[1], make_uint4(odd16(r[0]), odd16(r[1]), odd16(r[2]), odd16(r[3])), pb[kb].x, pb[kb].y, kb ? quad(c[1]) : magic);
                }
#pragma unroll
                for (int n = 0; n < 2; ++n) {  // the 7s and offsets come off exactly
                    const float ua = n ? wa * 0.0625f : wa, ub = n ? wb * 0.0625f : wb;
                    const float ma = n ? fmaf(a7, -16.f, 15.f * 12582912.f) : -a7, mb = n ? fmaf(b7, -16.f, 15.f * 12582912.f) : -b7;
                    const F2 na = float_bits(c[n][0], c[n][2]) + F2(ma, ma), nb = float_bits(c[n][1], c[n][3]) + F2(mb, mb);
                    F2& at = o[i][2 * j + n];
                    at = fma2(na, F2(ua, ua), fma2(nb, F2(ub, ub), at * F2(alpha, alpha)));
                }
            }
            // (a scale that is negative or no number has no digits)
            if (big >= kNoWeight)
#pragma unroll
                for (int n = 0; n < 4; ++n) o[i][n] = F2(NAN, NAN);
        }
    }

    __device__ __forceinline__ float sum_lanes() {
        float lw = l.x() + l.y();
        lw += __shfl_xor_sync(0xffffffffu, lw, 4);
        lw += __shfl_xor_sync(0xffffffffu, lw, 8);
        lw += __shfl_xor_sync(0xffffffffu, lw, 16);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int n = 0; n < 4; ++n)
                o[i][n] = o[i][n] + F2(__shfl_xor_sync(0xffffffffu, o[i][n].x(), 1), __shfl_xor_sync(0xffffffffu, o[i][n].y(), 1));
        return lw;
    }
    __device__ __forceinline__ void put(float* row) const {
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float2* at = reinterpret_cast<float2*>(row + 64 * i + 32 * k + 2 * g);
                at[0] = make_float2(o[i][2 * k].x(), o[i][2 * k + 1].x());
                at[8] = make_float2(o[i][2 * k].y(), o[i][2 * k + 1].y());
            }
    }
    __device__ __forceinline__ void add(float* row, float f, float fo) const {
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float2* at = reinterpret_cast<float2*>(row + 64 * i + 32 * k + 2 * g);
                const float2 a = at[0], b = at[8];
                at[0] = make_float2(fmaf(o[i][2 * k].x(), f, a.x * fo), fmaf(o[i][2 * k + 1].x(), f, a.y * fo));
                at[8] = make_float2(fmaf(o[i][2 * k].y(), f, b.x * fo), fmaf(o[i][2 * k + 1].y(), f, b.y * fo));
            }
    }
};

template <int HD, typename Form>
struct Layout : Geo<HD> {  // of shared memory
    static constexpr int kRow = HD + 4;                                             // floats of a head in the join (no bank twice)
    static constexpr int kOffForm = kWarps * kStages * Geo<HD>::kSlot;              // the form's
    static constexpr int kOffRed = kOffForm + Form::kSmem;                          // [warp][heads][kRow] sums of warps
    static constexpr int kOffMl = kOffRed + kJoin * Form::kHeads * kRow * 4;        // [warp][heads] m, then l
    static constexpr int kOffBar = kOffMl + 2 * kJoin * Form::kHeads * 4;
    static constexpr int kSmem = kOffBar + kWarps * kStages * 8;
};

template <int HD, template <int> class Form>
__global__ void __launch_bounds__(kThreads, Form<HD>::kCtas) k_kv4_decode(const Kv4Args a) {
    using X = Layout<HD, Form<HD>>;
    constexpr int NG = X::kNG, kHeads = Form<HD>::kHeads;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = lane & 3;
    uint8_t* ring = smem + warp * kStages * X::kSlot;
    float* red = reinterpret_cast<float*>(smem + X::kOffRed);
    float* sm_m = reinterpret_cast<float*>(smem + X::kOffMl);
    float* sm_l = sm_m + kJoin * kHeads;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + X::kOffBar) + warp * kStages;
    __shared__ int s_last;
    Form<HD> f(smem + X::kOffForm, warp, lane);

    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&full[s], 1);
        fence_mbar_init();
    }
    __syncwarp();  // (before the lane that issues the first copies arrives on them)

    // ---- the line's length; sequences without tiles are answered here
    const int n0 = lane < a.B ? tiles_of(a, lane) : 0;
    int total = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        const int b = b0 + lane;
        const int n = b0 == 0 ? n0 : b < a.B ? tiles_of(a, b) : 0;
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
        total += __reduce_add_sync(0xffffffffu, n > 0 ? n + kPairUnits : 0);
    }
    total *= a.ph;
    const int per = max(kMinUnits, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int start = (int)blockIdx.x * per, end = min(total, start + per);
    if (start >= end) return;

    // ---- the pair in which this CTA's range starts
    Place at{0, 0, 0, 0};
    for (int b0 = 0;; b0 += 32) {  // at.base: first unit of slot b0
        const int b = b0 + lane;
        const int n = max(0, b0 == 0 ? n0 : b < a.B ? tiles_of(a, b) : 0), un = n ? n + kPairUnits : 0;
        int inc = un;
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += u;
        }
        const unsigned past = __ballot_sync(0xffffffffu, at.base + inc * a.ph > start);
        if (past) {
            const int w = __ffs(past) - 1;
            at.n = __shfl_sync(0xffffffffu, n, w);
            const int units = at.n + kPairUnits;
            at.base += (__shfl_sync(0xffffffffu, inc, w) - units) * a.ph;
            at.b = b0 + w;
            at.pair = (start - at.base) / units;
            at.base += at.pair * units;
            break;
        }
        at.base += __shfl_sync(0xffffffffu, inc, 31) * a.ph;
    }

    // ---- copies of this warp's tiles: lane 4 i + k copies array k (K codes, V codes, K scales, V scales) of the
    // tile's i-th page
    const int arr = lane & 3;
    const int unit = arr < 2 ? HD / 2 : NG * 2;  // bytes a row
    const int slot_off = arr == 0 ? 0 : arr == 1 ? X::kCodes : 2 * X::kCodes + (arr - 2) * X::kScales;
    const uint8_t* array = arr == 0 ? a.c.k : arr == 1 ? a.c.v : (const uint8_t*)(arr == 2 ? a.c.ks : a.c.vs);
    Place in = at;
    int in_j = in.mine(in.lo(start), warp), n_in = 0;
    uint32_t poison = 0;      // slots whose tile names a page outside the pool
    int in_rows = 0;          // rows of the pair's sequence, in eights
    int64_t in_row0 = 0;      // contiguous: its first row in the arrays; paged: KV head
    const int32_t* in_table = nullptr;
    bool entered = false;
    auto issue = [&]() {
        while (in_j >= in.hi(end)) {
            if (in.base >= end) return;
            in.next(a);
            in_j = in.mine(0, warp);
            entered = false;
        }
        if (!entered) {
            const int sq = a.seq ? a.seq[in.b] : in.b, kvh = in.pair / a.nhb;
            in_rows = (a.pos[in.b] + 8) & ~7;
            in_row0 = a.c.table ? kvh : ((int64_t)sq * a.c.n_kv_head + kvh) * a.c.lmax;
            in_table = a.c.table ? a.c.table + (int64_t)sq * a.c.max_pages : nullptr;
            entered = true;
        }
        const int s = n_in % kStages, key0 = in_j * kKeys;
        const int rows = min(kKeys, in_rows - key0);
        uint8_t* slot = ring + s * X::kSlot;
        if (!in_table) {
            // (one thread and no loop: addresses in uniform registers, which a copy wants, four times cheaper than by lane)
            if (elect_one()) {
                const int64_t row = in_row0 + key0;
                const uint64_t once = l2_evict_first();
                mbar_arrive_expect_tx(&full[s], rows * (HD + 4 * NG));
                bulk_g2s_stream(slot, a.c.k + row * (HD / 2), rows * (HD / 2), &full[s], once);
                bulk_g2s_stream(slot + X::kCodes, a.c.v + row * (HD / 2), rows * (HD / 2), &full[s], once);
                bulk_g2s_stream(slot + 2 * X::kCodes, a.c.ks + row * NG, rows * (NG * 2), &full[s], once);
                bulk_g2s_stream(slot + 2 * X::kCodes + X::kScales, a.c.vs + row * NG, rows * (NG * 2), &full[s], once);
            }
        } else {
            if (lane == 0) mbar_arrive_expect_tx(&full[s], rows * (HD + 4 * NG));
            __syncwarp();
            uint8_t* dst = slot + slot_off;
            const int pt = a.c.page_tokens, pg0 = key0 / pt + (lane >> 2);
            const int r0 = max(0, pg0 * pt - key0), r1 = min(rows, (pg0 + 1) * pt - key0);
            bool bad = false;
            if (r0 < r1) {
                int pg = in_table[pg0];
                bad = (unsigned)pg >= (unsigned)a.c.num_pages;
                if (bad) {
                    atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
                    pg = 0;
                }
                const int64_t row = ((int64_t)pg * a.c.n_kv_head + in_row0) * pt + (key0 + r0 - pg0 * pt);
                bulk_g2s_stream(dst + r0 * unit, array + row * unit, (r1 - r0) * unit, &full[s], l2_evict_first());
            }
            poison &= ~(1u << s);
            if (__any_sync(0xffffffffu, bad)) poison |= 1u << s;
        }
        in_j += kWarps;
        ++n_in;
    };
    // q of a pair (dims 64 i + 16 t .. + 15 of the form's head), loaded before what it can be loaded before
    float4 v[NG][4];
    auto load_q = [&](const Place& p) {
        const int h0 = (p.pair % a.nhb) * kHeads;
        const float* q = a.q + ((size_t)p.b * a.H + p.pair / a.nhb * a.G + h0 + f.q_head()) * HD + 16 * t;
        const bool mine = p.lo(start) < p.hi(end) && f.q_head() < a.G - h0;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[i][j] = mine ? *reinterpret_cast<const float4*>(q + 64 * i + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    load_q(at);
    for (int s = 0; s < kStages; ++s) issue();

    int n_out = 0;
    bool dead = false;  // a wait ran out: nothing more is read
    for (Place following = at; at.base < end; at = following) {
        // ---- one pair: tiles [j0, j1)
        const int j0 = at.lo(start), j1 = at.hi(end);
        if (j0 >= j1) break;  // (the range ends before the pair's first tile)
        const int kvh = at.pair / a.nhb, h0 = (at.pair % a.nhb) * kHeads, nh = min(kHeads, a.G - h0);
        const size_t qrow = (size_t)at.b * a.H + kvh * a.G + h0;

        f.stage(v, a.scale_log2);
        __syncthreads();
#pragma unroll 1
        for (int j = at.mine(j0, warp); j < j1; j += kWarps) {
            if (dead) break;
            const int s = n_out % kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(&full[s], (n_out / kStages) & 1, a.err))) {
                dead = true;  // the copies in flight get the same time again to land before the CTA exits
                ring_drain<kStages>(n_out, n_in, [&](int slot, int parity) { mbar_wait(&full[slot], parity, a.err); });
                break;
            }
            const int left = j + 1 < at.n ? kKeys : a.pos[at.b] + 1 - j * kKeys;  // keys of the tile

            f.tile(ring + s * X::kSlot, left);
            if (poison >> s & 1) f.l = F2(NAN, NAN);
            ++n_out;
            __syncwarp();
            issue();
        }
        if (dead) f.l = F2(NAN, NAN);
        following.next(a);
        load_q(following);

        // ---- join the warps: the upper half's sums into the lower half's, then those over the CTA
        const float lw = f.sum_lanes();
        const int slot = warp % kJoin * kHeads + f.h;
        float* mine = red + slot * X::kRow;
        const bool holds = f.holds() && f.h < nh;
        if (warp >= kJoin && holds) {
            f.put(mine);
            if (f.first()) {
                sm_m[slot] = f.m;
                sm_l[slot] = lw;
            }
        }
        __syncthreads();
        const float mo = sm_m[slot], lo = sm_l[slot];
        __syncwarp();
        if (warp < kJoin && holds) {
            const float mj = fmaxf(f.m, mo);
            const float fm = f.m == -INFINITY ? 0.f : ex2(f.m - mj), fo = mo == -INFINITY ? 0.f : ex2(mo - mj);
            if (f.first()) {
                sm_m[slot] = mj;
                sm_l[slot] = isnan(lo) || isnan(lw) ? NAN : fmaf(lw, fm, lo * fo);
            }
            f.add(mine, fm, fo);
        }
        __syncthreads();
        const int unit0 = at.base + kPairUnits, cfirst = unit0 / per, clast = (unit0 + at.n - 1) / per;
        float* part = a.partial + ((size_t)blockIdx.x * 2 + ((int)blockIdx.x == cfirst)) * kHeads * (HD + 2);
        for (int idx = threadIdx.x; idx < nh * (HD / 4); idx += kThreads) {
            const int h = idx / (HD / 4), d = idx % (HD / 4) * 4;
            float mj = -INFINITY, lj = 0.f;
#pragma unroll
            for (int w = 0; w < kJoin; ++w) mj = fmaxf(mj, sm_m[w * kHeads + h]);
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kJoin; ++w) {
                const float mw = sm_m[w * kHeads + h], lv = sm_l[w * kHeads + h];
                const float fw = mw == -INFINITY ? 0.f : ex2(mw - mj);
                lj = isnan(lv) ? lv : fmaf(lv, fw, lj);
                const float4 r = *reinterpret_cast<const float4*>(red + (w * kHeads + h) * X::kRow + d);
                v.x = fmaf(r.x, fw, v.x); v.y = fmaf(r.y, fw, v.y); v.z = fmaf(r.z, fw, v.z); v.w = fmaf(r.w, fw, v.w);
            }
            const float il = 1.f / lj;
            v.x *= il; v.y *= il; v.z *= il; v.w *= il;
            if (cfirst == clast) {
                *reinterpret_cast<float4*>(a.out + (qrow + h) * HD + d) = v;
            } else {
                float2* dst = reinterpret_cast<float2*>(part + h * (HD + 2) + d);
                dst[0] = make_float2(v.x, v.y);
                dst[1] = make_float2(v.z, v.w);
                if (d == 0) {
                    part[h * (HD + 2) + HD] = mj;
                    part[h * (HD + 2) + HD + 1] = lj;
                }
            }
        }
        if (cfirst == clast) continue;
        // ---- the last of the pair's CTAs joins them: the block barrier orders the partial's stores before thread 0's
        // release
        __syncthreads();
        if (threadIdx.x == 0) {
            uint32_t old;
            const uint32_t top = clast - cfirst;  // the counter returns to 0 after the last
            asm volatile("fence.acq_rel.gpu;" ::: "memory");
            asm volatile("atom.inc.acq_rel.gpu.global.u32 %0, [%1], %2;"
                         : "=r"(old) : "l"(a.counters + (size_t)at.b * a.ph + at.pair), "r"(top) : "memory");
            s_last = old == top;
        }
        __syncthreads();
        if (!s_last) continue;
        const int nc = clast - cfirst + 1;
        for (int hh = warp; hh < nh; hh += kWarps) {
            // contribution c: the pair starts in the first CTA's range and before every other's
            auto slot = [&](int c) {
                return a.partial + ((size_t)(cfirst + c) * 2 + (c == 0)) * kHeads * (HD + 2) + hh * (HD + 2);
            };
            constexpr int E = HD / 32;
            float2 p[8][E / 2];
            auto fetch = [&](int c) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int e = 0; e < E / 2; ++e)
                        if (c + k < nc) p[k][e] = __ldcg(reinterpret_cast<const float2*>(slot(c + k)) + 32 * e + lane);
            };
            fetch(0);
            float mm = -INFINITY;
            for (int c = lane; c < nc; c += 32) mm = fmaxf(mm, __ldcg(slot(c) + HD));
            for (int d = 16; d; d >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
            float acc[E] = {}, sum = 0.f, wl = 0.f;
            for (int c = 0; c < nc; c += 8) {
                if (c % 32 == 0 && c + lane < nc) {
                    const float mc = __ldcg(slot(c + lane) + HD), lc = __ldcg(slot(c + lane) + HD + 1);
                    wl = mc == -INFINITY && !isnan(lc) ? 0.f : lc * ex2(mc - mm);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float w = __shfl_sync(0xffffffffu, wl, (c + k) & 31);
                    if (c + k < nc) {
                        sum += w;
#pragma unroll
                        for (int e = 0; e < E / 2; ++e) {
                            acc[2 * e] = w == 0.f ? acc[2 * e] : fmaf(w, p[k][e].x, acc[2 * e]);
                            acc[2 * e + 1] = w == 0.f ? acc[2 * e + 1] : fmaf(w, p[k][e].y, acc[2 * e + 1]);
                        }
                    }
                }
                fetch(c + 8);
            }
#pragma unroll
            for (int e = 0; e < E / 2; ++e)
                reinterpret_cast<float2*>(a.out + (qrow + hh) * HD)[32 * e + lane] = make_float2(acc[2 * e] / sum, acc[2 * e + 1] / sum);
        }
    }
}

int configure() {
    static bool done[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return forge_fail(-1, "forge_flash_decode_kv4: no device");
    if (done[dev]) return 0;
    cudaError_t e = cudaSuccess;
    auto set = [&](auto kernel, int smem) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    };
    set(k_kv4_decode<64, Few>, Layout<64, Few<64>>::kSmem);
    set(k_kv4_decode<128, Few>, Layout<128, Few<128>>::kSmem);
    set(k_kv4_decode<64, Many>, Layout<64, Many<64>>::kSmem);
    set(k_kv4_decode<128, Many>, Layout<128, Many<128>>::kSmem);
    if (e != cudaSuccess) return forge_fail(-1, "forge_flash_decode_kv4: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
    return 0;
}

// Passes over a KV head's keys for the G query heads that read it.
int heads_of_a_pass(int G) { return G <= kHeadsFew ? kHeadsFew : kHeadsMany; }
int passes(int G) { return (G + heads_of_a_pass(G) - 1) / heads_of_a_pass(G); }

// A B200's CTAs; fixed so that workspace sizes do not depend on the device.
int most_ctas(int G) { return 148 * (heads_of_a_pass(G) == kHeadsFew ? kCtasFew : kCtasMany); }
// The partials, at the workspace's start; the counters behind them lie in the same place for every batch, so that one
// call's partials never become another's counters.
int64_t partial_bytes(int G, int hd) { return (int64_t)most_ctas(G) * 2 * heads_of_a_pass(G) * (hd + 2) * 4; }
}  // namespace
extern "C" FORGE_API int64_t forge_flash_decode_kv4_workspace_bytes(int B, int H, int n_kv_head, int head_dim) {
    if (B <= 0 || H <= 0 || n_kv_head <= 0 || H % n_kv_head || (head_dim != 64 && head_dim != 128)) return -1;
    const int64_t pairs = (int64_t)B * n_kv_head * passes(H / n_kv_head);
    return partial_bytes(H / n_kv_head, head_dim) + (pairs * 4 + 255) / 256 * 256;
}

extern "C" FORGE_API int forge_flash_decode_kv4(const float* q, const ForgeKv4* cache, const int32_t* seq,
                                                const int32_t* pos, int B, int H, float* out, void* workspace,
                                                void* stream) {
    if (int rc = forge_kv4_check(cache, "forge_flash_decode_kv4")) return rc;
    if (!q || !pos || !out || !workspace || B <= 0 || B > 65535 || H <= 0 || H % cache->n_kv_head ||
        (!seq && B > cache->n_seq) || (((uintptr_t)q | (uintptr_t)out | (uintptr_t)workspace) & 15))
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_decode_kv4: bad args (arrays 16-byte aligned, H a multiple of the KV heads)");
    const int hd = cache->head_dim, cap = cache->table ? cache->max_pages * cache->page_tokens : cache->lmax;
    const int64_t units = (int64_t)B * cache->n_kv_head * passes(H / cache->n_kv_head) * ((cap + kKeys - 1) / kKeys + kPairUnits);
    if (units > (1ll << 30))
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_decode_kv4: B x KV heads x rows of a sequence is too large (%lld tiles of 64 keys)", (long long)units);
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_flash_decode_kv4: no device");
    if (configure()) return -1;
    Kv4Args a{};
    a.c = *cache; a.q = q; a.seq = seq; a.pos = pos; a.B = B; a.H = H;
    a.G = H / cache->n_kv_head;
    a.nhb = passes(a.G);
    a.ph = cache->n_kv_head * a.nhb;
    a.cap = cap;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)hd));
    a.out = out; a.err = err;
    a.partial = (float*)workspace;
    a.counters = (uint32_t*)((char*)workspace + partial_bytes(a.G, hd));
    // no more CTAs than the longest sequences could feed
    const int64_t most = (units + kMinUnits - 1) / kMinUnits;
    const int grid = (int)std::min<int64_t>(most, most_ctas(a.G));
    auto go = [&](auto kernel, int smem) { kernel<<<grid, kThreads, smem, (cudaStream_t)stream>>>(a); };
    if (heads_of_a_pass(a.G) == kHeadsFew) {
        if (hd == 128) go(k_kv4_decode<128, Few>, Layout<128, Few<128>>::kSmem);
        else go(k_kv4_decode<64, Few>, Layout<64, Few<64>>::kSmem);
    } else {
        if (hd == 128) go(k_kv4_decode<128, Many>, Layout<128, Many<128>>::kSmem);
        else go(k_kv4_decode<64, Many>, Layout<64, Many<64>>::kSmem);
    }
    return forge_check_launch("forge_flash_decode_kv4");
}
