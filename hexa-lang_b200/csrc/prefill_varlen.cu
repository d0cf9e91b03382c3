// prefill_varlen.cu — causal attention of packed prompts (grouped heads,
// sequences of any length back to back) on the tcgen05 tensor cores, bf16 in
// and out, fp32 sums.
//
// O[i] = sum_j softmax_j(q_i . k_j / sqrt(hd)) v_j over j <= i of i's
// sequence, LSE[i] = log sum_j exp(q_i . k_j / sqrt(hd)).
//
// A work item is two tiles of 128 query rows that share every K/V block: two
// query heads of one KV head where the group is even (the tiles then have the
// same blocks, and a short prompt fills both), else two consecutive tiles of
// one head. CTAs are persistent, one per SM. Items are dealt out longest
// first: for every depth (position of the tile in its sequence) from the
// deepest, its items raise the CTAs' loads to a common level.
// Heads are dealt a group at a time, as many as keep their K and V in half of
// L2 (for 8 prompts of 4096 with 32 KV heads all heads at once read HBM 2.6
// times and took 1.12 ms instead of 1.01). Every CTA works this out for
// itself, in a warp of its own that runs ahead of the others, so that any mix
// of lengths is even without a table, a counter or a second launch (dealing
// the sorted items out back and forth instead took up to 1.4 times as long).
//
//   warps 0-3 / 4-7    softmax of tile A / B, one thread per query row
//   warp 8             TMA: Q of both tiles, K and V through a 5-slot ring
//   warp 9 (one lane)  tensor-core issue, tiles alternating
//   warp 10            items
//
// Keys are taken 64 at a time (half a block): S = Q K^T (128 x 64 x hd) goes to
// one of two TMEM buffers of its tile; its thread takes the row into
// registers and writes P = 2^(S c - m) over it as bf16 pairs, the A operand of
// O += P V. With two buffers the tensor cores run S of the next half block
// while the exponentials of this one run: a tile's softmax never waits for
// its own products (with blocks of 128 keys TMEM has room for one buffer, and
// softmax, P V and the next S of a tile came one after the other). P is rounded
// to bf16 since V is bf16 and a product's operands have one type: 1.1e-3 rms of O
// beside the 1.5e-3 of O's own rounding to bf16 (P as two bf16 terms would double
// the products of P V). Its sum is taken of the fp32 values. m is raised
// only when a score exceeds it by more than 2^8, so O in TMEM is rarely
// rescaled.
//
// What bounds it: 8 prompts of 4096 with 32 heads take 1.01 ms in a burst
// (1.1 PFLOP/s) and 1.13 under the power cap; the tensor cores' operands from
// shared memory take as long as the products (1280 of about 1660 cycles for 64
// keys of both tiles). 16 ragged prompts up to 4096, 32 heads on 8: 228-231 us
// (0.93 PFLOP/s, clock 1.67 GHz). Short prompts: the longest item's steps.
//
// A sequence may end inside a key block. Keys behind it are masked by the
// causal mask already; their V rows are zeroed in shared memory before the
// product (0 times what the next sequence holds there might be NaN). Rows
// behind the end are computed and not stored.
// Every wait is bounded (error word, then the CTA drains its copies and
// tensor-core work and frees its TMEM).
#include <cmath>
#include "tcgen05.cuh"
#include "f32x2.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"

namespace {
constexpr int kBM = 128;       // query rows per tile, keys per block
constexpr int kHalf = kBM * 64 * 2;  // 16 KB: 64 columns x 128 rows, swizzled
constexpr int kSub = 64;       // keys per softmax step
constexpr int kSoftWarps = 8, kTmaWarp = 8, kMmaWarp = 9, kItemWarp = 10;
constexpr int kThreads = 352;
constexpr int kMaxCtas = 160;  // (5 loads per lane of the items warp)
constexpr int kItemCost = 1;   // what an item costs beside its key blocks, in blocks
constexpr int kSlots = 5;      // K/V ring
// Where a row's maximum score times c = log2(e) / sqrt(hd) is beyond kFar, its rounding is a step of 64 and more, and the
// largest P would be anything. Two scores that differ do so by 2^9 there, and the smaller has no weight, with c or with
// the power of two next to it, whose product with the maximum is exact.
constexpr float kFar = 0x1p30f, kFarScale = 0.125f;
constexpr int kMostOverlap = 4;  // how often the sequences may name a row, on average
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kIdescS = umma_idesc_bf16_f32(kBM, kSub, false);
template <int HD> constexpr int tile_bytes() { return kBM * HD * 2; }
template <int HD> constexpr int off_bar() { return (2 + kSlots) * tile_bytes<HD>(); }
template <int HD> constexpr int smem_bytes() { return off_bar<HD>() + 512 + 1024; }

struct VarlenArgs {
    const int32_t* cu;
    int n_seq, total, H, Hkv;
    int group;            // items per tile (heads or pairs of them) whose K/V are worked on together
    int pair_heads;       // items are (tile, head pair), else (tile pair, head)
    float scale_log2;     // log2(e) / sqrt(hd)
    uint16_t* o;
    int64_t ldo;
    float* lse;
    uint32_t* err;
};

// Two tiles: rows row0 + 128 tile .. of `head`, of a sequence of `len` rows.
struct Item {
    int row0, len, kvh;
    int head[2], tile[2];  // tile -1: none; head[0] -1: no more items
};

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// 2^x on the FMA pipe, two values: x = i + f with i the nearest integer (the
// sum with 1.5 2^23 holds it in its low bits), a polynomial of degree 5 in f
// in [-1/2, 1/2] (minimax fit with p(0) = 1, relative error 1.7e-7 in fp32, as
// the hardware's: the sum and the LSE are fp32; degree 4 is off by 2.9e-6), i
// added to the exponent. Below -127 (masked scores) exactly 0.
__device__ __forceinline__ F2 exp2_fma(F2 x) {
    const F2 c(fmaxf(x.x(), -127.f), fmaxf(x.y(), -127.f)), magic(12582912.f, 12582912.f);
    const F2 y = c + magic, i = y + F2(-12582912.f, -12582912.f), f = fma2(i, F2(-1.f, -1.f), c);
    F2 p = fma2(f, F2(0.00132647273f, 0.00132647273f), F2(0.00967151299f, 0.00967151299f));
    p = fma2(p, f, F2(0.0555073358f, 0.0555073358f));
    p = fma2(p, f, F2(0.240222424f, 0.240222424f));
    p = fma2(p, f, F2(0.693147004f, 0.693147004f));
    p = fma2(p, f, F2(1.f, 1.f));
    return F2(__int_as_float(__float_as_int(p.x()) + (__float_as_int(y.x()) << 23)),
              __int_as_float(__float_as_int(p.y()) + (__float_as_int(y.y()) << 23)));
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if any is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// This CTA's items, one after the other (a whole warp calls it).
struct Dealer {
    const VarlenArgs& a;
    int rows, heads;        // rows of an item's tiles in a sequence, items per tile
    int group, h0, hn;      // items per tile dealt together; those in hand: [h0, h0 + hn)
    int deepest, p, used;   // the deepest tile, the depth being dealt; CTAs that have an item while some have none
    int load[kMaxCtas / 32];  // of CTAs lane, lane + 32, ...
    int next, last;         // this CTA's items [next, last) of depth p

    __device__ int length(int s) const {  // of sequence s; 0 where its bounds are bad
        if (s >= a.n_seq) return 0;
        const int b = a.cu[s], e = a.cu[s + 1];
        return b < 0 || e < b || e > a.total ? 0 : e - b;
    }
    __device__ int depth(int s) const { return (length(s) + rows - 1) / rows; }  // in tiles
    __device__ explicit Dealer(const VarlenArgs& args) : a(args) {}
    __device__ void start() {
        rows = a.pair_heads ? kBM : 2 * kBM;
        heads = a.pair_heads ? a.H / 2 : a.H;
        int most = 0;
        unsigned whole = 0;  // whole tiles of 128 rows
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
            const int n = length(s0 + (threadIdx.x & 31));
            most = max(most, (n + rows - 1) / rows);
            whole = min(whole + n / kBM, 1u << 26);  // (no overflow of the warp's sum)
        }
        deepest = (int)__reduce_max_sync(0xffffffffu, most);
        // Bounds that decrease can name the rows many times over, more work than any packing of them: nothing is done.
        // (Of sequences that do not overlap, the whole tiles are at most total / 128, which is below 2^23.)
        if (__reduce_add_sync(0xffffffffu, whole) > (unsigned)kMostOverlap * (a.total / kBM + 1)) deepest = 0;
        group = a.group;
        p = deepest;
        h0 = 0;
        hn = min(group, heads);
        used = 0;
        next = last = 0;
#pragma unroll
        for (int i = 0; i < kMaxCtas / 32; ++i) load[i] = 0;
    }
    // The next depth's items over the CTAs.
    __device__ void deal() {
        const int lane = threadIdx.x & 31, G = gridDim.x, c = blockIdx.x;
        --p;
        int n = 0;
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) n += __popc(__ballot_sync(0xffffffffu, depth(s0 + lane) > p));
        n *= hn;
        const int w = (a.pair_heads ? p + 1 : 2 * p + 2) + kItemCost;
        if (used + n <= G || used == 0) {  // to CTAs without one, or evenly over all
            const int each = used ? 0 : n / G, more = used ? n : n % G;
            const int mine = each + (c >= used && c < used + more);
            next = each * c + min(max(c - used, 0), more);
            last = next + mine;
#pragma unroll
            for (int i = 0; i < kMaxCtas / 32; ++i) {
                const int k = 32 * i + lane;
                if (k < G) load[i] += w * (each + (k >= used && k < used + more));
            }
            used = each ? G : used + more;
            if (used >= G) used = G;
            return;
        }
        used = G;
        // The level that takes the most items without passing n. (In fp32, the same in every CTA: what matters is that
        // all agree.) It is the mean of what will be there, or less where some loads lie above it.
        int low = 0x7fffffff, high = 0, sum = 0;
#pragma unroll
        for (int i = 0; i < kMaxCtas / 32; ++i)
            if (32 * i + lane < G) low = min(low, load[i]);
        low = (int)__reduce_min_sync(0xffffffffu, low);
#pragma unroll
        for (int i = 0; i < kMaxCtas / 32; ++i)
            if (32 * i + lane < G) {
                load[i] -= low;
                high = max(high, load[i]);
                sum += load[i];
            }
        sum = (int)__reduce_add_sync(0xffffffffu, sum);
        high = (int)__reduce_max_sync(0xffffffffu, high);
        const float inv = 1.0f / (float)w;
        auto takes = [&](int level, int i) {
            return 32 * i + lane < G && load[i] < level ? (int)(((float)(level - load[i]) + 0.5f) * inv) : 0;
        };
        auto total = [&](int level) {
            int t = 0;
#pragma unroll
            for (int i = 0; i < kMaxCtas / 32; ++i) t += takes(level, i);
            return (int)__reduce_add_sync(0xffffffffu, t);
        };
        const int mean = (int)min(((long long)sum + (long long)n * w) / G, 0x3fffffffll);
        int lo = 0, hi = max(high, mean) + w + 1;
        if (mean > 1 && total(mean - 1) <= n) lo = mean - 1;
        while (lo < hi) {
            const int mid = lo + (hi - lo + 1) / 2;
            if (total(mid) <= n) lo = mid;
            else hi = mid - 1;
        }
        // what is left goes to the CTAs that a level higher would give one, in order
        int rest = n - total(lo), before = 0, mine = 0;
#pragma unroll
        for (int i = 0; i < kMaxCtas / 32; ++i) {
            int t = takes(lo, i);
            const bool more = takes(lo + 1, i) > t;
            const unsigned who = __ballot_sync(0xffffffffu, more);
            if (more && __popc(who & ((1u << lane) - 1)) < rest) ++t;
            rest = max(0, rest - __popc(who));
            load[i] += t * w;
            if (32 * i + lane < c) before += t;
            if (32 * i + lane == c) mine = t;
        }
        next = (int)__reduce_add_sync(0xffffffffu, before);
        last = next + (int)__reduce_add_sync(0xffffffffu, mine);
    }
    __device__ Item take() {
        const int lane = threadIdx.x & 31;
        Item it{};
        it.head[0] = -1;
        while (next == last) {
            if (p == 0) {  // the next heads
                h0 += hn;
                hn = min(group, heads - h0);
                p = deepest;
                if (hn <= 0 || p == 0) return it;
            }
            deal();
        }
        const int r0 = next / hn, hh = h0 + next % hn;
        ++next;
        int r = r0;  // the r-th sequence deeper than p
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
            const unsigned deep = __ballot_sync(0xffffffffu, depth(s0 + lane) > p);
            const int n = __popc(deep);
            if (r < n) {
                const int s = s0 + (int)__fns(deep, 0, r + 1);
                it.row0 = a.cu[s];
                it.len = a.cu[s + 1] - it.row0;
                it.head[0] = a.pair_heads ? 2 * hh : hh;
                it.head[1] = a.pair_heads ? 2 * hh + 1 : hh;
                it.kvh = it.head[0] / (a.H / a.Hkv);
                it.tile[0] = a.pair_heads ? p : 2 * p;
                it.tile[1] = a.pair_heads ? p : (2 * p + 1) * kBM < it.len ? 2 * p + 1 : -1;
                return it;
            }
            r -= n;
        }
        return it;
    }
};

// 3-D tiled TMA load (no multicast): box {64 columns, 1 head, 128 rows}.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// One lane of a converged warp. (In a branch on elect.sync the compiler knows
// that one thread is left, and an MMA's operands go straight to uniform
// registers; in `if (lane == 0)` it loops over possible values of each, about
// 100 cycles per 64-cycle product.)
__device__ __forceinline__ bool elect_one() {
    uint32_t p = 0;
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xFFFFFFFF;\n\t@e mov.s32 %0, 1;\n\t}" : "+r"(p));
    return p != 0;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    k_prefill_varlen(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                     const __grid_constant__ CUtensorMap tv, const VarlenArgs a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    uint8_t* base = smem_raw + (((raw + 1023u) & ~1023u) - raw);
    const uint32_t sbase = smem_u32(base);
    constexpr int kTile = tile_bytes<HD>();
    constexpr int kNH = HD / 64;              // 64-column halves of a tile
    constexpr int kOffKV = 2 * kTile;
    constexpr uint32_t kIdescO = umma_idesc_bf16_f32(kBM, HD, true);
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + off_bar<HD>());
    uint64_t* q_full = bars + 0;
    uint64_t* q_empty = bars + 1;
    uint64_t* s_full = bars + 2;              // [2 tiles][2 buffers]
    uint64_t* p_full = bars + 6;              // [2 tiles][2 buffers]
    uint64_t* o_done = bars + 10;             // [2], a phase per P V but an item's last
    uint64_t* o_last = bars + 12;             // [2], a phase per item
    uint64_t* o_free = bars + 14;             // [2]
    uint64_t* item_full = bars + 16;          // [2]
    uint64_t* item_empty = bars + 18;         // [2]
    uint64_t* kv_full = bars + 20;            // [kSlots]
    uint64_t* kv_empty = kv_full + kSlots;    // [kSlots]
    uint64_t* drain = kv_empty + kSlots;
    uint64_t* done = drain + 1;               // every warp finished (one arrival per warp)
    uint32_t* tslot = reinterpret_cast<uint32_t*>(done + 1);
    Item* items = reinterpret_cast<Item*>(tslot + 2);  // [2]

    __shared__ uint32_t s_abort;
    // a wait ran out in an earlier launch: nothing is started before the host has read the word
    if (threadIdx.x == 0) s_abort = *reinterpret_cast<volatile uint32_t*>(a.err) & FORGE_DEVERR_MBAR_TIMEOUT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[2 * i], 1);
            mbar_init(&s_full[2 * i + 1], 1);
            mbar_init(&p_full[2 * i], 128);
            mbar_init(&p_full[2 * i + 1], 128);
            mbar_init(&o_done[i], 1);
            mbar_init(&o_last[i], 1);
            mbar_init(&o_free[i], 128);
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], 2 + kSoftWarps);  // TMA, MMA and softmax warps
        }
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        mbar_init(drain, 1);
        mbar_init(done, kThreads / 32);
        fence_mbar_init();
    }
    Dealer dealer(a);
    Item first{};
    if (warp == kItemWarp) {  // (its loads run beside the barriers' and TMEM's setup)
        dealer.start();
        first = dealer.take();
    }
    if (warp == kTmaWarp && lane < 3) {
        const CUtensorMap* m = lane == 0 ? &tq : lane == 1 ? &tk : &tv;
        asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
    }
    __syncthreads();
    if (s_abort) return;
    if (warp == kMmaWarp) tmem_alloc(tslot, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tslot, 0);
    // TMEM columns: S_A 0-63 and 64-127, O_A 128-255, S_B 256-383, O_B 384-511
    const uint32_t tS[2] = {tmem, tmem + 256}, tO[2] = {tmem + 128, tmem + 384};

    // item n of this CTA, from the items warp
    auto take = [&](int n, Item& it) {
        if (!__all_sync(0xffffffffu, mbar_wait(&item_full[n & 1], (n >> 1) & 1, a.err))) return false;
        it = items[n & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[n & 1]);
        return it.head[0] >= 0;
    };
    auto blocks = [](const Item& it, int t) { return it.tile[t] + 1; };  // key blocks of tile t (0: none)
    // its half blocks: those with keys in the sequence
    auto steps = [](const Item& it, int t) { return it.tile[t] < 0 ? 0 : 2 * it.tile[t] + (it.len - it.tile[t] * kBM > kSub ? 2 : 1); };

    if (warp >= kSoftWarps) {
        if (warp == kItemWarp) {
            // ------------------------------------------------------------ items
            // sequences with bad bounds
            if (blockIdx.x == 0)
                for (int s = lane; s < a.n_seq; s += 32)
                    if (a.cu[s] < 0 || a.cu[s + 1] < a.cu[s] || a.cu[s + 1] > a.total) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
            for (int n = 0;; ++n) {
                const Item it = n ? dealer.take() : first;
                if (!__all_sync(0xffffffffu, mbar_wait(&item_empty[n & 1], ((n >> 1) & 1) ^ 1, a.err))) break;
                if (lane == 0) {
                    items[n & 1] = it;
                    mbar_arrive(&item_full[n & 1]);
                }
                __syncwarp();
                if (it.head[0] < 0) break;
            }
        } else if (warp == kTmaWarp) {
            // --------------------------------------------------------------- TMA
            Item it;
            int slot = 0;        // K/V tiles issued
            int q_waits = 0;     // Q loads issued
            bool ok = true;
            for (int n = 0; ok && take(n, it); ++n) {
                if (lane == 0) {
                    const int nblk = max(blocks(it, 0), blocks(it, 1));
                    ok = mbar_wait(q_empty, (n & 1) ^ 1, a.err);
                    if (ok) {
                        mbar_arrive_expect_tx(q_full, it.tile[1] >= 0 ? 2 * kTile : kTile);
#pragma unroll
                        for (int h2 = 0; h2 < kNH; ++h2) {
                            tma_load_3d(base + h2 * kHalf, &tq, 64 * h2, it.head[0], it.row0 + it.tile[0] * kBM, q_full);
                            if (it.tile[1] >= 0)
                                tma_load_3d(base + kTile + h2 * kHalf, &tq, 64 * h2, it.head[1], it.row0 + it.tile[1] * kBM, q_full);
                        }
                        q_waits = n + 1;
                    }
                    // K0 V0 K1 V1 ...
                    for (int b = 0; ok && b < 2 * nblk; ++b, ++slot) {
                        const int st = slot % kSlots;
                        ok = mbar_wait(&kv_empty[st], ((slot / kSlots) & 1) ^ 1, a.err);
                        if (!ok) break;
                        uint8_t* dst = base + kOffKV + st * kTile;
                        mbar_arrive_expect_tx(&kv_full[st], kTile);
#pragma unroll
                        for (int h2 = 0; h2 < kNH; ++h2)
                            tma_load_3d(dst + h2 * kHalf, b & 1 ? &tv : &tk, 64 * h2, it.kvh, it.row0 + (b >> 1) * kBM, &kv_full[st]);
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if (lane == 0) {  // every copy issued has landed before the CTA may exit
                if (q_waits) mbar_wait(q_full, (q_waits - 1) & 1, a.err);
                for (int i = max(0, slot - kSlots); i < slot; ++i) mbar_wait(&kv_full[i % kSlots], (i / kSlots) & 1, a.err);
            }
        } else if (warp == kMmaWarp) {
            // ------------------------------------------------------ tensor cores
            // (one thread, from here to the end: see elect_one)
            if (elect_one()) {
                const uint64_t desc_q = umma_desc_sw128(sbase, 16, 1024), desc_k = umma_desc_sw128(sbase + kOffKV, 16, 1024);
                const uint64_t desc_v = umma_desc_sw128(sbase + kOffKV, kHalf, 1024);
                uint32_t slot = 0, phase = 0;  // next ring slot and its parity
                uint32_t par = 0;              // parities: bit 2 t + buffer: P taken; bit 4 + t: items that used O of tile t
                bool ok = true;
                for (uint32_t n = 0;; ++n) {
                    if (!mbar_wait(&item_full[n & 1], (n >> 1) & 1, a.err)) break;
                    const Item it = items[n & 1];
                    mbar_arrive(&item_empty[n & 1]);
                    if (it.head[0] < 0) break;
                    // steps of both tiles; a tile's step j: S into buffer j % 2, later O += P V
                    const int n0 = steps(it, 0), n1 = steps(it, 1), most = max(n0, n1);
                    auto next_kv = [&](uint32_t& at) {
                        at = slot;
                        const uint32_t p = phase;
                        if (++slot == kSlots) {
                            slot = 0;
                            phase ^= 1;
                        }
                        return mbar_wait(&kv_full[at], p, a.err);
                    };
                    auto issue_s = [&](int t, int buf, uint32_t ring) {
                        const uint64_t q = desc_q + t * (kTile >> 4), k = desc_k + ring * (kTile >> 4) + buf * (kSub * 128 >> 4);
#pragma unroll
                        for (int s = 0; s < HD / 16; ++s) {
                            const uint32_t off = ((s >> 2) * kHalf + (s & 3) * 32) >> 4;
                            umma_bf16(tS[t] + kSub * buf, q + off, k + off, kIdescS, s > 0);
                        }
                        umma_commit(&s_full[2 * t + buf]);
                    };
                    // P (A operand) lies in TMEM over S, 8 columns per 16 keys
                    auto issue_pv = [&](int t, int buf, uint32_t ring, bool more, bool last) {
                        if (!mbar_wait(&p_full[2 * t + buf], (par >> (2 * t + buf)) & 1, a.err)) return false;
                        par ^= 1u << (2 * t + buf);
                        tc_fence_after();
                        const uint64_t v = desc_v + ring * (kTile >> 4) + buf * (kSub * 128 >> 4);
#pragma unroll
                        for (int s = 0; s < kSub / 16; ++s)
                            umma_bf16_ta(tO[t], tS[t] + kSub * buf + 8 * s, v + s * (2048 >> 4), kIdescO, more || s > 0);
                        umma_commit(last ? &o_last[t] : &o_done[t]);
                        return true;
                    };
                    uint32_t k_at = 0, v_at = 0;
                    if (!mbar_wait(q_full, n & 1, a.err) || !next_kv(k_at)) break;
                    tc_fence_after();
                    if (n0) issue_s(0, 0, k_at);
                    if (n1) issue_s(1, 0, k_at);
                    if (n0 > 1) issue_s(0, 1, k_at);
                    if (n1 > 1) issue_s(1, 1, k_at);
                    umma_commit(&kv_empty[k_at]);
                    if (most <= 2) umma_commit(q_empty);  // the item's last S is issued
                    // the softmax warps have taken the last item's O
                    if (n0) {
                        ok = mbar_wait(&o_free[0], ((par >> 4) & 1) ^ 1, a.err);
                        par ^= 1u << 4;
                    }
                    if (ok && n1) {
                        ok = mbar_wait(&o_free[1], ((par >> 5) & 1) ^ 1, a.err);
                        par ^= 1u << 5;
                    }
                    for (int j = 0; ok && j < most; j += 2) {
                        const bool more_k = j + 2 < most;
                        if (!next_kv(v_at)) { ok = false; break; }
                        bool have_k = false;
#pragma unroll
                        for (int buf = 0; buf < 2; ++buf)
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
                                const int nt = t ? n1 : n0;
                                if (ok && j + buf < nt) {
                                    ok = issue_pv(t, buf, v_at, j + buf > 0, j + buf + 1 == nt);
                                    if (ok && more_k && !have_k) {
                                        have_k = ok = next_kv(k_at);
                                        tc_fence_after();
                                    }
                                    if (ok && j + buf + 2 < nt) issue_s(t, buf, k_at);
                                }
                            }
                        if (!ok) break;
                        umma_commit(&kv_empty[v_at]);
                        if (more_k) umma_commit(&kv_empty[k_at]);
                        if (more_k && j + 4 >= most) umma_commit(q_empty);
                    }
                    if (!ok) break;
                }
                umma_commit(drain);
                mbar_wait(drain, 0, a.err);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ softmax
        const int t = warp >> 2;                  // tile 0 (A) or 1 (B)
        const int r = threadIdx.x & 127;          // query row within the tile
        const uint32_t lrow = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tSm = tS[t] + lrow, tOm = tO[t] + lrow;
        const float c = a.scale_log2;
        Item it;
        uint32_t ns[2] = {0, 0};  // parity of the S taken from either buffer
        uint32_t np = 0;          // P V of this tile so far
        uint32_t no = 0;          // items that had this tile
        int slot0 = 0;            // ring index of the item's K0
        for (int n = 0; take(n, it); ++n) {
            const int nmine = steps(it, t), qt = it.tile[t];
            // Running max in log2 units (m = max * c), raised only when a new score exceeds it by more than 8 (P stays
            // below 2^8, exact enough in bf16 and fp32), so O in TMEM is rescaled rarely; l and O refer to the same m.
            float m = -INFINITY, l = 0.f, cr = c, nm = 0.f;  // P = 2^(S cr + nm)
            bool ok = nmine > 0;
            for (int j = 0; j < nmine; ++j, np += j < nmine) {  // (the last P V has a barrier of its own)
                const int buf = j & 1;
                if (!__all_sync(0xffffffffu, mbar_wait(&s_full[2 * t + buf], buf ? ns[1] : ns[0], a.err))) { ok = false; break; }
                if (buf) ns[1] ^= 1;
                else ns[0] ^= 1;
                tc_fence_after();
                const uint32_t tSb = tSm + kSub * buf;
                uint32_t sv[2][32];
                tmem_ld32(tSb, sv[0]);
                tmem_ld32(tSb + 32, sv[1]);
                tmem_wait_ld();
                if (j >= 2 * qt) {  // the diagonal block
                    const int first = kSub * buf;
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (first + 32 * q + i > r) sv[q][i] = 0xFF800000u;
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        mx4[(i >> 1) & 3] = max3_nan(mx4[(i >> 1) & 3], __uint_as_float(sv[q][i]), __uint_as_float(sv[q][i + 1]));
                const float mx = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]), mxc = mx * c;
                const bool raise = mxc > m + 8.0f || j == 0;
                if (__any_sync(0xffffffffu, raise)) {
                    const float alpha = raise && j > 0 ? ex2(m - mxc) : 1.0f;
                    if (raise) {
                        m = mxc;
                        cr = fabsf(m) > kFar ? kFarScale : c;
                        nm = fabsf(m) > kFar ? -kFarScale * mx : -m;
                    }
                    l *= alpha;
                    if (j > 0) {
                        // P V of the step before has to be in O
                        if (!__all_sync(0xffffffffu, mbar_wait(&o_done[t], (np - 1) & 1, a.err))) { ok = false; break; }
                        tc_fence_after();
#pragma unroll
                        for (int q = 0; q < HD / 32; ++q) {
                            uint32_t ov[32];
                            tmem_ld32(tOm + 32 * q, ov);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                            tmem_st32(tOm + 32 * q, ov);
                        }
                    }
                }
                const F2 c2(cr, cr), nm2(nm, nm);
                F2 sum(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const F2 x = fma2(F2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), c2, nm2);
                        // of 4 pairs, 1 on the FMA pipe (the exp2 unit takes 8 cycles for a warp's value)
                        const F2 p = e % 4 == 1 ? exp2_fma(x) : F2(ex2(x.x()), ex2(x.y()));
                        sum = sum + p;
                        pk[e] = pack_bf16x2(p.x(), p.y());
                    }
                    tmem_st16(tSb + 16 * q, pk);
                }
                l += isnan(mxc) ? NAN : sum.x() + sum.y();  // (a NaN score makes the row NaN)
                // the sequence ends inside the half block: V rows behind its end count for nothing
                const int valid = it.len - j * kSub;
                if (valid < kSub) {
                    const int b = slot0 + (j | 1), row = r & (kSub - 1), half = r / kSub;
                    mbar_wait(&kv_full[b % kSlots], (b / kSlots) & 1, a.err);
                    if (row >= valid && half < kNH) {
                        uint4* z = reinterpret_cast<uint4*>(base + kOffKV + (b % kSlots) * kTile + half * kHalf + (kSub * buf + row) * 128);
#pragma unroll
                        for (int i = 0; i < 8; ++i) z[i] = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[2 * t + buf]);
            }
            slot0 += 2 * max(blocks(it, 0), blocks(it, 1));
            if (nmine == 0) continue;
            if (!ok || !__all_sync(0xffffffffu, mbar_wait(&o_last[t], no & 1, a.err))) break;
            ++no;
            tc_fence_after();
            const float inv = 1.0f / l;
            const int i = qt * kBM + r;           // row in the sequence
            uint16_t* orow = a.o + (int64_t)(it.row0 + i) * a.ldo + (int64_t)it.head[t] * HD;
            uint32_t ov[HD / 32][32];
#pragma unroll
            for (int q = 0; q < HD / 32; ++q) tmem_ld32(tOm + 32 * q, ov[q]);
            tmem_wait_ld();
            tc_fence_before();
            mbar_arrive(&o_free[t]);
            if (i < it.len) {
#pragma unroll
                for (int q = 0; q < HD / 32; ++q)
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = pack_bf16x2(__uint_as_float(ov[q][k + 2 * e]) * inv, __uint_as_float(ov[q][k + 2 * e + 1]) * inv);
                        *reinterpret_cast<uint4*>(orow + 32 * q + k) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                if (a.lse) a.lse[(int64_t)it.head[t] * a.total + it.row0 + i] = (m + log2f(l)) * 0.6931471805599453f;
            }
        }
    }
    // End: every warp reports on an mbarrier and the TMEM-owning warp waits
    // for all of them before it frees TMEM.
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(done);
    if (warp == kMmaWarp) {
        mbar_wait(done, 0, a.err);
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---- host ------------------------------------------------------------------------
// [total][heads][hd] bf16 rows ld apart as boxes of 64 columns x 1 head x 128 rows, 128-byte swizzle.
int make_map(CUtensorMap* m, const void* ptr, int total, int heads, int hd, int64_t ld) {
    ForgeEncodeTiled enc = forge_tensor_map_encoder();
    if (!enc) return forge_fail(-1, "forge_flash_prefill_varlen: cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)total};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)ld * 2};
    const cuuint32_t box[3] = {64, 1, kBM};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(ptr), dims, strides, box, estr,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : forge_fail(-1, "forge_flash_prefill_varlen: tensor map encode failed (%d)", (int)r);
}

int configure() {
    static bool done[64] = {false};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return forge_fail(-1, "forge_flash_prefill_varlen: no device");
    if (done[dev]) return 0;
    cudaError_t e = cudaFuncSetAttribute(k_prefill_varlen<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<128>());
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_prefill_varlen<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<64>());
    if (e != cudaSuccess) return forge_fail(-1, "forge_flash_prefill_varlen: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    done[dev] = true;
    return 0;
}
}  // namespace

extern "C" FORGE_API int forge_flash_prefill_varlen(const uint16_t* q, int64_t ldq, const uint16_t* k, int64_t ldk,
                                                    const uint16_t* v, int64_t ldv, const int32_t* cu_seqlens, int n_seq,
                                                    int total, int H, int Hkv, int hd, uint16_t* o, int64_t ldo,
                                                    float* lse, void* stream) {
    if (!q || !k || !v || !o || !cu_seqlens || n_seq < 0 || total < 0 || H <= 0 || Hkv <= 0 || H % Hkv || n_seq > 65535 ||
        H > 65535 || total > (1 << 30))
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_prefill_varlen: bad args");
    if (hd != 128 && hd != 64)
        return forge_fail(FORGE_KERNEL_UNSUPPORTED, "forge_flash_prefill_varlen: head_dim %d (128 or 64)", hd);
    if (ldq < (int64_t)H * hd || ldo < (int64_t)H * hd || ldk < (int64_t)Hkv * hd || ldv < (int64_t)Hkv * hd ||
        (ldq | ldk | ldv | ldo) % 8 || (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) & 15))
        return forge_fail(FORGE_INVALID_ARGS, "forge_flash_prefill_varlen: rows must be 16-byte aligned and at least their heads long");
    if (n_seq == 0 || total == 0) return 0;
    VarlenArgs a{};
    a.pair_heads = (H / Hkv) % 2 == 0;
    // the most items there can be: whole tiles of the rows, and one more per sequence
    const int rows = a.pair_heads ? kBM : 2 * kBM;
    const int64_t items = ((int64_t)total / rows + n_seq) * (a.pair_heads ? H / 2 : H);
    if (items > 0x3fffffff) return forge_fail(FORGE_INVALID_ARGS, "forge_flash_prefill_varlen: total x heads is too large");
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_flash_prefill_varlen: no device");
    if (configure()) return -1;
    CUtensorMap mq, mk, mv;
    if (make_map(&mq, q, total, H, hd, ldq) || make_map(&mk, k, total, Hkv, hd, ldk) || make_map(&mv, v, total, Hkv, hd, ldv)) return -1;
    a.cu = cu_seqlens; a.n_seq = n_seq; a.total = total; a.H = H; a.Hkv = Hkv;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt((double)hd));
    a.o = o; a.ldo = ldo; a.lse = lse; a.err = err;
    // half of L2 for the K and V of a group's heads
    const int64_t kv_bytes = (int64_t)total * hd * 4, per_tile = a.pair_heads ? H / 2 : H;
    const int64_t kv_heads = (60ll << 20) / kv_bytes;
    const int64_t group = (kv_heads < 1 ? 1 : kv_heads) * per_tile / Hkv;
    a.group = (int)(group < 1 ? 1 : group < per_tile ? group : per_tile);
    const int sms = forge_sm_count() < kMaxCtas ? forge_sm_count() : kMaxCtas;
    const unsigned grid = (unsigned)(items < sms ? items : sms);
    if (hd == 128) k_prefill_varlen<128><<<grid, kThreads, smem_bytes<128>(), (cudaStream_t)stream>>>(mq, mk, mv, a);
    else k_prefill_varlen<64><<<grid, kThreads, smem_bytes<64>(), (cudaStream_t)stream>>>(mq, mk, mv, a);
    return forge_check_launch("forge_flash_prefill_varlen");
}
