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
// one head. CTAs are persistent, one per SM; items are ordered by the number
// of their key blocks, longest first, and dealt out back and forth, so each
// CTA gets about the same work whatever the lengths. The order needs no table:
// item k's depth p is where the number of tiles at depth p or more, a sum over
// the sequences, passes k (a few warp-wide sums by a warp of its own, one item
// ahead of the others).
//
//   warps 0-3 / 4-7    softmax of tile A / B, one thread per query row
//   warp 8             TMA: Q of both tiles, K and V through a 4-slot ring
//   warp 9 (one lane)  tensor-core issue, tiles alternating
//   warp 10            items
//
// S = Q K^T (128 x 128 x hd) goes to TMEM; its thread takes the whole row into
// registers (setmaxnreg moves registers from the other warps), so TMEM is read
// once and P = 2^(S c - m) can overwrite S as bf16 pairs, the A operand of
// O += P V. P is handed over in two halves: the product of the first 64 keys
// runs while the second half's exponentials do. m is raised only when a score
// exceeds it by more than 2^8, so O in TMEM is rarely rescaled.
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
constexpr int kThreads = 384;
constexpr int kSlots = 4;      // K/V ring
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kIdescS = umma_idesc_bf16_f32(kBM, kBM, false);
template <int HD> constexpr int tile_bytes() { return kBM * HD * 2; }
template <int HD> constexpr int off_bar() { return (2 + kSlots) * tile_bytes<HD>(); }
template <int HD> constexpr int smem_bytes() { return off_bar<HD>() + 512 + 1024; }

struct VarlenArgs {
    const int32_t* cu;
    int n_seq, total, H, Hkv;
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

// Item `i` of the launch (a whole warp calls it).
__device__ Item find_item(const VarlenArgs& a, int i) {
    const int lane = threadIdx.x & 31;
    const int rows = a.pair_heads ? kBM : 2 * kBM, per_tile = a.pair_heads ? a.H / 2 : a.H;
    const int k = i / per_tile, hh = i % per_tile;
    auto depth = [&](int s) {  // tiles of sequence s; a sequence with bad bounds has none
        if (s >= a.n_seq) return 0;
        const int b = a.cu[s], e = a.cu[s + 1];
        return b < 0 || e < b || e > a.total ? 0 : (e - b + rows - 1) / rows;
    };
    const int first = depth(lane);
    auto each = [&](int s0) { return s0 ? depth(s0 + lane) : first; };
    auto from = [&](int p) {  // tiles at depth p or more
        int n = 0;
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) n += max(0, each(s0) - p);
        return (int)__reduce_add_sync(0xffffffffu, n);
    };
    Item it{};
    it.head[0] = -1;
    int lo = 0, hi = a.total / rows + 1;  // from(hi) == 0 <= k; the least p with from(p) <= k
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (from(mid) <= k) hi = mid;
        else lo = mid + 1;
    }
    if (lo == 0) return it;  // k is behind the last tile
    const int p = lo - 1;
    int r = k - from(lo);    // the r-th sequence deeper than p
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        const unsigned deep = __ballot_sync(0xffffffffu, each(s0) > p);
        const int n = __popc(deep);
        if (r < n) {
            const int s = s0 + __fns(deep, 0, r + 1);
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

// 3-D tiled TMA load (no multicast): box {64 columns, 1 head, 128 rows}.
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
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
    uint64_t* s_full = bars + 2;              // [2] per tile
    uint64_t* p_full = bars + 4;              // [2 tiles][2 halves]
    uint64_t* o_done = bars + 8;              // [2]
    uint64_t* o_free = bars + 10;             // [2]
    uint64_t* item_full = bars + 12;          // [2]
    uint64_t* item_empty = bars + 14;         // [2]
    uint64_t* kv_full = bars + 16;            // [kSlots]
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
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[2 * i], 128);
            mbar_init(&p_full[2 * i + 1], 128);
            mbar_init(&o_done[i], 1);
            mbar_init(&o_free[i], 128);
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], 10);  // TMA, MMA and 8 softmax warps
        }
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(&kv_full[i], 1);
            mbar_init(&kv_empty[i], 1);
        }
        mbar_init(drain, 1);
        mbar_init(done, kThreads / 32);
        fence_mbar_init();
    }
    __syncthreads();
    if (s_abort) return;
    if (warp == 9) tmem_alloc(tslot, kTmemCols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tslot;
    // TMEM columns: S_A 0-127, O_A 128-255, S_B 256-383, O_B 384-511
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

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
        if (warp == 10) {
            // ------------------------------------------------------------ items
            // sequences with bad bounds
            if (blockIdx.x == 0)
                for (int s = lane; s < a.n_seq; s += 32)
                    if (a.cu[s] < 0 || a.cu[s + 1] < a.cu[s] || a.cu[s + 1] > a.total) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
            for (int n = 0;; ++n) {
                // the ordered items back and forth over the CTAs
                const long long i = (long long)n * gridDim.x + (n & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
                Item it = find_item(a, i > 0x7fffffff ? 0x7fffffff : (int)i);
                if (!__all_sync(0xffffffffu, mbar_wait(&item_empty[n & 1], ((n >> 1) & 1) ^ 1, a.err))) break;
                if (lane == 0) {
                    items[n & 1] = it;
                    mbar_arrive(&item_full[n & 1]);
                }
                __syncwarp();
                if (it.head[0] < 0) break;
            }
        } else if (warp == 8) {
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
        } else if (warp == 9) {
            // ------------------------------------------------------ tensor cores
            Item it;
            int slot0 = 0;              // ring index of the item's K0
            int np[2] = {0, 0};         // P blocks taken of each tile
            int no[2] = {0, 0};         // items that used O of each tile
            bool ok = true;
            for (int n = 0; ok && take(n, it); ++n) {
                const int nA = blocks(it, 0), nB = blocks(it, 1), nblk = max(nA, nB);
                if (lane == 0) {
                    auto slot_addr = [&](int b) { return sbase + (uint32_t)(kOffKV + ((slot0 + b) % kSlots) * kTile); };
                    auto wait_kv = [&](int b) {
                        const int i = slot0 + b;
                        return mbar_wait(&kv_full[i % kSlots], (i / kSlots) & 1, a.err);
                    };
                    auto free_kv = [&](int b) { umma_commit(&kv_empty[(slot0 + b) % kSlots]); };
                    auto issue_s = [&](int t, int j) {
                        const uint32_t kb = slot_addr(2 * j), qb = sbase + (uint32_t)(t * kTile);
#pragma unroll
                        for (int s = 0; s < HD / 16; ++s) {
                            const uint32_t off = (uint32_t)((s >> 2) * kHalf + (s & 3) * 32);
                            umma_bf16(tS[t], umma_desc_sw128(qb + off, 16, 1024), umma_desc_sw128(kb + off, 16, 1024), kIdescS,
                                      s > 0 ? 1u : 0u);
                        }
                        umma_commit(&s_full[t]);
                    };
                    // O += P V in two halves as P arrives; P (A operand) lies in TMEM over S, 8 columns per 16 keys
                    auto issue_pv = [&](int t, int j, bool last) {
                        const uint32_t vb = slot_addr(2 * j + 1);
                        for (int hf = 0; hf < 2; ++hf) {
                            if (!mbar_wait(&p_full[2 * t + hf], np[t] & 1, a.err)) return false;
                            tc_fence_after();
#pragma unroll
                            for (int s = 4 * hf; s < 4 * hf + 4; ++s)
                                umma_bf16_ta(tO[t], tS[t] + (uint32_t)(8 * s), umma_desc_sw128(vb + (uint32_t)s * 2048u, kHalf, 1024),
                                             kIdescO, (j > 0 || s > 0) ? 1u : 0u);
                        }
                        ++np[t];
                        if (last) umma_commit(&o_done[t]);
                        return true;
                    };
                    ok = mbar_wait(q_full, n & 1, a.err) && wait_kv(0);
                    if (ok) {
                        tc_fence_after();
                        issue_s(0, 0);
                        if (nB) issue_s(1, 0);
                        free_kv(0);
                        if (nblk == 1) umma_commit(q_empty);
                    }
                    // the softmax warps have taken the last item's O
                    for (int t = 0; t < 2; ++t)
                        if (ok && (t ? nB : nA)) {
                            ok = mbar_wait(&o_free[t], (no[t] & 1) ^ 1, a.err);
                            ++no[t];
                        }
                    for (int j = 0; ok && j < nblk; ++j) {
                        ok = wait_kv(2 * j + 1);
                        if (ok && j < nA) ok = issue_pv(0, j, j + 1 == nA);
                        // tile A's next S overlaps tile B's softmax of this block
                        const bool nextA = j + 1 < nA, nextB = j + 1 < nB;
                        if (ok && (nextA || nextB)) {
                            ok = wait_kv(2 * j + 2);
                            if (!ok) break;
                            tc_fence_after();
                            if (nextA) issue_s(0, j + 1);
                        }
                        if (ok && j < nB) ok = issue_pv(1, j, j + 1 == nB);
                        if (!ok) break;
                        free_kv(2 * j + 1);
                        if (nextB) issue_s(1, j + 1);
                        if (nextA || nextB) free_kv(2 * j + 2);
                        if (j + 2 == nblk) umma_commit(q_empty);  // the item's last S is issued
                    }
                }
                slot0 += 2 * nblk;
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if (lane == 0) {
                umma_commit(drain);
                mbar_wait(drain, 0, a.err);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int t = warp >> 2;                  // tile 0 (A) or 1 (B)
        const int r = threadIdx.x & 127;          // query row within the tile
        const uint32_t lrow = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tSm = tS[t] + lrow, tOm = tO[t] + lrow;
        const float c = a.scale_log2;
        Item it;
        int ns = 0;      // S blocks taken
        int no = 0;      // items that used O
        int slot0 = 0;   // ring index of the item's K0
        for (int n = 0; take(n, it); ++n) {
            const int nmine = blocks(it, t), nblk = max(blocks(it, 0), blocks(it, 1));
            const int qt = it.tile[t];
            // Running max in log2 units (m = max * c), raised only when a new score exceeds it by more than 8 (P stays
            // below 2^8, exact enough in bf16 and fp32), so O in TMEM is rescaled rarely; l and O refer to the same m.
            float m = -INFINITY, l = 0.f;
            bool ok = nmine > 0;
            for (int j = 0; j < nmine; ++j, ++ns) {
                if (!__all_sync(0xffffffffu, mbar_wait(&s_full[t], ns & 1, a.err))) { ok = false; break; }
                tc_fence_after();
                uint32_t sv[4][32];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32(tSm + 32 * q, sv[q]);
                tmem_wait_ld();
                if (j == qt) {  // the diagonal block
#pragma unroll
                    for (int q = 0; q < 4; ++q)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (32 * q + i > r) sv[q][i] = 0xFF800000u;
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 32; i += 2)
                        mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(sv[q][i]), __uint_as_float(sv[q][i + 1]));
                const float mxc = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * c;
                const bool raise = mxc > m + 8.0f || m == -INFINITY;
                const float m_new = raise ? mxc : m;
                const float alpha = raise && j > 0 ? ex2(m - m_new) : 1.0f;
                // (S of block j is complete, so is O += P V of block j - 1, issued before it)
                if (j > 0 && __any_sync(0xffffffffu, raise)) {
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
                const F2 c2(c, c), nm2(-m_new, -m_new);
                F2 sum(0.f, 0.f);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t pk[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const F2 x = fma2(F2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), c2, nm2);
                        const F2 p(ex2(x.x()), ex2(x.y()));
                        sum = sum + p;
                        pk[e] = pack_bf16x2(p.x(), p.y());
                    }
                    tmem_st16(tSm + 16 * q, pk);
                    if (q == 1) {
                        tmem_wait_st();
                        // the sequence ends inside the block: V rows behind its end count for nothing
                        const int valid = it.len - j * kBM;
                        if (valid < kBM) {
                            const int b = slot0 + 2 * j + 1;
                            mbar_wait(&kv_full[b % kSlots], (b / kSlots) & 1, a.err);
                            if (r >= valid) {
                                uint4* row = reinterpret_cast<uint4*>(base + kOffKV + (b % kSlots) * kTile + r * 128);
#pragma unroll
                                for (int h2 = 0; h2 < kNH; ++h2)
#pragma unroll
                                    for (int i = 0; i < 8; ++i) row[h2 * (kHalf / 16) + i] = make_uint4(0, 0, 0, 0);
                            }
                            fence_proxy_async_smem();
                        }
                        tc_fence_before();
                        mbar_arrive(&p_full[2 * t]);
                    }
                }
                l = l * alpha + (sum.x() + sum.y());
                m = m_new;
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(&p_full[2 * t + 1]);
            }
            slot0 += 2 * nblk;
            if (nmine == 0) continue;
            if (!ok || !__all_sync(0xffffffffu, mbar_wait(&o_done[t], no & 1, a.err))) break;
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
    if (warp == 9) {
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
    const int sms = forge_sm_count();
    const unsigned grid = (unsigned)(items < sms ? items : sms);
    if (hd == 128) k_prefill_varlen<128><<<grid, kThreads, smem_bytes<128>(), (cudaStream_t)stream>>>(mq, mk, mv, a);
    else k_prefill_varlen<64><<<grid, kThreads, smem_bytes<64>(), (cudaStream_t)stream>>>(mq, mk, mv, a);
    return forge_check_launch("forge_flash_prefill_varlen");
}
