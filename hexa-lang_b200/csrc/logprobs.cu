// logprobs.cu — log probabilities of given tokens, entropy, rank and the top
// alternatives of logits rows, in one pass over the logits.
//
// Per row, in units of log 2, with w_i = z_i log2 e - c, c near the row's
// maximum, s = sum 2^w and t = sum w 2^w:
//   log p_i = (w_i - log2 s) ln 2,   entropy = (log2 s - t / s) ln 2.
// Every thread keeps (c, s, t) of what it has read, one exponential per
// logit, and moves them when its maximum grows; threads, warps and the CTAs
// of a row join them in a fixed order. The rank is a count of the logits
// above the token's (or equal and before it), in the same pass.
//
// Top alternatives: entries are ordered by a 64-bit key, the logit as an
// ordered integer above the complement of its index, so that no two are
// equal and the lowest index wins. Candidates are the vectors of a thread in a
// group, ordered by their largest logit: when `top` candidates reach a
// threshold, every one that does not has `top` entries before its own. The
// first group sets the threshold (the top-th largest of what is left of each
// warp's largest few), and it is raised in the same way in groups 2, 8, 32; a
// group's maximum, which the softmax needs, is compared with it, and the few
// that reach it go to a list. At the end their logits are read again and the
// keys of those that reach it ordered by counting, each thread those above its
// own. Rows whose list overflows (rising logits) are collected once
// more, with the list cut to the best whenever it is full.
//
// What bounds it: 2048 rows of 50257 in bf16 with 20 alternatives take 68 us
// (3.0 TB/s, the bytes alone 31), by instructions: 0.68 of the issue slots,
// about 80 for 8 logits of a thread without alternatives (45 us) and 45 more
// with them. For few rows a row is shared by a cluster of CTAs that join
// through distributed shared memory, without a workspace or a second launch:
// one row of 32000 takes 6 us, launch and latencies. CTAs that stay and load
// their next row during the end of one took 104 us: rows then start and end
// together, and their ends no longer hide behind other rows' streams.
#include <climits>
#include <cmath>
#include <cooperative_groups.h>
#include "common.cuh"
#include "f32x2.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"

namespace {
namespace cg = cooperative_groups;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kVecs = 4;             // vectors of a thread in a group, in flight together
constexpr int kMaxTop = FORGE_LOGPROBS_MAX_TOP;
constexpr int kList = 512;           // candidates (all threads' of the first group fit)
constexpr int kKeys = 256;           // keys that are ordered by counting (a cluster's 8 times 32)
constexpr int kCtasPerSm = 4;
// Logits below kFloor count as kFloor and c is at least kLeast log2 e: such
// logits have no weight beside any above kLeast, and no infinity arises. c is
// m log2 e rounded, 2^-24 of it beside the exponent of the maximum itself: rows
// with a maximum beyond +-kFar, where that is 0.09, are summed again, slowly.
constexpr float kFloor = -1e30f, kLeast = -1e29f, kFar = 1e6f;
constexpr int kMaxCluster = 8;

struct LogprobArgs {
    const void* z;
    int64_t ld;
    int V, top, rows;
    const int32_t* tok;
    float *logprob, *entropy;
    int32_t *rank, *ids;
    float* tops;
    uint32_t* err;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Order of the logits as an unsigned number: NaN as -inf, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
    if (isnan(x)) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float x, int i) { return (uint64_t)ordered(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u >> 31 ? u & 0x7FFFFFFFu : ~u);
}

// A 16-byte vector of logits: its elements as fp32 pairs, those below kFloor
// raised to it (NaN kept); its maximum (NaN left out, -inf at least); a count
// of the elements above a bound; kNone, a vector of -inf.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int kN = 4;
    static constexpr uint32_t kNone = 0xFF800000u;
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ float raised(uint32_t x) {
        float r;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(x)), "f"(kFloor));
        return r;
    }
    static __device__ __forceinline__ F2 pair(const uint4& v, int i) {
        return i ? F2(raised(v.z), raised(v.w)) : F2(raised(v.x), raised(v.y));
    }
    static __device__ __forceinline__ F2 raw(const uint4& v, int i) {
        return i ? F2(__uint_as_float(v.z), __uint_as_float(v.w)) : F2(__uint_as_float(v.x), __uint_as_float(v.y));
    }
    static __device__ __forceinline__ float below(float x) { return nextafterf(x, -INFINITY); }
    struct Max {
        float m = -INFINITY;
        __device__ __forceinline__ void add(const uint4& v) {
            m = max3(m, __uint_as_float(v.x), __uint_as_float(v.y));
            m = max3(m, __uint_as_float(v.z), __uint_as_float(v.w));
        }
        __device__ __forceinline__ float get() const { return m; }
    };
    struct Count {
        int n = 0;
        __device__ __forceinline__ void add(const uint4& v, float f) {
            n += (__uint_as_float(v.x) > f) + (__uint_as_float(v.y) > f) + (__uint_as_float(v.z) > f) + (__uint_as_float(v.w) > f);
        }
        __device__ __forceinline__ int get() const { return n; }
    };
};
template <> struct Vec<uint16_t> {
    static constexpr int kN = 8;
    static constexpr uint32_t kNone = 0xFF80FF80u;
    static __device__ __forceinline__ float one(const uint16_t* p) { return bf16_bits_to_f32(*p); }
    static __device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
    static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
    static __device__ __forceinline__ F2 pair(const uint4& v, int i) {
        const __nv_bfloat162 r = __hmax2_nan(two(word(v, i)), __float2bfloat162_rn(kFloor));
        const uint32_t w = *reinterpret_cast<const uint32_t*>(&r);
        return F2(bf16_lo_f32(w), bf16_hi_f32(w));
    }
    static __device__ __forceinline__ F2 raw(const uint4& v, int i) { return F2(bf16_lo_f32(word(v, i)), bf16_hi_f32(word(v, i))); }
    static __device__ __forceinline__ float below(float x) {  // the next bf16 down
        const uint32_t u = __float_as_uint(x + 0.0f);
        return __uint_as_float(u == 0 ? 0x80010000u : u >> 31 ? u + 0x10000u : u - 0x10000u);
    }
    struct Max {
        __nv_bfloat162 m = __floats2bfloat162_rn(-INFINITY, -INFINITY);
        __device__ __forceinline__ void add(const uint4& v) {
#pragma unroll
            for (int i = 0; i < 4; ++i) m = __hmax2(m, two(word(v, i)));
        }
        __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
    };
    struct Count {  // (bf16 counts to 256: a group has 16 in each half)
        __nv_bfloat162 n = __floats2bfloat162_rn(0.f, 0.f);
        __device__ __forceinline__ void add(const uint4& v, float f) {
            const __nv_bfloat162 f2 = __float2bfloat162_rn(f);  // (a bf16 logit: exact)
#pragma unroll
            for (int i = 0; i < 4; ++i) n = __hadd2(n, __hgt2(two(word(v, i)), f2));
        }
        __device__ __forceinline__ int get() const { return (int)(__low2float(n) + __high2float(n)); }
    };
};

// Sums of a set of logits relative to c (all finite, or NaN in s and t).
struct Stats {
    float c, s, t;
    __device__ __forceinline__ void join(const Stats& o) {
        const float n = fmaxf(c, o.c), a = c - n, b = o.c - n, ea = ex2(a), eb = ex2(b);
        t = fmaf(ea, fmaf(s, a, t), eb * fmaf(o.s, b, o.t));
        s = fmaf(s, ea, o.s * eb);
        c = n;
    }
};

struct Shared {
    int list[kList];                        // candidates: a thread's vectors of a group, by the first of them
    alignas(16) uint64_t keys[kKeys];
    uint64_t best[kMaxTop];                 // largest first; 0 where there are fewer
    uint64_t gather[kKeys];                 // the cluster's best, in its first CTA
    uint64_t edge[16], bound[kMaxTop];
    Stats stat[kWarps], gstat[kMaxCluster];
    float max[kWarps], gmax[kMaxCluster];
    int rank[kWarps], grank[kMaxCluster], part[kWarps];
    int n;
};

// The warp's largest number.
__device__ __forceinline__ uint64_t warp_max(uint64_t x) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32));
    const uint32_t lo = __reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u);
    return (uint64_t)hi << 32 | lo;
}

__device__ __forceinline__ uint32_t warp_max(uint32_t x) { return __reduce_max_sync(0xffffffffu, x); }

// A number that at least `top` threads' numbers reach, close below the top-th
// largest: the top-th of the `rounds` largest of each warp. 0 where that finds
// fewer that are not 0.
template <typename N>
__device__ __forceinline__ N top_th(Shared& sh, N x, int rounds, int top) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto drop = [&](N& x) {  // the warp's largest, taken out once
        const N big = warp_max(x);
        if (lane == __ffs(__ballot_sync(0xffffffffu, x == big)) - 1) x = 0;
        return big;
    };
    N* bound = reinterpret_cast<N*>(sh.bound);
    __syncthreads();
    for (int r = 0; r < rounds; ++r) {
        const N big = drop(x);
        if (lane == 0) bound[r * kWarps + warp] = big;
    }
    __syncthreads();
    N b = lane < rounds * kWarps ? bound[lane] : 0;
    const int n = __popc(__ballot_sync(0xffffffffu, b != 0));
    if (n < top) return 0;
    if (top <= n - top) {
        for (int r = 1; r < top; ++r) drop(b);
        return warp_max(b);
    }
    b = b ? ~b : 0;
    for (int r = 0; r < n - top; ++r) drop(b);
    return ~warp_max(b);
}

// Sum over the block.
__device__ __forceinline__ int block_sum(Shared& sh, int c) {
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) sh.part[threadIdx.x >> 5] = c;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) n += sh.part[w];
    __syncthreads();
    return n;
}

// A threshold that at least `want` and, keys being distinct, at most `most`
// keys of the block reach, by bisection; count(T) is the calling thread's
// number of keys at or above T, and at least `want` keys exist.
template <typename F>
__device__ uint64_t bisect(Shared& sh, int want, int most, F count) {
    uint64_t lo = 0, hi = ~0ull;  // `want` keys reach lo, fewer reach hi + 1
    while (lo < hi) {
        const uint64_t mid = lo + (hi - lo) / 2 + 1;
        const int n = block_sum(sh, count(mid));
        if (n < want) {
            hi = mid - 1;
        } else {
            lo = mid;
            if (n <= most) break;
        }
    }
    return lo;
}

// The largest `top` of the n keys in sh.keys (fewer if there are fewer) into
// sh.best, in order: a thread counts the keys above its own.
__device__ __forceinline__ void select(Shared& sh, int n, int top) {
    static_assert(kKeys == kThreads, "a key a thread");
    const uint64_t k = (int)threadIdx.x < n ? sh.keys[threadIdx.x] : 0;
    if (threadIdx.x < kMaxTop) sh.best[threadIdx.x] = 0;
    if ((int)threadIdx.x >= n && (int)threadIdx.x < ((n + 7) & ~7)) sh.keys[threadIdx.x] = 0;
    __syncthreads();
    if (k) {
        int above = 0;
        for (int i = 0; i < n; i += 8)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(sh.keys + i + j);
                above += (x.x > k) + (x.y > k);
            }
        if (above < top) sh.best[above] = k;
    }
    __syncthreads();
}

// The best of the listed candidates, the keys in sh.edge and those already in
// sh.best, into sh.best; a candidate is `per` vectors kThreads apart, those
// behind v1 left out; floor: a key that at least `top` of them reach (or 1).
template <typename T, int per>
__device__ __forceinline__ void settle(Shared& sh, const T* z, int head, int v1, int listed, int top, uint64_t floor) {
    using V = Vec<T>;
    uint64_t own = 0;
    if (threadIdx.x < kMaxTop) own = sh.best[threadIdx.x];
    else if (threadIdx.x < kMaxTop + 16) own = sh.edge[threadIdx.x - kMaxTop];
    auto each = [&](float least, auto f) {  // the keys of logits not below `least`
        if (own) f(own);
#pragma unroll 1
        for (int i = threadIdx.x; i < listed * per; i += kThreads) {
            const int at = sh.list[i / per] + i % per * kThreads, first = head + at * V::kN;
            if (at >= v1) continue;
            const uint4 v = *reinterpret_cast<const uint4*>(z + first);
#pragma unroll
            for (int j = 0; j < V::kN / 2; ++j) {
                const F2 x = V::raw(v, j);
                if (!(x.x() < least)) f(key_of(x.x(), first + 2 * j));
                if (!(x.y() < least)) f(key_of(x.y(), first + 2 * j + 1));
            }
        }
    };
    auto gather = [&](uint64_t cut) {
        __syncthreads();
        if (threadIdx.x == 0) sh.n = 0;
        __syncthreads();
        each(cut > 1 ? value_of(cut) : -INFINITY, [&](uint64_t key) {
            if (key >= cut) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kKeys) sh.keys[at] = key;
            }
        });
        __syncthreads();
        return sh.n;
    };
    int n = gather(floor);
    if (n > kKeys) {  // equal or rising logits
        floor = bisect(sh, top, kKeys, [&](uint64_t x) { int c = 0; each(-INFINITY, [&](uint64_t key) { c += key >= x; }); return c; });
        n = gather(floor);
    }
    if (threadIdx.x < 16) sh.edge[threadIdx.x] = 0;
    select(sh, n, top);
}

// The best of vectors [v0, v1) and the keys in sh.edge into sh.best, for rows
// whose candidates do not fit the list: 256 vectors at a time.
template <typename T>
__device__ __noinline__ void collect(Shared& sh, const T* z, int head, int v0, int v1, int top) {
    using V = Vec<T>;
    uint64_t thr = 0;  // vectors (largest logit, index) below it are out
    int listed = 0;
    for (int base = v0; base < v1; base += kThreads) {
        const int i = base + (int)threadIdx.x;
        uint64_t key = 0;
        if (i < v1) {
            typename V::Max m;
            m.add(*reinterpret_cast<const uint4*>(z + head + (int64_t)i * V::kN));
            key = key_of(m.get(), i);
        }
        bool in = key && key >= thr;
        if (listed + __syncthreads_count(in) > kList) {
            settle<T, 1>(sh, z, head, v1, listed, top, thr ? sh.best[top - 1] : 1);
            listed = 0;
            if (const uint64_t last = sh.best[top - 1]) thr = key_of(value_of(last), max(0, index_of(last) - head) / V::kN);
            in = key && key >= thr;
            __syncthreads();
        }
        if (threadIdx.x == 0) sh.n = listed;
        __syncthreads();
        if (in) sh.list[atomicAdd(&sh.n, 1)] = i;
        __syncthreads();
        listed = sh.n;
    }
    settle<T, 1>(sh, z, head, v1, listed, top, thr ? sh.best[top - 1] : 1);
}

// exp(z - m) and (z - m) exp(z - m) over a row by the calling CTA, for
// maxima so far out that log2 e times them is too coarse, or no fp32 number.
template <typename T>
__device__ __noinline__ void slow_sums(Shared& sh, const T* z, int n, float m, float* s_out, float* t_out) {
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float d = Vec<T>::one(z + i) - m, e = ex2(d * kLog2e);
        s += e;
        t = fmaf(e, d < -1e4f ? -1e4f : d, t);
    }
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.stat[threadIdx.x >> 5] = Stats{0.f, s, t};
    __syncthreads();
    s = t = 0.f;
    for (int w = 0; w < kWarps; ++w) {
        s += sh.stat[w].s;
        t += sh.stat[w].t;
    }
    *s_out = s;
    *t_out = t;
}

// One cluster of `cluster` CTAs per row (a CTA alone where that is 1).
template <typename T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) k_logprobs(const LogprobArgs a, const int cluster) {
    __shared__ Shared sh;
    using V = Vec<T>;
    constexpr int kPairs = V::kN / 2, kGroup = kThreads * kVecs;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = cluster > 1 ? (int)cg::this_cluster().block_rank() : 0;
    if (cluster > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // every CTA runs
    const int row = blockIdx.x / cluster;
    const T* z = (const T*)a.z + (int64_t)row * a.ld;
    const int top = a.top;

    // the CTA's vectors [v0, v1) of the row, cut at 16-byte boundaries of memory
    const int head = min(a.V, (int)(((16 - ((uintptr_t)z & 15)) & 15) / sizeof(T)));
    const int vecs = (a.V - head) / V::kN;
    const int v0 = (int)((unsigned)vecs * part / cluster), v1 = (int)((unsigned)vecs * (part + 1) / cluster);
    const uint4* zv = reinterpret_cast<const uint4*>(z + head);
    uint4 v[kVecs];
    auto load = [&](int k, int base) {  // vector k of this thread in the group at base
        const int i = base + k * kThreads + (int)threadIdx.x;
        if (base + (k + 1) * kThreads <= v1) v[k] = __ldcs(zv + i);  // (no thread is past the end)
        else v[k] = i < v1 ? __ldcs(zv + i) : make_uint4(V::kNone, V::kNone, V::kNone, V::kNone);
    };
#pragma unroll
    for (int k = 0; k < kVecs; ++k) load(k, v0);

    const int y = a.tok ? a.tok[row] : -1;
    const bool bad = y >= a.V, has = y >= 0 && !bad;
    const float zy = has ? V::one(z + y) : 0.f, fy = fmaxf(zy, -INFINITY);  // (NaN as -inf)
    // vectors before the token's: also logits equal to its
    const int yv = has ? (y - head < 0 ? -1 : (y - head) / V::kN) : -1;
    const float f_after = has ? fy : INFINITY, f_before = V::below(f_after);

    if (top) {
        if (threadIdx.x < 16) sh.edge[threadIdx.x] = 0;
        if (threadIdx.x < kMaxTop) sh.best[threadIdx.x] = 0;
        if (threadIdx.x == 0) sh.n = 0;
    }
    float m = -INFINITY, c = kLeast * kLog2e;
    F2 s(0.f, 0.f), t(0.f, 0.f);
    int rank = 0;
    // the row's ends outside the vectors (an element each for a few threads), and the token's own vector
    const int tail = head + vecs * V::kN;
    const int edge = (int)threadIdx.x < head ? (int)threadIdx.x : tail + (int)threadIdx.x - head;
    const bool has_edge = part == 0 && edge < a.V;
    const float ze = has_edge ? V::one(z + edge) : 0.f;
    const bool beside = part == 0 && has && threadIdx.x < V::kN && yv >= 0 && yv < vecs;
    const float zb = beside ? V::one(z + head + yv * V::kN + (int)threadIdx.x) : 0.f;

    // A group's vectors of a thread are a candidate where their largest logit reaches the threshold: in the first group
    // by (logit, index), later by being larger than thr.
    float thr = -INFINITY;
    bool have = false;
    const int rounds = min(kMaxTop / kWarps, (top + 4 + kWarps - 1) / kWarps);  // at least `top` numbers, a few more if there is room
    int group = 0;
    for (int base = v0; base < v1; base += kGroup, ++group) {
        typename V::Max vm;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) vm.add(v[k]);
        const float gm = vm.get();
        if (top) {
            bool in;
            if (group == 0) {
                uint64_t key = 0;  // 0: no vector
#pragma unroll
                for (int k = 0; k < kVecs; ++k) {
                    const int i = base + k * kThreads + (int)threadIdx.x;
                    typename V::Max x;
                    x.add(v[k]);
                    if (i < v1) key = max(key, key_of(x.get(), i));
                }
                const uint64_t b = top_th<uint64_t>(sh, key, rounds, top);
                have = b != 0;
                if (have) thr = value_of(b);
                in = key && key >= b;
            } else {
                in = gm > thr;
                if (group == 2 || group == 8 || group == 32) {  // (those that reach it may be this group's: not yet without equality)
                    thr = fmaxf(thr, value_of((uint64_t)top_th<uint32_t>(sh, ordered(fmaxf(m, gm)), rounds, top) << 32));
                    in = in && gm >= thr;
                }
            }
            if (in) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kList) sh.list[at] = base + (int)threadIdx.x;
            }
        }
        if (gm > m) {
            m = gm;
            const float n = fmaxf(m, kLeast) * kLog2e, d = c - n, f = ex2(d);
            t = fma2(s, F2(d, d), t) * F2(f, f);
            s = s * F2(f, f);
            c = n;
        }
        const F2 nc(-c, -c);
        typename V::Count cnt;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            if (base + k * kThreads >= v1) break;  // (nothing in it for any thread)
#pragma unroll
            for (int j = 0; j < kPairs; ++j) {
                const F2 w = fma2(V::pair(v[k], j), F2(kLog2e, kLog2e), nc), e(ex2(w.x()), ex2(w.y()));
                s = s + e;
                t = fma2(e, w, t);
            }
            cnt.add(v[k], base + k * kThreads + (int)threadIdx.x < yv ? f_before : f_after);
            load(k, base + kGroup);  // the next group's, where this one's was
        }
        rank += cnt.get();
    }
    if (has_edge) {
        if (top) sh.edge[threadIdx.x] = key_of(ze, edge);
        if (has) rank += edge < y ? !(fmaxf(ze, -INFINITY) < fy) : ze > fy;
        m = fmaxf(m, ze);
        const float n = fmaxf(m, kLeast) * kLog2e, d = c - n, f = ex2(d);
        const float w = fmaf(ze < kFloor ? kFloor : ze, kLog2e, -n), e = ex2(w);
        t = fma2(s, F2(d, d), t) * F2(f, f) + F2(e * w, 0.f);
        s = s * F2(f, f) + F2(e, 0.f);
        c = n;
    }
    if (beside) rank += head + yv * V::kN + (int)threadIdx.x < y && fmaxf(zb, -INFINITY) == fy;
    // ---- the block's sums and order
    Stats r{c, s.x() + s.y(), t.x() + t.y()};
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        r.join(Stats{__shfl_down_sync(0xffffffffu, r.c, o), __shfl_down_sync(0xffffffffu, r.s, o), __shfl_down_sync(0xffffffffu, r.t, o)});
        m = fmaxf(m, __shfl_down_sync(0xffffffffu, m, o));
    }
    if (has && fy == -INFINITY) {  // a token that is masked itself: every entry above -inf, and all before it
        rank = 0;
        for (int i = (int)threadIdx.x + kThreads * part; i < a.V; i += kThreads * cluster) rank += i < y || V::one(z + i) > fy;
    }
    rank = __reduce_add_sync(0xffffffffu, rank);
    if (lane == 0) {
        sh.stat[warp] = r;
        sh.max[warp] = m;
        sh.rank[warp] = rank;
    }
    __syncthreads();
    if (top) {
        const int listed = sh.n;
        __syncthreads();
        if (listed > kList) collect(sh, z, head, v0, v1, top);
        else settle<T, kVecs>(sh, z, head, v1, listed, top, have ? (uint64_t)ordered(thr) << 32 : (uint64_t)1);
    }
    // (the first warp alone: fewer instructions for the other rows' CTAs to wait behind)
    if (warp == 0) {
        r = sh.stat[0];
        m = sh.max[0];
        rank = sh.rank[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) {
            r.join(sh.stat[w]);
            m = fmaxf(m, sh.max[w]);
            rank += sh.rank[w];
        }
    }
    // ---- the cluster's, in its first CTA
    if (cluster > 1) {
        cg::cluster_group cl = cg::this_cluster();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
        Shared* first = cl.map_shared_rank(&sh, 0);
        if (threadIdx.x == 0) {
            first->gstat[part] = r;
            first->gmax[part] = m;
            first->grank[part] = rank;
        }
        if ((int)threadIdx.x < top) first->gather[part * top + threadIdx.x] = sh.best[threadIdx.x];
        cl.sync();
        if (part) return;
        if (top) {
            if ((int)threadIdx.x < cluster * top) sh.keys[threadIdx.x] = sh.gather[threadIdx.x];
            __syncthreads();
            select(sh, cluster * top, top);
        }
        if (warp == 0) {
            r = sh.gstat[0];
            m = sh.gmax[0];
            rank = sh.grank[0];
            for (int k = 1; k < cluster; ++k) {
                r.join(sh.gstat[k]);
                m = fmaxf(m, sh.gmax[k]);
                rank += sh.grank[k];
            }
        }
    }
    // ---- answers
    auto answer = [&](bool odd) {
        const float ls = isinf(m) ? NAN : odd ? logf(r.s) : log2f(r.s);
        auto log_p = [&](float x) { return odd ? x - m - ls : (fmaf(x, kLog2e, -r.c) - ls) * kLn2; };
        if (threadIdx.x == 0) {
            if (bad) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
            if (a.logprob) a.logprob[row] = y < 0 ? 0.f : bad ? NAN : log_p(zy);
            if (a.entropy) a.entropy[row] = odd ? ls - r.t / r.s : (ls - r.t / r.s) * kLn2;
            if (a.rank) a.rank[row] = has ? rank : -1;
        }
        if ((int)threadIdx.x < top) {
            const int id = index_of(sh.best[threadIdx.x]);
            if (a.ids) a.ids[(int64_t)row * top + threadIdx.x] = id;
            if (a.tops) a.tops[(int64_t)row * top + threadIdx.x] = log_p(value_of(sh.best[threadIdx.x]));
        }
    };
    const bool odd = fabsf(m) > kFar && !isinf(m);
    if (!__syncthreads_or(warp == 0 && odd)) {
        if (warp == 0) answer(false);
        return;
    }
    if (threadIdx.x == 0) sh.max[0] = m;
    __syncthreads();
    m = sh.max[0];
    slow_sums(sh, z, a.V, m, &r.s, &r.t);
    if (warp == 0) answer(true);
}

template <typename T>
int launch(const LogprobArgs& a, cudaStream_t stream) {
    // as many CTAs per row (a power of two) as keep the GPU's slots filled once, each with a few vectors per thread
    const int vecs = a.V / Vec<T>::kN;
    int cluster = 1;
    while (cluster < kMaxCluster && (int64_t)a.rows * cluster * 2 <= (int64_t)kCtasPerSm * forge_sm_count() &&
           vecs / (cluster * 2) >= 2 * kThreads)
        cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_logprobs<T>, a, cluster);
    return e == cudaSuccess ? 0 : forge_fail(-1, "forge_token_logprobs: launch failed: %s", cudaGetErrorString(e));
}
}  // namespace

extern "C" FORGE_API int forge_token_logprobs(const void* logits, int dtype, int64_t ld, int rows, int vocab,
                                              const int32_t* tokens, int n_top, float* logprob, float* entropy,
                                              int32_t* rank, int32_t* top_ids, float* top_logprobs, void* stream) {
    if (!logits || (dtype != FORGE_LOGITS_F32 && dtype != FORGE_LOGITS_BF16) || rows < 0 || vocab <= 0 || ld < vocab ||
        n_top < 0 || n_top > FORGE_LOGPROBS_MAX_TOP || n_top > vocab || (!tokens && (logprob || rank)) ||
        (n_top > 0 && !top_ids && !top_logprobs) || ((uintptr_t)logits & (dtype == FORGE_LOGITS_F32 ? 3 : 1)) ||
        rows > (1 << 27) || vocab > (1 << 30))
        return forge_fail(FORGE_INVALID_ARGS, "forge_token_logprobs: bad args (rows %d, vocab %d, ld %lld, n_top %d of at most %d)",
                          rows, vocab, (long long)ld, n_top, FORGE_LOGPROBS_MAX_TOP);
    if (rows == 0) return 0;
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_token_logprobs: no device");
    LogprobArgs a{logits, ld, vocab, n_top, rows, tokens, logprob, entropy, rank, top_ids, top_logprobs, err};
    return dtype == FORGE_LOGITS_F32 ? launch<float>(a, (cudaStream_t)stream) : launch<uint16_t>(a, (cudaStream_t)stream);
}
