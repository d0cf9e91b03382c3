// logprobs.cu — log probabilities of given tokens, entropy, rank and the top
// alternatives of logits rows.
#include <cmath>
#include "common.cuh"
#include "forge_internal.h"
#include "../../include/forge_b200.h"

namespace {
struct LogprobArgs {
    const void* z;
    int64_t ld;
    int V, top;
    const int32_t* tok;
    float *logprob, *entropy;
    int32_t *rank, *ids;
    float* tops;
    uint32_t* err;
};

__device__ float logit(const float* z, int i) { return z[i]; }
__device__ float logit(const uint16_t* z, int i) { return bf16_bits_to_f32(z[i]); }
// Order of the logits as an unsigned number: NaN as -inf, -0 as 0.
__device__ uint32_t ordered(float x) {
    if (isnan(x)) x = -INFINITY;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

// One warp per row.
template <typename T>
__global__ void __launch_bounds__(32) k_logprobs(const LogprobArgs a) {
    const int r = blockIdx.x, lane = threadIdx.x;
    const T* z = (const T*)a.z + (int64_t)r * a.ld;
    float m = -INFINITY;
    bool nan = false;
    for (int i = lane; i < a.V; i += 32) { m = fmaxf(m, logit(z, i)); nan |= isnan(logit(z, i)); }
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    nan = __any_sync(0xffffffffu, nan);
    const int y = a.tok ? a.tok[r] : -1;
    const bool bad = y >= a.V;
    const float zy = y >= 0 && !bad ? logit(z, y) : 0.f;
    const uint64_t ky = (uint64_t)ordered(zy) << 32 | (uint32_t)~y;
    float s = 0.f, t = 0.f;
    int rank = 0;
    for (int i = lane; i < a.V; i += 32) {
        const float d = logit(z, i) - m, e = expf(d);
        s += e;
        t += d == -INFINITY ? 0.f : e * d;
        rank += ((uint64_t)ordered(logit(z, i)) << 32 | (uint32_t)~i) > ky;
    }
    for (int o = 16; o; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
        rank += __shfl_xor_sync(0xffffffffu, rank, o);
    }
    const float ls = nan || isinf(m) ? NAN : logf(s);
    if (lane == 0) {
        if (bad) atomicOr(a.err, FORGE_DEVERR_BAD_INDEX);
        if (a.logprob) a.logprob[r] = y < 0 ? 0.f : bad ? NAN : zy - m - ls;
        if (a.entropy) a.entropy[r] = ls - t / s;
        if (a.rank) a.rank[r] = y < 0 || bad ? -1 : rank;
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        uint64_t best = 0;
        for (int i = lane; i < a.V; i += 32) {
            const uint64_t key = (uint64_t)ordered(logit(z, i)) << 32 | (uint32_t)~i;
            if (key < last && key > best) best = key;
        }
        for (int o = 16; o; o >>= 1) {
            const uint64_t u = __shfl_xor_sync(0xffffffffu, best, o);
            best = u > best ? u : best;
        }
        last = best;
        const int id = (int)~(uint32_t)best;
        if (lane == 0 && a.ids) a.ids[(int64_t)r * a.top + k] = id;
        if (lane == 0 && a.tops) a.tops[(int64_t)r * a.top + k] = logit(z, id) - m - ls;
    }
}
}  // namespace

extern "C" FORGE_API int forge_token_logprobs(const void* logits, int dtype, int64_t ld, int rows, int vocab,
                                              const int32_t* tokens, int n_top, float* logprob, float* entropy,
                                              int32_t* rank, int32_t* top_ids, float* top_logprobs, void* stream) {
    if (!logits || (dtype != FORGE_LOGITS_F32 && dtype != FORGE_LOGITS_BF16) || rows < 0 || vocab <= 0 || ld < vocab ||
        n_top < 0 || n_top > FORGE_LOGPROBS_MAX_TOP || n_top > vocab || (!tokens && (logprob || rank)) ||
        (n_top > 0 && !top_ids && !top_logprobs) || ((uintptr_t)logits & (dtype == FORGE_LOGITS_F32 ? 3 : 1)))
        return forge_fail(FORGE_INVALID_ARGS, "forge_token_logprobs: bad args (rows %d, vocab %d, ld %lld, n_top %d of at most %d)",
                          rows, vocab, (long long)ld, n_top, FORGE_LOGPROBS_MAX_TOP);
    if (rows == 0) return 0;
    uint32_t* err = forge_ops_err_word();
    if (!err) return forge_fail(-1, "forge_token_logprobs: no device");
    LogprobArgs a{logits, ld, vocab, n_top, tokens, logprob, entropy, rank, top_ids, top_logprobs, err};
    if (dtype == FORGE_LOGITS_F32) k_logprobs<float><<<rows, 32, 0, (cudaStream_t)stream>>>(a);
    else k_logprobs<uint16_t><<<rows, 32, 0, (cudaStream_t)stream>>>(a);
    return forge_check_launch("forge_token_logprobs");
}
