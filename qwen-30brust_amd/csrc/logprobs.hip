// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits, with the padding-vocabulary mask of src/main.rs:262-266 (masked
// ids read as f32::MIN, as the sampler reads them):
//   m = max x,  S = sum exp(x - m),  log p_t = x_t - m - log S,
//   H = log S - sum (x - m) exp(x - m) / S
// in 32 bits.  The alternatives are in descending total order, the lower id on
// ties.  A row that holds NaN or +inf gives NaN; one of -inf alone gives -inf
// and no entropy; a target outside the vocabulary gives NaN.
#include <cfloat>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr uint32_t kLpBlock = 1024, kLpWaves = kLpBlock / 64;

__device__ __forceinline__ float logit(const Logprobs& a, const uint8_t* row, uint32_t i) {
    return a.valid && !gld<uint8_t>(a.valid + i) ? -FLT_MAX : elem_kind(a.kind, row, i);
}

// One row per workgroup: a pass each for the maximum, the sums and every
// alternative (the largest below the one before).
__global__ __launch_bounds__(kLpBlock) void k_logprobs(Logprobs a) {
    __shared__ float red[2][kLpWaves];
    __shared__ uint64_t best[kLpWaves];
    const uint32_t r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const uint32_t es = a.kind == F32 ? 4 : 2;
    const uint8_t* row = static_cast<const uint8_t*>(a.x) + r * a.stride * es;
    float m = -INFINITY;
    int bad = 0;
    for (uint32_t i = tid; i < a.vocab; i += kLpBlock) {
        const float x = logit(a, row, i);
        bad |= !(x < INFINITY);
        m = fmaxf(m, x);
    }
    m = wave_max(m);
    if (lane == 0) red[0][wv] = m;
    bad = __syncthreads_or(bad);
    for (uint32_t i = 0; i < kLpWaves; i++) m = fmaxf(m, red[0][i]);
    __syncthreads();
    float S = 0.f, U = 0.f;
    for (uint32_t i = tid; i < a.vocab; i += kLpBlock) {
        const float x = logit(a, row, i), e = x == -INFINITY ? 0.f : expf(x - m);
        S += e;
        if (e > 0.f) U = fmaf(x - m, e, U);
    }
    S = wave_sum(S);
    U = wave_sum(U);
    if (lane == 0) {
        red[0][wv] = S;
        red[1][wv] = U;
    }
    __syncthreads();
    S = U = 0.f;
    for (uint32_t i = 0; i < kLpWaves; i++) {
        S += red[0][i];
        U += red[1][i];
    }
    const float logS = logf(S);
    auto logp = [&](float x) { return bad ? __builtin_nanf("") : x == -INFINITY ? x : x - m - logS; };
    if (tid == 0) {
        if (a.logp) {
            const uint32_t t = (uint32_t)gld<int32_t>(a.target + r);
            a.logp[r] = t < a.vocab ? logp(logit(a, row, t)) : __builtin_nanf("");
        }
        if (a.entropy) a.entropy[r] = bad ? __builtin_nanf("") : S > 0.f ? logS - U / S : 0.f;
    }
    uint64_t last = ~(uint64_t)0;
    for (uint32_t j = 0; j < a.top; j++) {
        uint64_t top = 0;
        for (uint32_t i = tid; i < a.vocab; i += kLpBlock) {
            const uint64_t c = (uint64_t)order_key(logit(a, row, i)) << 32 | (uint32_t)~i;
            if (c < last && c > top) top = c;
        }
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint64_t)__shfl_xor((unsigned long long)top, o, 64));
        __syncthreads();
        if (lane == 0) best[wv] = top;
        __syncthreads();
        for (uint32_t i = 0; i < kLpWaves; i++) top = max(top, best[i]);
        last = top;
        if (tid == 0) {
            a.ids[(size_t)r * a.top + j] = (int32_t) ~(uint32_t)top;
            a.alt[(size_t)r * a.top + j] = logp(key_value((uint32_t)(top >> 32)));
        }
    }
}

size_t logprobs_bytes(uint32_t, uint32_t, uint32_t) { return 0; }

void launch_logprobs(const Logprobs& a, hipStream_t s) {
    hipLaunchKernelGGL(k_logprobs, dim3(a.rows), dim3(kLpBlock), 0, s, a);
}

}  // namespace qh
