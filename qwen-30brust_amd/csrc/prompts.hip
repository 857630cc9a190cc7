// Attention of several new tokens per sequence over the key-value cache in
// pages: whole prompts, pieces of them and single tokens (causal), and trees of
// drafted tokens.
#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

// Sequence b's new tokens: rows [f0, f0 + count), of `len` keys in all; bad: its
// rows become NaN.
struct Seq {
    uint32_t f0, count;
    int32_t len;
    bool bad;
};
__device__ __forceinline__ Seq seq_of(const PageMany& a, uint32_t b) {
    const int32_t f = gld<int32_t>(a.first + b), e = gld<int32_t>(a.first + b + 1), len = length_of(a.r, b);
    const bool rows = f >= 0 && f <= e && (uint32_t)e <= a.n;
    const uint32_t count = rows ? (uint32_t)(e - f) : 0;
    const bool bad = len < 0 || count > (uint32_t)len || (a.seen && count > kTreeMost);
    return {rows ? (uint32_t)f : 0, count, len, bad};
}

// A wave per row and head: a key at a time, its dot product over the lanes.
__global__ __launch_bounds__(kBlock) void k_page_many(PageMany a) {
    constexpr uint32_t E = kPageMaxDim / 64;
    const uint32_t lane = threadIdx.x & 63, d = a.c.dim, h = blockIdx.y, b = blockIdx.z;
    const uint32_t g = h / (a.heads / a.c.kvheads);
    const Seq s = seq_of(a, b);
    for (uint32_t i = blockIdx.x * kWaves + (threadIdx.x >> 6); i < s.count; i += gridDim.x * kWaves) {
        const uint32_t row = s.f0 + i;
        float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < E; j++) {
            const uint32_t e = lane + 64 * j;
            q[j] = e < d ? elem_kind(a.q.kind, a.q.p, row * a.q.row + h * a.q.head + e) : 0.f;
            o[j] = 0.f;
        }
        const uint32_t c0 = s.bad ? 0 : (uint32_t)s.len - s.count;
        const uint32_t end = s.bad ? 0 : a.seen ? (uint32_t)s.len : c0 + i + 1;
        const uint64_t bits = a.seen ? gld<uint64_t>(a.seen + row) : 0;
        bool bad = s.bad;
        for (uint32_t t = 0; t < end; t++) {
            const int32_t page = gld<int32_t>(a.r.table + b * a.r.stride + t / a.c.page);
            if ((uint32_t)page >= a.c.count) {
                bad = true;
                break;
            }
            if (a.seen && t >= c0 && !(bits >> (t - c0) & 1)) continue;
            const size_t at = (size_t)page * a.c.ps + (size_t)(t % a.c.page) * a.c.ts + g * a.c.hs;
            auto value = [&](const uint8_t* p, const _Float16* sc, size_t e) {
                return a.c.kind == Q8_0 ? elem<Q8_0>(p, e) * (float)gld<_Float16>(sc + e / 32) : elem_kind(a.c.kind, p, e);
            };
            float x = 0.f;
#pragma unroll
            for (uint32_t j = 0; j < E; j++)
                if (lane + 64 * j < d) x = fmaf(q[j], value(a.c.k, a.c.ks, at + lane + 64 * j), x);
            x = wave_sum(x) * a.scale;
            const float M = fmaxf(m, x), f = M == -INFINITY ? 0.f : M;
            const float was = expf(m - f), p = expf(x - f);
            m = M;
            l = l * was + p;
#pragma unroll
            for (uint32_t j = 0; j < E; j++)
                if (lane + 64 * j < d) o[j] = fmaf(p, value(a.c.v, a.c.vs, at + lane + 64 * j), o[j] * was);
        }
#pragma unroll
        for (uint32_t j = 0; j < E; j++)
            if (lane + 64 * j < d)
                put_kind(a.out.kind, a.out.p, row * a.out.row + h * a.out.head + lane + 64 * j,
                         bad ? __builtin_nanf("") : l == 0.f ? 0.f : o[j] / l);
    }
}

void launch_page_many(const PageMany& a, hipStream_t s) {
    const uint32_t x = (a.n + kWaves - 1) / kWaves;
    hipLaunchKernelGGL(k_page_many, dim3(x < 64 ? x : 64, a.heads, a.r.batch), dim3(kBlock), 0, s, a);
}

}  // namespace qh
