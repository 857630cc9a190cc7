// Eviction from the key-value cache in pages by accumulated attention weight.
// Of a sequence longer than `keep`, every KV head keeps its first keys, its
// last ones and, of those between, the heaviest (total order of the weights,
// the lower index on ties); they move, in their order, to new pages.  Other
// sequences move whole.  Attention does not depend on the keys' order or
// places, so each KV head keeps keys of its own in the same pages.
#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr uint32_t kSelBlock = 1024, kSelWaves = kSelBlock / 64;

// The kept keys of one KV head: a workgroup per sequence and head.
// The needed-th largest weight between the ends by four counting passes over
// the weights' key bytes, then the keys above it and the first of those equal
// to it, by a running count in index order: no atomics but the counts' own, so
// the same keys on every call.  A sequence with a length or page out of range
// keeps nothing.
__global__ __launch_bounds__(kSelBlock) void k_page_select(PageEvict a) {
    __shared__ uint32_t hist[256], cnt[2][kSelWaves], pick[2];
    const uint32_t g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int32_t len = length_of(a.r, b);
    uint32_t n = len < 0 ? 0u : (uint32_t)len, m = min(n, a.keep);
    int bad = len < 0;
    for (uint32_t i = tid; i * (uint64_t)a.c.page < n; i += kSelBlock)
        bad |= (uint32_t)gld<int32_t>(a.r.table + b * a.r.stride + i) >= a.c.count;
    for (uint32_t i = tid; i * (uint64_t)a.c.page < m; i += kSelBlock)
        bad |= (uint32_t)gld<int32_t>(a.to + b * a.to_stride + i) >= a.c.count;
    if (__syncthreads_or(bad)) n = m = 0;
    const float* w = a.w + b * a.w_row + g * a.w_head;
    const size_t row = ((size_t)b * a.c.kvheads + g) * a.keep;
    if (g == 0 && tid == 0) a.length[b] = (int32_t)m;
    for (uint32_t j = m + tid; j < a.keep; j += kSelBlock) {
        a.kept[row + j] = -1;
        a.wout[row + j] = 0.f;
    }
    const uint32_t lo = n > a.keep ? a.first : 0, hi = n > a.keep ? n - a.recent : 0;  // the keys to choose from
    uint32_t need = n > a.keep ? a.keep - a.first - a.recent : 0, cut = 0;
    if (need) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (uint32_t t = lo + tid; t < hi; t += kSelBlock) {
                const uint32_t k = order_key(gld<float>(w + t));
                if (shift == 24 || (k ^ cut) >> (shift + 8) == 0) atomicAdd(&hist[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t d = 255;
                while (hist[d] < need && d > 0) need -= hist[d--];
                pick[0] = d;
                pick[1] = need;
            }
            __syncthreads();
            cut |= pick[0] << shift;
            need = pick[1];
        }
    }
    // need: how many of the keys equal to cut stay (0: none between the ends)
    const bool choose = n > a.keep && a.keep > a.first + a.recent;
    uint32_t sure = 0, equal = 0;  // of the keys before this round's
    for (uint32_t t0 = 0; t0 < n; t0 += kSelBlock) {
        const uint32_t t = t0 + tid;
        const float x = t < n ? gld<float>(w + t) : 0.f;
        const uint32_t k = order_key(x);
        const bool mid = t >= lo && t < hi;
        const bool is_sure = t < n && (!mid || (choose && k > cut)), is_equal = mid && choose && k == cut;
        const uint64_t ms = __ballot(is_sure), me = __ballot(is_equal), below = ((uint64_t)1 << lane) - 1;
        if (lane == 0) {
            cnt[0][wv] = __popcll(ms);
            cnt[1][wv] = __popcll(me);
        }
        __syncthreads();
        uint32_t ps = sure + __popcll(ms & below), pe = equal + __popcll(me & below);
        for (uint32_t i = 0; i < kSelWaves; i++) {
            if (i < wv) ps += cnt[0][i], pe += cnt[1][i];
            sure += cnt[0][i];
            equal += cnt[1][i];
        }
        if (is_sure || (is_equal && pe < need)) {
            const uint32_t j = ps + min(pe, need);
            a.kept[row + j] = (int32_t)t;
            a.wout[row + j] = x;
        }
        __syncthreads();
    }
}

// Moves the kept keys' rows: a workgroup per kMoveKeys of them.
__global__ __launch_bounds__(kBlock) void k_page_move(PageEvict a) {
    const uint32_t g = blockIdx.y, b = blockIdx.z, d = a.c.dim;
    const int32_t* kept = a.kept + ((size_t)b * a.c.kvheads + g) * a.keep;
    const uint32_t m = (uint32_t)gld<int32_t>(a.length + b);
    const uint32_t es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2;
    for (uint32_t i = threadIdx.x >> 6; i < kMoveKeys; i += kWaves) {
        const uint32_t j = blockIdx.x * kMoveKeys + i;
        if (j >= m) return;
        const uint32_t t = (uint32_t)gld<int32_t>(kept + j);
        const uint32_t from = (uint32_t)gld<int32_t>(a.r.table + b * a.r.stride + t / a.c.page);
        const uint32_t into = (uint32_t)gld<int32_t>(a.to + b * a.to_stride + j / a.c.page);
        const size_t src = (size_t)from * a.c.ps + (size_t)(t % a.c.page) * a.c.ts + g * a.c.hs;
        const size_t dst = (size_t)into * a.c.ps + (size_t)(j % a.c.page) * a.c.ts + g * a.c.hs;
        for (uint32_t e = threadIdx.x & 63; e < d; e += 64) {
            if (es == 4) {
                reinterpret_cast<uint32_t*>(a.c.k)[dst + e] = gld<uint32_t>(a.c.k + 4 * (src + e));
                reinterpret_cast<uint32_t*>(a.c.v)[dst + e] = gld<uint32_t>(a.c.v + 4 * (src + e));
            } else if (es == 2) {
                reinterpret_cast<uint16_t*>(a.c.k)[dst + e] = gld<uint16_t>(a.c.k + 2 * (src + e));
                reinterpret_cast<uint16_t*>(a.c.v)[dst + e] = gld<uint16_t>(a.c.v + 2 * (src + e));
            } else {
                a.c.k[dst + e] = gld<uint8_t>(a.c.k + src + e);
                a.c.v[dst + e] = gld<uint8_t>(a.c.v + src + e);
                if (e % 32 == 0) {
                    reinterpret_cast<uint16_t*>(a.c.ks)[(dst + e) / 32] = gld<uint16_t>(a.c.ks + (src + e) / 32);
                    reinterpret_cast<uint16_t*>(a.c.vs)[(dst + e) / 32] = gld<uint16_t>(a.c.vs + (src + e) / 32);
                }
            }
        }
    }
}

void launch_page_evict(const PageEvict& a, hipStream_t s) {
    hipLaunchKernelGGL(k_page_select, dim3(a.c.kvheads, a.r.batch), dim3(kSelBlock), 0, s, a);
    const uint32_t most = a.keep < a.r.most ? a.keep : a.r.most;
    if (most)
        hipLaunchKernelGGL(k_page_move, dim3((most + kMoveKeys - 1) / kMoveKeys, a.c.kvheads, a.r.batch), dim3(kBlock), 0,
                           s, a);
}

}  // namespace qh
