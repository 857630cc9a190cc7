// Eviction from the key-value cache in pages by accumulated attention weight.
// Of a sequence longer than `keep`, every KV head keeps its first keys, its
// last ones and, of those between, the heaviest (total order of the weights,
// the lower index on ties); they move, in their order, to new pages.  Other
// sequences move whole.  Attention does not depend on the keys' order or
// places, so each KV head keeps keys of its own in the same pages.
#include <type_traits>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr uint32_t kSelBlock = 1024, kSelWaves = kSelBlock / 64;

// The kept keys of one KV head: a workgroup per sequence and head, that takes the
// weights in spans of 16,384, four times four to a thread; the first span's stay in
// registers from the first pass on, others are read again (from L2).
// The needed-th largest weight between the ends by counting passes over the key
// bits (11, 11 and 10), then the keys above it and the first of those equal to it,
// by a running count in index order: no atomics but the counts' own, so the same
// keys on every call.  A sequence with a length or page out of range keeps nothing.
// The length is read once a workgroup, and a place is compared with `keep` before it
// is written: weights or lengths that change meanwhile choose wrong keys, no more.
// One workgroup a head is simple and needs no workspace; a long history pays for it
// with all but a few compute units idle, and is bound by one unit's issue rate, some
// 20 operations a key, and by the steps between the passes: 51 us for 8,192 of 65,537
// keys (4 heads), 15 us for 1,024 of up to 4,096 (16 sequences).  Reading the next
// span ahead changes nothing; with every key's place looked at 62 and 17, with one
// copy of the counts and 8 rounds, whose weights do not fit the registers, 91 and 30.
constexpr uint32_t kSelPer = 4, kSelRound = kSelBlock * kSelPer, kSelRounds = 4, kSelSpan = kSelRound * kSelRounds;
constexpr uint32_t kBins = 2048, kCopies = 8;  // copies of a count, for lanes that hit the same one

// Inclusive scan over a wave.
template <typename T> __device__ __forceinline__ T scan_wave(T v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T t = __shfl_up(v, o, 64);
        if ((threadIdx.x & 63) >= (uint32_t)o) v += t;
    }
    return v;
}

__global__ __launch_bounds__(kSelBlock) void k_page_select(PageEvict a) {
    __shared__ __align__(16) uint32_t hist[kBins * kCopies];
    __shared__ uint32_t pick[2], part[kSelRounds * kSelWaves];
    __shared__ int32_t held;
    const uint32_t g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    if (tid == 0) held = length_of(a.r, b);
    __syncthreads();
    const int32_t len = held;
    uint32_t n = len < 0 ? 0u : (uint32_t)len, m = min(n, a.keep);
    const float* w = a.w + b * a.w_row + g * a.w_head;
    float x[kSelRounds][kSelPer];  // weights t0 + r kSelRound + 4 tid .. + 3
    auto load = [&](uint32_t t0) {
        typedef float four __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
        for (uint32_t r = 0; r < kSelRounds; r++) {
            const uint32_t t = t0 + r * kSelRound + tid * kSelPer;
            if (t + kSelPer <= n) {
                const four v = gld<four>(w + t);
                x[r][0] = v.x, x[r][1] = v.y, x[r][2] = v.z, x[r][3] = v.w;
            } else if (t < n) {
#pragma unroll
                for (uint32_t k = 0; k < kSelPer; k++) x[r][k] = gld<float>(w + min(t + k, n - 1));
            }
        }
    };
    load(0);
    int bad = len < 0;
    for (uint32_t i = tid; i * (uint64_t)a.c.page < n; i += kSelBlock)
        bad |= (uint32_t)gld<int32_t>(a.r.table + b * a.r.stride + i) >= a.c.count;
    for (uint32_t i = tid; i * (uint64_t)a.c.page < m; i += kSelBlock)
        bad |= (uint32_t)gld<int32_t>(a.to + b * a.to_stride + i) >= a.c.count;
    if (__syncthreads_or(bad)) n = m = 0;
    const size_t row = ((size_t)b * a.c.kvheads + g) * a.keep;
    if (g == 0 && tid == 0) a.length[b] = (int32_t)m;
    for (uint32_t j = m + tid; j < a.keep; j += kSelBlock) {
        a.kept[row + j] = -1;
        a.wout[row + j] = 0.f;
    }
    const bool longer = n > a.keep;
    const uint32_t lo = longer ? a.first : 0, hi = longer ? n - a.recent : 0;  // the keys to choose from
    uint32_t need = longer ? a.keep - a.first - a.recent : 0, cut = 0, known = 0;  // known: bits of cut
    const bool choose = need != 0;
    // f(whether all of round r's keys lie in [lo, hi)): most rounds', whose keys need no look at their place
    auto by_place = [&](uint32_t t0, uint32_t r, auto f) {
        const uint32_t from = t0 + r * kSelRound;
        if (from >= lo && from + kSelRound <= hi) f(std::true_type());
        else if (from < n) f(std::false_type());
    };
    for (uint32_t pass = 0; choose && pass < 3; pass++) {
        const uint32_t bits = pass < 2 ? 11 : 10, shift = 32 - known - bits, mask = (1u << bits) - 1;
        const uint32_t above = known ? ~0u << (32 - known) : 0;
        for (uint32_t i = tid; i < kBins * kCopies / 4; i += kSelBlock) ((uint4*)hist)[i] = make_uint4(0, 0, 0, 0);
        __syncthreads();
        for (uint32_t t0 = 0; t0 < n; t0 += kSelSpan) {
            if (n > kSelSpan && (pass || t0)) load(t0);
#pragma unroll
            for (uint32_t r = 0; r < kSelRounds; r++)
                by_place(t0, r, [&](auto inside) {
#pragma unroll
                    for (uint32_t k = 0; k < kSelPer; k++) {
                        const uint32_t t = t0 + r * kSelRound + tid * kSelPer + k, key = order_key(x[r][k]);
                        if ((key & above) == cut && (inside || (t >= lo && t < hi)))
                            atomicAdd(&hist[(key >> shift & mask) * kCopies + lane % kCopies], 1u);
                    }
                });
        }
        __syncthreads();
        // the digit that holds the need-th largest: two digits a thread, the largest first
        const uint32_t d = kBins - 1 - 2 * tid;
        auto count = [&](uint32_t digit) {
            const uint4 u = ((const uint4*)hist)[digit * 2], v = ((const uint4*)hist)[digit * 2 + 1];
            return u.x + u.y + u.z + u.w + (v.x + v.y + v.z + v.w);
        };
        static_assert(kCopies == 8, "two loads of four");
        const uint32_t c0 = count(d), c1 = count(d - 1);
        const uint32_t sum = scan_wave(c0 + c1);
        if (lane == 63) part[wv] = sum;
        __syncthreads();
        uint32_t before = sum - c0 - c1;
        for (uint32_t i = 0; i < wv; i++) before += part[i];
        if (before < need && before + c0 + c1 >= need) {
            const bool second = before + c0 < need;
            pick[0] = second ? d - 1 : d;
            pick[1] = need - before - (second ? c0 : 0);
        }
        __syncthreads();
        cut |= pick[0] << shift;
        need = pick[1];
        known += bits;
        __syncthreads();
    }
    // need: how many of the keys equal to cut stay
    const uint32_t above = choose ? cut : ~0u;  // no key is larger than the latter
    uint32_t sure0 = 0, equal0 = 0;  // of the spans before
    for (uint32_t t0 = 0; t0 < n; t0 += kSelSpan) {
        if (n > kSelSpan) load(t0);
        auto sort_of = [&](auto inside, uint32_t r, uint32_t k, bool& is_sure, bool& is_equal) {
            const uint32_t t = t0 + r * kSelRound + tid * kSelPer + k, key = order_key(x[r][k]);
            const bool mid = inside || (t >= lo && t < hi);
            is_sure = inside ? key > above : t < n && (!mid || key > above);
            is_equal = mid && choose && key == cut;
        };
        uint32_t upto[kSelRounds];  // of the wave: equal ones in the low half, sure ones in the high half
#pragma unroll
        for (uint32_t r = 0; r < kSelRounds; r++) {
            uint32_t mine = 0;
            by_place(t0, r, [&](auto inside) {
#pragma unroll
                for (uint32_t k = 0; k < kSelPer; k++) {
                    bool is_sure, is_equal;
                    sort_of(inside, r, k, is_sure, is_equal);
                    mine += (is_sure ? 1u << 16 : 0u) + is_equal;
                }
            });
            upto[r] = scan_wave(mine);
            if (lane == 63) part[r * kSelWaves + wv] = upto[r];
            upto[r] -= mine;
        }
        __syncthreads();
        // all rounds' and waves' counts, one a lane: a span's fit 16 bits each
        static_assert(kSelRounds * kSelWaves == 64 && kSelSpan < 65536, "a count a lane, 16 bits");
        const uint32_t mine = part[lane], sum = scan_wave(mine), all = __shfl(sum, 63, 64);
#pragma unroll
        for (uint32_t r = 0; r < kSelRounds; r++) {
            const uint32_t base = __shfl(sum - mine, r * kSelWaves + wv, 64) + upto[r];
            uint32_t ps = sure0 + (base >> 16), pe = equal0 + (base & 0xffff);
            by_place(t0, r, [&](auto inside) {
#pragma unroll
                for (uint32_t k = 0; k < kSelPer; k++) {
                    bool is_sure, is_equal;
                    sort_of(inside, r, k, is_sure, is_equal);
                    if (is_sure || (is_equal && pe < need)) {
                        const uint32_t j = ps + min(pe, need);
                        if (j < m) {
                            a.kept[row + j] = (int32_t)(t0 + r * kSelRound + tid * kSelPer + k);
                            a.wout[row + j] = x[r][k];
                        }
                    }
                    ps += is_sure;
                    pe += is_equal;
                }
            });
        }
        sure0 += all >> 16;
        equal0 += all & 0xffff;
        __syncthreads();
    }
}

// Moves the kept keys' rows: a workgroup per kMoveKeys of them, `lanes` lanes (a
// power of two) with B bytes each a row, K and V of several rows in flight.  B is
// 16 where rows are aligned so, else an element; the work is two dependent
// look-ups (kept, then the page; both compared with their ranges once more) and a copy, 8.0 us for 8,192 keys of four heads
// of 128 in f16 (33.5 MB moved, 4.2 TB/s) and 13.1 us for 16 sequences' 1,024;
// 13.8 and 27.6 with an element a lane.
template <uint32_t B> struct Bytes;
template <> struct Bytes<16> { typedef uint4 type; };
template <> struct Bytes<4> { typedef uint32_t type; };
template <> struct Bytes<2> { typedef uint16_t type; };
template <> struct Bytes<1> { typedef uint8_t type; };

template <uint32_t B> __global__ __launch_bounds__(kBlock) void k_page_move(PageEvict a, uint32_t row, uint32_t lanes) {
    typedef typename Bytes<B>::type word;
    constexpr uint32_t kAhead = 4;  // rows of a thread in flight
    __shared__ uint64_t src[kMoveKeys], dst[kMoveKeys];
    const uint32_t g = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, j0 = blockIdx.x * kMoveKeys;
    const uint32_t m = min((uint32_t)gld<int32_t>(a.length + b), a.keep), es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2;
    if (j0 >= m) return;
    const uint32_t n = min(kMoveKeys, m - j0);
    int bad = 0;
    if (tid < n) {
        const uint32_t j = j0 + tid, t = (uint32_t)gld<int32_t>(a.kept + ((size_t)b * a.c.kvheads + g) * a.keep + j);
        const uint32_t pt = t / a.c.page, pj = j / a.c.page;
        const uint32_t into = (uint32_t)gld<int32_t>(a.to + b * a.to_stride + pj);
        const uint32_t from = t < a.r.most ? (uint32_t)gld<int32_t>(a.r.table + b * a.r.stride + pt) : ~0u;
        bad = from >= a.c.count || into >= a.c.count;
        src[tid] = from * a.c.ps + (t - pt * a.c.page) * a.c.ts + g * a.c.hs;
        dst[tid] = into * a.c.ps + (j - pj * a.c.page) * a.c.ts + g * a.c.hs;
    }
    if (__syncthreads_or(bad)) return;  // only where what the choice was made from changed meanwhile
    const uint32_t c = tid % lanes, per = kBlock / lanes;
    for (uint32_t o = c * B; o < row; o += lanes * B)
        for (uint32_t i0 = tid / lanes; i0 < n; i0 += per * kAhead) {
            word k[kAhead], v[kAhead];
#pragma unroll
            for (uint32_t i = 0; i < kAhead; i++) {
                const size_t at = src[min(i0 + i * per, n - 1)] * es + o;
                k[i] = gld<word>(a.c.k + at);
                v[i] = gld<word>(a.c.v + at);
            }
#pragma unroll
            for (uint32_t i = 0; i < kAhead; i++) {
                if (i0 + i * per >= n) break;
                const size_t at = dst[i0 + i * per] * es + o;
                *reinterpret_cast<word*>(a.c.k + at) = k[i];
                *reinterpret_cast<word*>(a.c.v + at) = v[i];
            }
        }
    if (a.c.kind != Q8_0) return;
    const uint32_t blocks = a.c.dim / 32;
    for (uint32_t i = tid; i < n * blocks; i += kBlock) {
        const size_t from = src[i / blocks] / 32 + i % blocks, into = dst[i / blocks] / 32 + i % blocks;
        a.c.ks[into] = gld<_Float16>(a.c.ks + from);
        a.c.vs[into] = gld<_Float16>(a.c.vs + from);
    }
}

void launch_page_evict(const PageEvict& a, hipStream_t s) {
    hipLaunchKernelGGL(k_page_select, dim3(a.c.kvheads, a.r.batch), dim3(kSelBlock), 0, s, a);
    const uint32_t most = a.keep < a.r.most ? a.keep : a.r.most;
    if (!most) return;
    const uint32_t es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2, row = a.c.dim * es;
    const uint64_t all = ((uint64_t)a.c.ps | a.c.ts | a.c.hs) * es | row | (uintptr_t)a.c.k | (uintptr_t)a.c.v;
    const uint32_t wide = all % 16 ? es : 16;
    uint32_t lanes = 1;
    while (lanes < 64 && lanes * wide < row) lanes *= 2;
    const dim3 grid((most + kMoveKeys - 1) / kMoveKeys, a.c.kvheads, a.r.batch), block(kBlock);
    if (wide == 16) hipLaunchKernelGGL(k_page_move<16>, grid, block, 0, s, a, row, lanes);
    else if (wide == 4) hipLaunchKernelGGL(k_page_move<4>, grid, block, 0, s, a, row, lanes);
    else if (wide == 2) hipLaunchKernelGGL(k_page_move<2>, grid, block, 0, s, a, row, lanes);
    else hipLaunchKernelGGL(k_page_move<1>, grid, block, 0, s, a, row, lanes);
}

}  // namespace qh
