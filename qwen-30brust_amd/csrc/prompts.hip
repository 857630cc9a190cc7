// Attention of several new tokens per sequence over the key-value cache in
// pages: whole prompts, pieces of them and single tokens (causal), and trees of
// drafted tokens.
//   s_t = scale * log2(e) * q . k_t,  o = sum 2^(s_t - m) v_t / sum 2^(s_t - m)
// over the keys t that a row sees.
//
// The query heads of a KV head read the same keys, so a sequence's rows of one KV
// head are (token, head) pairs, a token's heads beside each other, in tiles of 128.
// A tile's keys are those that its last row sees.  The work of all tiles, in keys, one
// tile behind the other, is dealt to the workgroups in equal runs, whatever the
// lengths: few rows over a long context, many short prompts and one long prompt all
// fill the chip.  A run may hold several tiles; one that it holds whole goes straight
// to out, and of the first and the last it may hold a part: its (m, l, o) go to the
// workgroup's two slots, and k_page_many_join folds them.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kTileRows = 128;  // query rows of a tile, 32 a wave
constexpr uint32_t kRunKeys = 128;   // keys of a run at least
constexpr uint32_t kXcds = 8;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef bf16_t b2 __attribute__((ext_vector_type(2)));
typedef bf16_t b8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t same64(uint64_t v) { return (uint64_t)same((uint32_t)(v >> 32)) << 32 | same((uint32_t)v); }
// The values of lanes l and l ^ 32.
__device__ __forceinline__ float2 halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// ------------------------------------------------------------ runs of work --
// Sequence b's new tokens are rows [f0, f0 + count) of q; c0 keys lie in front of
// them.  Its tiles of one KV head: tile i costs first + i * step, in keys times the
// query heads of a KV head; a tree's rows all go to its end.  bad: the rows become NaN.
struct Seq {
    uint32_t f0, count, c0, tiles;
    int32_t len;
    bool bad;
    uint64_t first, step;
    __device__ __forceinline__ uint64_t upto(uint32_t i) const { return first * i + step * ((uint64_t)i * (i - 1) / 2); }
    __device__ __forceinline__ uint64_t cost(uint32_t i) const { return first + step * i; }
};
struct Bounds {
    int32_t f, e, len;  // rows [f, e), keys or -1
};
__device__ __forceinline__ Bounds bounds_of(const PageMany& a, uint32_t b) {
    return {gld<int32_t>(a.first + b), gld<int32_t>(a.first + b + 1), length_of(a.r, b)};
}
__device__ __forceinline__ Seq seq_of(const PageMany& a, const Bounds& q) {
    Seq s{};
    const int32_t f = q.f, e = q.e;
    s.len = q.len;
    if (f < 0 || f > e || (uint32_t)e > a.n) return s;
    s.f0 = (uint32_t)f;
    s.count = (uint32_t)(e - f);
    s.tiles = (uint32_t)(((uint64_t)s.count * a.group + kTileRows - 1) / kTileRows);
    s.bad = s.len < 0 || s.count > (uint32_t)s.len || (a.seen && s.count > kTreeMost);
    s.c0 = s.bad ? 0 : (uint32_t)s.len - s.count;
    s.first = s.bad ? 1 : a.seen ? (uint64_t)(uint32_t)s.len * a.group : (uint64_t)(s.c0 + 1) * a.group + kTileRows - 1;
    s.step = s.bad || a.seen ? 0 : kTileRows;
    return s;
}
// Behind the last key of tile i.
__device__ __forceinline__ uint32_t end_of(const PageMany& a, const Seq& s, uint32_t i) {
    if (s.bad) return 0;
    if (a.seen) return (uint32_t)s.len;
    return s.c0 + min(i * kTileRows + kTileRows - 1, s.count * a.group - 1) / a.group + 1;
}
// The key at which the part from x on of a tile begins: at whole steps.
__device__ __forceinline__ uint32_t key_at(const PageMany& a, uint64_t x, uint32_t end, uint32_t step) {
    return (uint32_t)min((uint64_t)end, x / a.group / step * step);
}

__device__ __forceinline__ uint64_t run_begin(uint64_t total, uint32_t runs, uint32_t i) {
    return total / runs * i + min((uint64_t)i, total % runs);
}

// What the join has to know of the tile that a run begins inside of.
struct ManyMark {
    uint64_t at, cost;            // the tile's own place and cost; cost 0: the run begins with a tile
    uint32_t row, rows, kv, end;  // its first row (times the group), rows, KV head, keys
};
struct ManyHead {
    uint64_t total;
    uint32_t runs, pad;
};
size_t page_many_bytes(const PageMany& a) {
    const size_t slots = (size_t)a.runs * 2 * kTileRows;
    return slots * a.wide * 4 + slots * 8 + sizeof(ManyHead) + a.runs * sizeof(ManyMark);
}
__device__ __forceinline__ float* part_o(const PageMany& a, size_t slot) { return (float*)a.work + slot * kTileRows * a.wide; }
__device__ __forceinline__ float2* part_ml(const PageMany& a, size_t slot) {
    return (float2*)((float*)a.work + (size_t)a.runs * 2 * kTileRows * a.wide) + slot * kTileRows;
}
__device__ __forceinline__ ManyHead* head_of(const PageMany& a) { return (ManyHead*)part_ml(a, (size_t)a.runs * 2); }
__device__ __forceinline__ ManyMark* mark_of(const PageMany& a, uint32_t run) { return (ManyMark*)(head_of(a) + 1) + run; }

// A workgroup's run.
struct Run {
    uint64_t x, end;  // places
    uint32_t run, b, kv, i;
    uint64_t off;     // within the tile in hand
    Seq s;
    // Sequence b, read once for the workgroup: all its threads go one way whatever
    // becomes of the lengths.
    __device__ __forceinline__ void read(const PageMany& a) {
        __shared__ Bounds q;
        __syncthreads();
        if (threadIdx.x == 0) q = bounds_of(a, b);
        __syncthreads();
        s = seq_of(a, {(int32_t)same(q.f), (int32_t)same(q.e), (int32_t)same(q.len)});
    }
    // Finds it from the lengths; every loop ends with the batch.  Lengths that change
    // meanwhile give a wrong result, no more.
    __device__ __forceinline__ bool start(const PageMany& a) {
        __shared__ uint64_t part[kWaves];
        __shared__ uint64_t found[2];
        const uint32_t tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, G = a.c.kvheads;
        auto cost = [&](uint32_t j) {
            if (j >= a.r.batch) return (uint64_t)0;
            const Seq q = seq_of(a, bounds_of(a, j));
            return G * q.upto(q.tiles);
        };
        const uint64_t mine = cost(tid);
        uint64_t sum = mine;
        for (uint32_t j = tid + kBlock; j < a.r.batch; j += kBlock) sum += cost(j);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor((unsigned long long)sum, o, 64);
        if (lane == 0) part[wv] = sum;
        if (tid == 0) found[0] = ~0ull;
        __syncthreads();
        uint64_t total = 0;
        for (uint32_t w = 0; w < kWaves; w++) total += part[w];
        total = same64(total);
        const uint32_t runs = (uint32_t)max((uint64_t)1, min((uint64_t)a.runs, total / (kRunKeys * (uint64_t)a.group)));
        if (blockIdx.x == 0 && tid == 0) *head_of(a) = {total, total ? runs : 0, 0};
        // runs that lie beside each other, and read the same keys, on one XCD
        const uint32_t per = (runs + kXcds - 1) / kXcds;
        run = blockIdx.x % kXcds * per + blockIdx.x / kXcds;
        if (!total || blockIdx.x / kXcds >= per || run >= runs) return false;
        x = run_begin(total, runs, run);
        end = run_begin(total, runs, run + 1);
        if (tid == 0) mark_of(a, run)->cost = 0;
        uint64_t base = 0;
        for (uint32_t j = 0; j < a.r.batch; j += kBlock) {
            const uint64_t c = j ? cost(j + tid) : mine;
            uint64_t upto = c;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint64_t t = __shfl_up((unsigned long long)upto, o, 64);
                if (lane >= (uint32_t)o) upto += t;
            }
            __syncthreads();
            if (lane == 63) part[wv] = upto;
            __syncthreads();
            uint64_t all = 0;
            for (uint32_t w = 0; w < kWaves; w++) {
                if (w == wv) upto += base + all;
                all += part[w];
            }
            if (upto > x && upto - c <= x) found[0] = j + tid, found[1] = upto - c;
            __syncthreads();
            if (found[0] != ~0ull) break;
            base += all;
        }
        if (found[0] == ~0ull) return false;
        b = same((uint32_t)found[0]);
        read(a);
        const uint64_t each = same64(s.upto(s.tiles)), in = same64(x - found[1]);
        if (!each) return false;
        kv = (uint32_t)(in / each);
        off = in - kv * each;
        if (kv >= G) return false;
        uint32_t lo = 0, hi = s.tiles;  // the last tile whose place is not behind off
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (s.upto(mid) <= off) lo = mid;
            else hi = mid;
        }
        i = lo;
        off -= s.upto(lo);
        if (off && tid == 0)
            *mark_of(a, run) = {x - off, s.cost(i), s.f0 * a.group + i * kTileRows,
                                min(kTileRows, s.count * a.group - i * kTileRows), kv, end_of(a, s, i)};
        return true;
    }
    __device__ __forceinline__ uint64_t here() const { return min(s.cost(i) - off, end - x); }
    __device__ __forceinline__ bool next(const PageMany& a) {
        x += here();
        if (x >= end) return false;
        off = 0;
        if (++i < s.tiles) return true;
        i = 0;
        if (++kv < a.c.kvheads) return true;
        kv = 0;
        do {
            if (++b >= a.r.batch) return false;
            read(a);
        } while (!s.tiles);
        return true;
    }
};

// --------------------------------------------------------------- the tiles --
// Four consecutive values of a row of out.
__device__ __forceinline__ void put_row(const PageMany& a, uint32_t dim, uint32_t row, uint32_t h, uint32_t d, f4 x) {
    const size_t at = (size_t)row * a.out.row + (size_t)h * a.out.head + d;
    if (a.out_wide && d + 4 <= dim) {
        if (a.out.kind == F32) *reinterpret_cast<f4*>(a.out.p + 4 * at) = x;
        else if (a.out.kind == F16) *reinterpret_cast<__attribute__((ext_vector_type(4))) _Float16*>(a.out.p + 2 * at) = __builtin_convertvector(x, __attribute__((ext_vector_type(4))) _Float16);
        else *reinterpret_cast<__attribute__((ext_vector_type(4))) bf16_t*>(a.out.p + 2 * at) = __builtin_convertvector(x, __attribute__((ext_vector_type(4))) bf16_t);
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
        if (d + j < dim) put_kind(a.out.kind, a.out.p, at + j, x[j]);
}

// The 16-byte chunk of a tile's row that chunk c lies in: rows that are read together
// are spread over the banks (K: 32 rows a read at one chunk, 8 of them a cycle; V: four
// rows at four chunks).
template <uint32_t CH> __device__ __forceinline__ constexpr uint32_t turn(uint32_t row) {
    return CH >= 16 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

// T: type of the products; D: width of the tiles, at least the heads'; DIRECT: the
// cache's rows are T, D wide and aligned to 16 bytes, and go to LDS by themselves.
//
// A wave has 32 query rows.  It takes the scores as K Q^T, so that a lane has one
// row's scores (of the keys 8 i + 4 (lane / 32) + j), its maximum and sum need one
// exchange, and the weights lie where O^T = V^T P^T wants its second operand: for 16-bit
// types keys 16 c + 8 (e / 4) + 4 (lane / 32) + e % 4 are element e, for V^T read by the
// transposing LDS read.  K and V of the next step come in while one is worked on.
template <class T, uint32_t D, bool DIRECT>
__global__ __launch_bounds__(kBlock, D == 256 ? 1 : 2) void k_page_many(PageMany a) {
    constexpr bool F = std::is_same<T, float>::value, H = std::is_same<T, _Float16>::value;
    constexpr uint32_t KT = F || D == 256 ? 32 : 64;  // keys of a step
    constexpr uint32_t NS = KT / 32, ND = D / 32, CH = D * sizeof(T) / 16;
    constexpr uint32_t NQ = F ? D / 2 : D / 16;
    // weights are at most 2^(kAhead + kUp), so that f16 holds them and small ones too
    constexpr float kAhead = 8.f, kUp = H ? 7.f : 0.f;
    typedef typename std::conditional<H, h8, b8>::type T8;
    typedef typename std::conditional<F, float, T8>::type Q;
    __shared__ __align__(16) uint8_t ks[2][KT * D * sizeof(T)], vs[2][KT * D * sizeof(T)];
    __shared__ uint32_t bad_at;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wv = same(tid >> 6), n = lane & 31, half = lane >> 5;
    Run run;
    if (!run.start(a)) return;
    do {
        const Seq& s = run.s;
        const uint32_t end = same(end_of(a, s, run.i)), R = s.count * a.group;
        const uint32_t lo = same(key_at(a, run.off, end, KT));
        const bool whole = run.off == 0 && run.here() == s.cost(run.i);
        const uint32_t hi = same(run.off + run.here() == s.cost(run.i) ? end : key_at(a, run.off + run.here(), end, KT));
        const uint32_t r0 = run.i * kTileRows + wv * 32, r = r0 + n;  // rows of the sequence and KV head
        const bool mine = r < R;
        // hidden from the optimiser, that it keeps no comparison with it over the whole loop
        uint32_t dim = a.c.dim;
        asm volatile("" : "+s"(dim));
        const uint32_t token = mine ? r / a.group : 0, row = s.f0 + token, h = run.kv * a.group + (mine ? r % a.group : 0);
        if (s.bad) {
            if (run.off == 0 && mine)
                for (uint32_t d = half * 4; d < dim; d += 8) put_row(a, dim, row, h, d, f4(__builtin_nanf("")));
            continue;
        }
        if (lo >= hi) continue;
        // keys that all of the wave's rows see, and behind the last that one sees
        const uint32_t all = r0 >= R ? 0 : a.seen ? s.c0 : s.c0 + r0 / a.group + 1;
        const uint32_t most = r0 >= R ? 0 : a.seen ? end : s.c0 + min(r0 + 31, R - 1) / a.group + 1;
        const uint32_t own = a.seen ? end : s.c0 + token + 1;  // behind this row's last
        uint64_t bits = 0;
        if (a.seen && mine) bits = gld<uint64_t>(a.seen + row) & (s.count == 64 ? ~0ull : (1ull << s.count) - 1);

        Q q[NQ];
        {
            const size_t at = (size_t)row * a.q.row + (size_t)h * a.q.head;
            if constexpr (F) {
                auto load = [&](auto kind) {
#pragma unroll
                    for (uint32_t g = 0; g < D / 8; g++)
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) {
                            const uint32_t d = 8 * g + 4 * half + j;
                            q[4 * g + j] = mine && d < dim ? elem<kind()>(a.q.p, at + d) * a.sign : 0.f;
                        }
                };
                if (a.q.kind == F16) load(std::integral_constant<uint32_t, F16>());
                else if (a.q.kind == BF16) load(std::integral_constant<uint32_t, BF16>());
                else if (!a.q_wide) load(std::integral_constant<uint32_t, F32>());
                else {
#pragma unroll
                    for (uint32_t g = 0; g < D / 8; g++) {
                        const uint32_t d = 8 * g + 4 * half;
                        f4 x = {0.f, 0.f, 0.f, 0.f};
                        if (mine && d < dim) x = gld<f4>(a.q.p + 4 * (at + d)) * a.sign;
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) q[4 * g + j] = x[j];
                    }
                }
            } else {
                const uint32_t flip = a.sign < 0.f ? 0x80008000u : 0u, keep = a.sign == 0.f ? 0u : ~0u;
#pragma unroll
                for (uint32_t g = 0; g < D / 16; g++) {
                    const uint32_t d = 16 * g + 8 * half;
                    u4 x = {0, 0, 0, 0};
                    if (a.q_wide) {
                        if (mine && d < dim) x = gld<u4>(a.q.p + 2 * (at + d));
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 8; j++)
                            if (mine && d + j < dim) x[j / 2] |= (uint32_t)gld<uint16_t>(a.q.p + 2 * (at + d + j)) << 16 * (j & 1);
                    }
                    q[g] = __builtin_bit_cast(T8, (x ^ flip) & keep);
                }
            }
        }
        f16v o[ND];
#pragma unroll
        for (uint32_t d = 0; d < ND; d++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[d][j] = 0.f;
        float M = -INFINITY, L = 0.f;
        // the first step with a value that is not finite beside keys that some row does not
        // see: 0 times it is no 0, so from there on the products are taken key by key, below
        uint32_t odd = ~0u;
        uint32_t bad = ~0u;  // the first key that this lane found in a page out of range

        // ---- a step's K and V
        const int32_t* table = a.r.table + run.b * a.r.stride;
        const size_t base = run.kv * a.c.hs;
        auto place = [&](uint32_t t, int32_t page) {  // of key t; a page out of range is read as page 0
            const uint32_t in = t - (uint32_t)(((uint64_t)t * a.page_mul) >> a.page_shift) * a.c.page;
            if ((uint32_t)page >= a.c.count) bad = min(bad, t), page = 0;
            return (size_t)page * a.c.ps + (size_t)in * a.c.ts + base;
        };
        auto page_of = [&](uint32_t t) { return gld<int32_t>(table + (uint32_t)(((uint64_t)t * a.page_mul) >> a.page_shift)); };
        // keys behind the tile's last are read as that one: none of them is seen
        auto key = [&](uint32_t k0, uint32_t row) { return min(k0 + row, end - 1); };
        constexpr uint32_t ROUNDS = KT * D / 8 / kBlock;  // groups of 8 values a thread
        constexpr uint32_t PER = D / 8;                   // of a row
        int32_t pages[ROUNDS];
        auto group_row = [&](uint32_t r) { return DIRECT ? (r * kWaves + wv) * (64 / PER) + lane / PER : (r * kBlock + tid) / PER; };
        auto look = [&](uint32_t k0) {
#pragma unroll
            for (uint32_t r = 0; r < ROUNDS; r++) pages[r] = page_of(key(k0, group_row(r)));
        };
        typedef typename std::conditional<F, f4, u4>::type Word;
        constexpr uint32_t WORDS = F ? 2 : 1;
        Word kw[DIRECT ? 1 : ROUNDS][WORDS], vw[DIRECT ? 1 : ROUNDS][WORDS];
        auto fetch = [&](uint32_t k0, uint32_t buf) {
#pragma unroll
            for (uint32_t r = 0; r < ROUNDS; r++) {
                const uint32_t line = group_row(r);
                const size_t at = place(key(k0, line), pages[r]);
                if constexpr (DIRECT) {
#if defined(__HIP_DEVICE_COMPILE__)
                    const uint32_t c = lane % PER ^ turn<CH>(line);
                    const uint32_t to = (r * kWaves + wv) * 1024;
                    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(a.c.k + 2 * at + 16 * c),
                                                     (__attribute__((address_space(3))) void*)(ks[buf] + to), 16, 0, 0);
                    __builtin_amdgcn_global_load_lds((__attribute__((address_space(1))) void*)(a.c.v + 2 * at + 16 * c),
                                                     (__attribute__((address_space(3))) void*)(vs[buf] + to), 16, 0, 0);
#endif
                } else {
                    const uint32_t d = (r * kBlock + tid) % PER * 8;
                    auto load = [&](const uint8_t* p, const _Float16* sc, Word* w) {
                        if (d >= dim) {
                            for (uint32_t i = 0; i < WORDS; i++) w[i] = Word{0, 0, 0, 0};
                            return;
                        }
                        if constexpr (F) {
                            float x[8];
                            if (a.kv_wide) {
                                if (a.c.kind == F32) {
                                    w[0] = gld<f4>(p + 4 * (at + d)), w[1] = gld<f4>(p + 4 * (at + d) + 16);
                                    return;
                                }
                                if (a.c.kind == Q8_0) {
                                    const uint2 u = gld<uint2>(p + at + d);
                                    const float f = (float)gld<_Float16>(sc + (at + d) / 32);
#pragma unroll
                                    for (int j = 0; j < 8; j++) x[j] = (float)(int8_t)((j < 4 ? u.x : u.y) >> 8 * (j & 3)) * f;
                                } else {
                                    const u4 u = gld<u4>(p + 2 * (at + d));
#pragma unroll
                                    for (int j = 0; j < 8; j++) {
                                        const uint32_t v = j & 1 ? u[j / 2] >> 16 : u[j / 2] & 0xffff;
                                        x[j] = a.c.kind == F16 ? h2f(v) : __uint_as_float(v << 16);
                                    }
                                }
                            } else {
#pragma unroll
                                for (uint32_t j = 0; j < 8; j++) {
                                    const size_t e = at + min(d + j, dim - 1);
                                    x[j] = a.c.kind == Q8_0 ? elem<Q8_0>(p, e) * (float)gld<_Float16>(sc + e / 32) : elem_kind(a.c.kind, p, e);
                                    if (d + j >= dim) x[j] = 0.f;
                                }
                            }
                            w[0] = {x[0], x[1], x[2], x[3]}, w[1] = {x[4], x[5], x[6], x[7]};
                        } else if (a.kv_wide) {
                            w[0] = gld<u4>(p + 2 * (at + d));
                        } else {
                            uint32_t x[8];
#pragma unroll
                            for (uint32_t j = 0; j < 8; j++) x[j] = d + j < dim ? gld<uint16_t>(p + 2 * (at + d + j)) : 0;
                            w[0] = {x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16};
                        }
                    };
                    load(a.c.k, a.c.ks, kw[r]);
                    load(a.c.v, a.c.vs, vw[r]);
                }
            }
        };
        auto store = [&](uint32_t buf) {
            if constexpr (!DIRECT) {
#pragma unroll
                for (uint32_t r = 0; r < ROUNDS; r++) {
                    const uint32_t u = r * kBlock + tid, line = u / PER;
#pragma unroll
                    for (uint32_t w = 0; w < WORDS; w++) {
                        const uint32_t to = line * D * sizeof(T) + (u % PER * WORDS + w ^ turn<CH>(line)) * 16;
                        *reinterpret_cast<Word*>(ks[buf] + to) = kw[r][w];
                        *reinterpret_cast<Word*>(vs[buf] + to) = vw[r][w];
                    }
                }
            }
        };

        // ---- a step
        auto step = [&](uint32_t k0, uint32_t buf) {
            const uint8_t *kt = ks[buf], *vt = vs[buf];
            f16v sc[NS];
#pragma unroll
            for (uint32_t m = 0; m < NS; m++)
#pragma unroll
                for (int j = 0; j < 16; j++) sc[m][j] = 0.f;
            const uint8_t* krow = kt + n * D * sizeof(T);
            const uint32_t kturn = turn<CH>(n);
            if constexpr (F) {
#pragma unroll
                for (uint32_t g = 0; g < D / 8; g++) {
                    const f4 x = *reinterpret_cast<const f4*>(krow + ((2 * g + half) ^ opaque(kturn)) * 16);
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], q[4 * g + j], sc[0], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (uint32_t g = 0; g < D / 16; g++)
#pragma unroll
                    for (uint32_t m = 0; m < NS; m++) {
                        const T8 x = *reinterpret_cast<const T8*>(krow + m * 32 * D * 2 + ((2 * g + half) ^ kturn) * 16);
                        if constexpr (H) sc[m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, q[g], sc[m], 0, 0, 0);
                        else sc[m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, q[g], sc[m], 0, 0, 0);
                    }
            }
            // which of the step's keys the row sees, one a bit
            const bool masked = k0 + KT > all;
            uint64_t sees = ~0ull;
            if (masked) {
                if (a.seen) {
                    const uint32_t d = k0 >= s.c0 ? k0 - s.c0 : s.c0 - k0;
                    if (k0 >= s.c0) sees = d < 64 ? bits >> d : 0;
                    else sees = d < 64 ? bits << d | ((1ull << d) - 1) : ~0ull;
                } else {
                    const uint32_t d = own > k0 ? own - k0 : 0;
                    sees = d < 64 ? (1ull << d) - 1 : ~0ull;
                }
#pragma unroll
                for (uint32_t m = 0; m < NS; m++) {
                    const uint32_t w = (uint32_t)(sees >> 32 * m) >> 4 * half;
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++) sc[m][j] = w >> (j / 4 * 8 + j % 4) & 1 ? sc[m][j] : -INFINITY;
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (uint32_t m = 0; m < NS; m++)
#pragma unroll
                for (int j = 0; j < 16; j++) top = fmaxf(top, sc[m][j]);
            const float2 t2 = halves(top);
            top = fmaxf(t2.x, t2.y) * a.c2;
            // the reference follows the maximum only where that is far above it
            if (__any(top - kUp > M + (F ? 0.f : kAhead))) {
                const float Mn = fmaxf(M, top - kUp), f = Mn == -INFINITY ? 1.f : exp2_of(M - Mn);
                M = Mn;
                L *= f;
#pragma unroll
                for (uint32_t d = 0; d < ND; d++)
#pragma unroll
                    for (int j = 0; j < 16; j++) o[d][j] *= f;
            }
            const float Mf = M == -INFINITY ? 0.f : M;
            if (masked && odd == ~0u) {
                uint32_t found = 0;
                constexpr uint32_t top_bits = F ? 0x7f800000u : H ? 0x7c007c00u : 0x7f807f80u, one = F ? 0x00800000u : H ? 0x04000400u : 0x00800080u;
#pragma unroll 2
                for (uint32_t i = lane; i < KT * CH; i += 64) {
                    const u4 x = *reinterpret_cast<const u4*>(vt + i * 16);
#pragma unroll
                    for (int j = 0; j < 4; j++) found |= (x[j] & top_bits) + one;
                }
                if (__any((found & (F ? 0x80000000u : 0x80008000u)) != 0)) odd = k0;
            }
            if constexpr (F) {
                float p[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    p[j] = exp2_of(fmaf(sc[0][j], a.c2, -Mf));
                    L += p[j];
                }
                if (odd != ~0u) return;
#pragma unroll
                for (uint32_t j = 0; j < 16; j++) {
                    const uint32_t line = j / 4 * 8 + 4 * half + j % 4;
                    const uint32_t l = opaque(n);  // computed here: one operation a product is free, registers are not
                    const uint8_t* v = vt + line * D * 4 + l % 4 * 4;
#pragma unroll
                    for (uint32_t d = 0; d < ND; d++) {
                        const float x = *reinterpret_cast<const float*>(v + ((8 * d + l / 4) ^ turn<CH>(line)) * 16);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[j], o[d], 0, 0, 0);
                    }
                }
            } else {
                T8 p[2 * NS];
#pragma unroll
                for (uint32_t m = 0; m < NS; m++)
#pragma unroll
                    for (uint32_t j = 0; j < 16; j += 2) {
                        const float x = exp2_of(fmaf(sc[m][j], a.c2, -Mf)), y = exp2_of(fmaf(sc[m][j + 1], a.c2, -Mf));
                        // the sum is of the rounded weights, so that equal errors of all cancel
                        if constexpr (H) {
                            const h2 z = {(_Float16)x, (_Float16)y}, ones = {(_Float16)1.f, (_Float16)1.f};
                            L = __builtin_amdgcn_fdot2(z, ones, L, false);
                            p[2 * m + j / 8][j % 8] = z[0], p[2 * m + j / 8][j % 8 + 1] = z[1];
                        } else {
                            const b2 z = {(bf16_t)x, (bf16_t)y}, ones = {(bf16_t)1.f, (bf16_t)1.f};
                            L = __builtin_amdgcn_fdot2_f32_bf16(z, ones, L, false);
                            p[2 * m + j / 8][j % 8] = z[0], p[2 * m + j / 8][j % 8 + 1] = z[1];
                        }
                    }
                if (odd != ~0u) return;
                // lane's part of the transposing read: row (lane % 16) / 4 of four, values
                // 4 (lane % 4) .. + 3 of 16
#if defined(__HIP_DEVICE_COMPILE__)
                const uint32_t vrow = lane % 16 / 4, col = (lane >> 4 & 1) * 2 + (lane % 4 >> 1);
#pragma unroll
                for (uint32_t c = 0; c < 2 * NS; c++)
#pragma unroll
                    for (uint32_t d = 0; d < ND; d++) {
                        struct { s4 w[2]; } w;
#pragma unroll
                        for (uint32_t e = 0; e < 2; e++) {
                            const uint32_t line = 16 * c + 8 * e + 4 * half + vrow;
                            const uint8_t* v = vt + line * D * 2 + ((4 * d + col) ^ turn<CH>(line)) * 16 + lane % 2 * 8;
                            w.w[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)v);
                        }
                        const T8 x = __builtin_bit_cast(T8, w);
                        if constexpr (H) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, p[c], o[d], 0, 0, 0);
                        else o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, p[c], o[d], 0, 0, 0);
                    }
#endif
            }
        };

        // the loads that go to LDS by themselves are no ordinary accesses to it: the wave waits
        // for its own before it meets the others
        auto meet = [&] {
            if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        };
        if (tid == 0) bad_at = ~0u;
        look(lo);
        fetch(lo, 0);
        store(0);
        if (lo + KT < hi) look(lo + KT);
        meet();
        uint32_t buf = 0;
        for (uint32_t k0 = lo; k0 < hi; k0 += KT, buf ^= 1) {
            const bool more = k0 + KT < hi;
            if (more) {
                fetch(k0 + KT, buf ^ 1);
                if (k0 + 2 * KT < hi) look(k0 + 2 * KT);
            }
            if (k0 < most) step(k0, buf);
            if (more) store(buf ^ 1);
            meet();
        }
        // the steps left out, a key at a time: its row goes through the wave's part of LDS
        if (odd != ~0u) {
            float* line = reinterpret_cast<float*>(ks) + wv * 2 * D;
            auto settle = [] {  // the rows are this wave's own
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            };
            auto value = [&](const uint8_t* p, const _Float16* sc, size_t e) {
                return a.c.kind == Q8_0 ? elem<Q8_0>(p, e) * (float)gld<_Float16>(sc + e / 32) : elem_kind(a.c.kind, p, e);
            };
#pragma nounroll
            for (uint32_t t = odd; t < min(hi, most); t++) {
                const size_t at = place(t, page_of(t));
                settle();
                for (uint32_t d = lane; d < D; d += 64) {
                    line[d] = d < dim ? value(a.c.k, a.c.ks, at + d) : 0.f;
                    line[D + d] = d < dim ? value(a.c.v, a.c.vs, at + d) : 0.f;
                }
                settle();
                float x = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < D / 2; i++) {
                    constexpr uint32_t each = F ? 4 : 8;
                    float y;
                    if constexpr (F) y = q[i];
                    else y = (float)q[i / 8][i % 8];
                    x = fmaf(y, line[i / each * 2 * each + each * half + i % each], x);
                }
                const float2 x2 = halves(x);
                if (a.seen ? t >= s.c0 && !(bits >> (t - s.c0) & 1) : t >= own) continue;
                const float w = exp2_of(fmaf(x2.x + x2.y, a.c2, M == -INFINITY ? 0.f : -M));
#pragma unroll
                for (uint32_t i = 0; i < D / 2; i++)
                    o[i / 16][i % 16] = fmaf(w, line[D + i / 16 * 32 + i % 16 / 4 * 8 + 4 * half + i % 4], o[i / 16][i % 16]);
            }
        }
        if (bad != ~0u) atomicMin(&bad_at, bad);
        __syncthreads();
        const float2 l2 = halves(L);
        L = bad_at < own ? __builtin_nanf("") : l2.x + l2.y;
        __syncthreads();
        if (mine && whole) {
            const float f = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
            for (uint32_t d = 0; d < ND; d++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    f4 x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                    if (L == 0.f) x = f4(0.f);
                    put_row(a, dim, row, h, 32 * d + 8 * i + 4 * half, x * f);
                }
        } else if (mine) {
            const size_t slot = (size_t)run.run * 2 + (run.off == 0);
            const uint32_t line = wv * 32 + n;
            float* to = part_o(a, slot) + line * D;
#pragma unroll
            for (uint32_t d = 0; d < ND; d++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++)
                    *reinterpret_cast<f4*>(to + 32 * d + 8 * i + 4 * half) = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
            if (half == 0) part_ml(a, slot)[line] = make_float2(M, L);
        }
    } while (run.next(a));
}

// out of the tiles that several workgroups hold parts of: a workgroup for the first
// run that begins inside a tile, and 1,024 of its values; four a thread.
__global__ __launch_bounds__(kBlock) void k_page_many_join(PageMany a, uint32_t step) {
    const uint32_t D = a.wide, w = blockIdx.x + 1;
    const ManyHead hd = *head_of(a);
    const uint32_t runs = min(hd.runs, a.runs);
    if (w >= runs) return;
    const ManyMark m = *mark_of(a, w);
    if (!m.cost || m.kv >= a.c.kvheads || m.rows > kTileRows || run_begin(hd.total, runs, w - 1) > m.at) return;
    const uint32_t at = (blockIdx.y * kBlock + threadIdx.x) * 4, line = at / D, d = at % D;
    if (line >= m.rows) return;
    float M = -INFINITY, L = 0.f;
    f4 O = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t p = w - 1; p < runs; p++) {
        const uint64_t x0 = max(run_begin(hd.total, runs, p), m.at) - m.at, x1 = run_begin(hd.total, runs, p + 1) - m.at;
        if (x0 >= m.cost) break;
        const uint32_t lo = key_at(a, x0, m.end, step), hi = x1 >= m.cost ? m.end : key_at(a, x1, m.end, step);
        if (lo >= hi) continue;  // no step of its own
        const size_t slot = (size_t)p * 2 + (x0 == 0);
        const float2 ml = part_ml(a, slot)[line];
        const f4 o = *reinterpret_cast<const f4*>(part_o(a, slot) + line * D + d);
        const float Mn = fmaxf(M, ml.x), Mf = Mn == -INFINITY ? 0.f : Mn;
        const float f = exp2_of(M - Mf), e = exp2_of(ml.x - Mf);
        M = Mn;
        L = fmaf(ml.y, e, L * f);
#pragma unroll
        for (int j = 0; j < 4; j++) O[j] = fmaf(o[j], e, O[j] * f);
    }
    const uint32_t r = m.row + line, row = r / a.group;
    if (row >= a.n) return;
    put_row(a, a.c.dim, row, m.kv * a.group + r % a.group, d, L == 0.f ? f4(0.f) : O * (1.f / L));
}

// ---------------------------------------------------------------- launches --
// The type of a call's products and the width of its tiles; what its rows are aligned to.
void page_many_plan(PageMany& a, uint32_t cus) {
    const uint32_t d = a.c.dim, es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2;
    a.group = a.heads / a.c.kvheads;
    a.wide = d <= 64 ? 64 : d <= 128 ? 128 : 256;
    a.narrow = a.q.kind != F32 && a.out.kind != F32 && a.c.kind == a.q.kind;
    auto aligned = [](const Heads& h, uint32_t bytes) {
        const uint64_t e = h.kind == F32 ? 4 : 2;
        return (((uintptr_t)h.p | h.row * e | h.head * e) % bytes) == 0;
    };
    a.q_wide = d % 8 == 0 && aligned(a.q, 16);
    a.out_wide = aligned(a.out, a.out.kind == F32 ? 16 : 8);
    a.kv_wide = d % 8 == 0 && (((uintptr_t)a.c.k | (uintptr_t)a.c.v | (a.c.ps | a.c.ts | a.c.hs) * es) % std::min(8 * es, 16u)) == 0;
    // t / page for t < 2^31: t * ceil(2^shift / page) >> shift
    uint32_t log = 0;
    while ((1ull << log) < a.c.page) log++;
    a.page_shift = 31 + log;
    a.page_mul = (uint32_t)(((1ull << a.page_shift) + a.c.page - 1) / a.c.page);
    a.sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
    a.c2 = a.scale == 0.f ? 1.f : std::max(std::fabs(a.scale) * kLog2e, 1.17549435e-38f);
    const uint64_t tiles = ((uint64_t)a.n * a.group / kTileRows + a.r.batch) * a.c.kvheads;
    const uint64_t most = tiles * (a.r.most / kRunKeys + 2);
    a.runs = (uint32_t)std::min<uint64_t>(cus * (a.wide == 256 ? 1 : 2), std::max<uint64_t>(most, 1));
}

template <class T, uint32_t D> static void launch_tiles(const PageMany& a, bool direct, hipStream_t s) {
    const dim3 grid((a.runs + kXcds - 1) / kXcds * kXcds), block(kBlock);
    if constexpr (!std::is_same<T, float>::value)
        if (direct) {
            hipLaunchKernelGGL((k_page_many<T, D, true>), grid, block, 0, s, a);
            return;
        }
    hipLaunchKernelGGL((k_page_many<T, D, false>), grid, block, 0, s, a);
}
template <class T> static void launch_many(const PageMany& a, hipStream_t s) {
    const bool direct = a.narrow && a.kv_wide && a.c.dim == a.wide;
    if (a.wide == 64) launch_tiles<T, 64>(a, direct, s);
    else if (a.wide == 128) launch_tiles<T, 128>(a, direct, s);
    else launch_tiles<T, 256>(a, direct, s);
}
void launch_page_many(const PageMany& a, hipStream_t s) {
    if (!a.narrow) launch_many<float>(a, s);
    else if (a.c.kind == F16) launch_many<_Float16>(a, s);
    else launch_many<bf16_t>(a, s);
    if (a.runs > 1)
        hipLaunchKernelGGL(k_page_many_join, dim3(a.runs - 1, kTileRows * a.wide / (4 * kBlock)), dim3(kBlock), 0, s, a,
                           !a.narrow || a.wide == 256 ? 32 : 64);
}

}  // namespace qh
