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
//
// Bound by the products, but for few rows over a long context, which wait for the cache's
// bytes.  Measured, with 32 query heads over 4 KV heads of 128 values, on a card whose
// large products reach 1,104 TFLOP/s in f16, 1,160 in bf16 and 153 in f32, and whose large
// copies 4.6 TB/s (products that a causal row sees, join included):
//   16,381 tokens, f16                         3.17 ms   694 TFLOP/s, with the weights' second parts 1,041
//   24 prompts of 1 to 2,100 tokens, bf16      0.68 ms   523 TFLOP/s, 785
//   2 x 512 tokens behind 12,000 to 15,000, Q8_0   0.545 ms   424 TFLOP/s; the vector units: codes to f16, scales
//   517 tokens, f32                              59 us    37 TFLOP/s; runs of 4 to 5 steps
//   2 trees of 64 nodes behind 65,537 keys, f16 231 us   595 TFLOP/s, 893; 1.2 TB/s
//   48 trees behind up to 4,096 keys, bf16       89 us   326 TFLOP/s, 489; 203 MB of keys and values, of which trees of
//                                                        more than 128 rows read theirs once a tile: 324 MB
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLeast = 1.17549435e-38f, kMost = 3.40282347e38f;  // f32's normal numbers
constexpr uint32_t kTileRows = 128;  // query rows of a tile, 32 a wave
constexpr uint32_t kXcds = 8;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef bf16_t b2 __attribute__((ext_vector_type(2)));
typedef bf16_t b4 __attribute__((ext_vector_type(4)));
typedef bf16_t b8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t same64(uint64_t v) { return (uint64_t)same((uint32_t)(v >> 32)) << 32 | same((uint32_t)v); }
// The values of lanes l and l ^ 32.
__device__ __forceinline__ float2 halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The compiler moves no instruction across: products, the LDS reads ahead of them and the
// arithmetic between them are issued in the order that is written.
__device__ __forceinline__ void in_order() { __builtin_amdgcn_sched_barrier(0); }

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
__device__ __forceinline__ bool rows_fit(const PageMany& a, int32_t f, int32_t e) { return f >= 0 && f <= e && (uint32_t)e <= a.n; }
__device__ __forceinline__ bool with_tokens(const PageMany& a, uint32_t b) {
    const int32_t f = gld<int32_t>(a.first + b), e = gld<int32_t>(a.first + b + 1);
    return rows_fit(a, f, e) && f < e;
}
__device__ __forceinline__ Seq seq_of(const PageMany& a, const Bounds& q) {
    Seq s{};
    const int32_t f = q.f, e = q.e;
    s.len = q.len;
    if (!rows_fit(a, f, e)) return s;
    s.f0 = (uint32_t)f;
    s.count = (uint32_t)(e - f);
    s.tiles = (uint32_t)(((uint64_t)s.count * a.group + kTileRows - 1) / kTileRows);
    s.bad = s.len < 0 || s.count > (uint32_t)s.len || (a.seen && s.count > kTreeMost);
    s.c0 = s.bad ? 0 : (uint32_t)s.len - s.count;
    s.first = s.bad ? 1 : a.seen ? (uint64_t)(a.tile_keys + s.len) * a.group : (uint64_t)(a.tile_keys + s.c0 + 1) * a.group + kTileRows - 1;
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
    const uint64_t k = x / a.group;
    return k <= a.tile_keys ? 0 : (uint32_t)min((uint64_t)end, (k - a.tile_keys) / step * step);
}

__device__ __forceinline__ uint64_t run_begin(uint64_t total, uint32_t runs, uint32_t i) {
    return total / runs * i + min((uint64_t)i, total % runs);
}

// What the join has to know of the tile that a run begins inside of, where it is the
// first to: the tile's first row (times the group), rows and KV head, and the last run that
// holds a part of it.  rows 0: nothing to join.
struct ManyMark {
    uint32_t row, rows, kv, last;
};
size_t page_many_bytes(const PageMany& a) {
    const size_t slots = (size_t)a.runs * 2 * kTileRows;
    return slots * a.wide * 4 + slots * 8 + 16 + a.runs * sizeof(ManyMark);
}
__device__ __forceinline__ float* part_o(const PageMany& a, size_t slot) { return (float*)a.work + slot * kTileRows * a.wide; }
__device__ __forceinline__ float2* part_ml(const PageMany& a, size_t slot) {
    return (float2*)((float*)a.work + (size_t)a.runs * 2 * kTileRows * a.wide) + slot * kTileRows;
}
__device__ __forceinline__ uint32_t* runs_of(const PageMany& a) { return (uint32_t*)part_ml(a, (size_t)a.runs * 2); }
__device__ __forceinline__ ManyMark* mark_of(const PageMany& a, uint32_t run) { return (ManyMark*)(runs_of(a) + 4) + run; }

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
        const uint32_t runs = (uint32_t)max((uint64_t)1, min((uint64_t)a.runs, total / ((uint64_t)a.run_keys * a.group)));
        if (blockIdx.x == 0 && tid == 0) *runs_of(a) = total ? runs : 0;
        // runs that lie beside each other, and read the same keys, on one XCD
        const uint32_t per = (runs + kXcds - 1) / kXcds;
        run = blockIdx.x % kXcds * per + blockIdx.x / kXcds;
        if (!total || blockIdx.x / kXcds >= per || run >= runs) return false;
        x = same64(run_begin(total, runs, run));
        end = same64(run_begin(total, runs, run + 1));
        if (tid == 0) mark_of(a, run)->rows = 0;
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
        kv = same((uint32_t)(in / each));
        off = in - kv * each;
        if (kv >= G) return false;
        uint32_t lo = 0, hi = s.tiles;  // the last tile whose place is not behind off
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (s.upto(mid) <= off) lo = mid;
            else hi = mid;
        }
        i = same(lo);
        off = same64(off - s.upto(i));
        if (off && tid == 0 && !s.bad && run_begin(total, runs, run - 1) <= x - off) {
            uint32_t last = run;
            const uint64_t to = x - off + s.cost(i);
            if (end < to) {  // the run of the tile's last place
                const uint64_t each = total / runs, more = total % runs, wide = more * (each + 1);
                last = (uint32_t)(to - 1 < wide ? (to - 1) / (each + 1) : more + (to - 1 - wide) / each);
            }
            *mark_of(a, run) = {s.f0 * a.group + i * kTileRows, min(kTileRows, s.count * a.group - i * kTileRows), kv, last};
        }
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
        // The next sequence with new tokens: the next one, or of those behind it, kBlock at a time (one after the
        // other, five with tokens among 65,535 took 7.2 ms rather than 0.3).
        __shared__ uint32_t near;
        for (uint32_t to = b + 1;;) {
            if (to >= a.r.batch) return false;
            b = to;
            read(a);
            if (s.tiles) return true;
            uint32_t j0 = b + 1;
            do {
                if (threadIdx.x == 0) near = ~0u;
                __syncthreads();
                const uint32_t j = j0 + threadIdx.x;
                if (j < a.r.batch && with_tokens(a, j)) atomicMin(&near, j);
                __syncthreads();
                to = same(near);
                j0 += kBlock;
                __syncthreads();
            } while (to == ~0u && j0 < a.r.batch);
        }
    }
};

// --------------------------------------------------------------- the tiles --
// Values d .. d + 3 of the row of out at `at`.
__device__ __forceinline__ void put_row(const PageMany& a, uint32_t dim, size_t at, uint32_t d, f4 x) {
    if (a.out_wide && d + 4 <= dim) {
        if (a.out.kind == F32) *reinterpret_cast<f4*>(a.out.p + 4 * (at + d)) = x;
        else if (a.out.kind == F16) *reinterpret_cast<h4*>(a.out.p + 2 * (at + d)) = __builtin_convertvector(x, h4);
        else *reinterpret_cast<b4*>(a.out.p + 2 * (at + d)) = __builtin_convertvector(x, b4);
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
        if (d + j < dim) put_kind(a.out.kind, a.out.p, at + d + j, x[j]);
}

// The 16-byte chunk of a tile's row that chunk c lies in: rows that are read together
// are spread over the banks (K: 32 rows a read at one chunk, 8 of them a cycle; V: four
// rows at four chunks).
template <uint32_t CH> __device__ __forceinline__ constexpr uint32_t turn(uint32_t row) {
    return CH >= 16 ? (row & 3) << 2 | (row >> 2 & 3) : (row >> 1 & 1) << 2 | (row >> 2 & 3);
}

// Where a kernel's tiles come from: the cache's rows as they are, by loads that go to LDS
// by themselves (kDirect: rows of T, D wide, aligned to 16 bytes), or through registers, rows
// of that kind aligned to 8 values, or of any kind and alignment (kAny; 16 bits: of T).
constexpr uint32_t kDirect = 100, kAny = 101;

// T: type of the products; D: width of the tiles, at least the heads'.
//
// A wave has 32 query rows.  It takes the scores as K Q^T, so that a lane has one
// row's scores (of the keys 8 i + 4 (lane / 32) + j), its maximum and sum need one
// exchange, and the weights lie where O^T = V^T P^T wants its second operand: for 16-bit
// types keys 16 c + 8 (e / 4) + 4 (lane / 32) + e % 4 are element e, for V^T read by the
// transposing LDS read.  K and V of the next step come in while one is worked on, asked
// for between the products of the scores (16,381 tokens 2.73 -> 2.55 ms before a weight had two
// parts).  A weight meets its
// values in two parts of T, rounded and what that left: 17 bits in bf16, 23 in f16, as in the
// attention of single tokens, so that an output is off by its own rounding alone.  One part would
// be faster (16,381 tokens 2.26 ms rather than 3.17, 24 prompts 0.59 rather than 0.68, 48 trees 79
// rather than 89 us) and 1.2 to 1.4 times as far off.  Everything else between the products is in
// 32 bits, but over Q8_0, in f16 products under outputs of bf16, whose weights and values are rounded
// once, three bits finer than the outputs (both in two parts: two prompts behind 12,000 to 15,000 keys
// 0.71 ms rather than 0.55, and no nearer to 64 bits).  Written so that none of the kernels
// spills vector registers: what is wanted once a tile is computed there anew.
template <class T, uint32_t D, uint32_t SRC>
__global__ __launch_bounds__(kBlock, D == 256 || (SRC == Q8_0 && D == 128 && std::is_same<T, _Float16>::value) ? 1 : 2) void k_page_many(PageMany a) {
    constexpr bool F = std::is_same<T, float>::value, H = std::is_same<T, _Float16>::value;
    constexpr bool DIRECT = SRC == kDirect, Q8 = SRC == Q8_0 && !F;
    constexpr uint32_t KT = F || Q8 || D == 256 ? 32 : 64;  // keys of a step
    constexpr uint32_t NS = KT / 32, ND = D / 32, CH = D * sizeof(T) / 16, TILE = KT * D * sizeof(T);
    constexpr uint32_t NQ = F ? D / 2 : D / 16;
    constexpr uint32_t QKIND = F ? F32 : H && !Q8 ? F16 : BF16;  // of queries that are loaded as they are
    constexpr bool TWO = !F && !Q8;  // parts of a weight
    // weights are at most 2^(kAhead + kUp): in f16 2^15, so that small ones have their bits, the more the closer the
    // reference stays to the maximum (4 and 8 take as long; over Q8_0 4 0.573 ms rather than 0.549); in bf16, which has
    // f32's exponents, 1, so that sums of values up to 2^128 / keys fit
    constexpr float kAhead = TWO ? 4.f : 8.f, kUp = F ? 0.f : H ? 15.f - kAhead : -kAhead;
    typedef typename std::conditional<H, h8, b8>::type T8;
    typedef typename std::conditional<F, float, T8>::type Q;
    __shared__ __align__(16) uint8_t lds[4][TILE];  // K, K, V, V; in front and behind a part for each wave
    __shared__ __align__(16) float scales[Q8 ? 2 : 1][Q8 ? ND : 1][Q8 ? KT : 1];  // of K's blocks
    __shared__ uint32_t bad_at;
    const uint32_t wv = same(threadIdx.x >> 6);
    auto settle = [] {  // what the wave wrote to its own part of LDS can be read
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    auto shfl64 = [](size_t v, uint32_t from) { return (size_t)__shfl((unsigned long long)v, from, 64); };
    Run run;
    if (!run.start(a)) return;
    do {
        // hidden, so that what follows from it is not kept in registers from one tile to the next
        const uint32_t tid = opaque(threadIdx.x), lane = tid & 63, n = lane & 31, half = lane >> 5;
        const Seq& s = run.s;
        const uint32_t end = same(end_of(a, s, run.i)), R = s.count * a.group;
        const uint32_t lo = same(key_at(a, run.off, end, KT));
        const bool whole = run.off == 0 && run.here() == s.cost(run.i);
        const uint32_t hi = same(run.off + run.here() == s.cost(run.i) ? end : key_at(a, run.off + run.here(), end, KT));
        const uint32_t r0 = run.i * kTileRows + wv * 32, r = r0 + n;  // rows of the sequence and KV head
        const uint32_t rows = r0 >= R ? 0 : min(32u, R - r0);        // of the wave
        const bool mine = n < rows;
        const uint32_t dim = a.c.dim;
        const uint32_t token = mine ? r / a.group : 0, row = s.f0 + token, h = run.kv * a.group + (mine ? r % a.group : 0);
        // where a row of the wave's goes; found anew where it is wanted, to hold no registers
        auto out_at = [&](uint32_t n) {
            const uint32_t r = min(r0 + n, R - 1);
            return (size_t)(s.f0 + r / a.group) * a.out.row + (size_t)(run.kv * a.group + r % a.group) * a.out.head;
        };
        if (s.bad) {
            if (run.off == 0 && mine)
                for (uint32_t d = half * 4; d < dim; d += 8) put_row(a, dim, out_at(n), d, f4(__builtin_nanf("")));
            continue;
        }
        const size_t slot = (size_t)run.run * 2 + (run.off == 0);  // of a part
        if (lo >= hi) {  // no step of its own
            if (mine && half == 0) part_ml(a, slot)[wv * 32 + n] = make_float2(-INFINITY, 0.f);
            continue;
        }
        // behind the last key that one of the wave's rows sees
        const uint32_t most = !rows ? 0 : a.seen ? end : s.c0 + (r0 + rows - 1) / a.group + 1;
        const uint32_t own = a.seen ? end : s.c0 + token + 1;  // behind this row's last
        uint64_t bits = 0;
        if (a.seen && mine) bits = gld<uint64_t>(a.seen + row) & (s.count == 64 ? ~0ull : (1ull << s.count) - 1);

        Q q[NQ];
        float c2 = a.c2;
        f16v o[ND];
#pragma unroll
        for (uint32_t d = 0; d < ND; d++)
#pragma unroll
            for (int j = 0; j < 16; j++) o[d][j] = 0.f;
        f16v zeros;  // in registers, as sixteen moves a product would not be free
        if constexpr (Q8)
#pragma unroll
            for (int j = 0; j < 16; j++) zeros[j] = __uint_as_float(opaque(0u));
        float M = -INFINITY, L = 0.f;
        // the first step with a value that is not finite beside keys that some row does not
        // see: 0 times it is no 0, so from there on the products are taken key by key, below
        uint32_t odd = ~0u;
        uint32_t bad = ~0u;  // the first key that this lane found in a page out of range

        // ---- a step's K and V
        const int32_t* table = a.r.table + run.b * a.r.stride;
        const size_t base = run.kv * a.c.hs;
        auto page_number = [&](uint32_t t) { return __umulhi(t << 1, a.page_mul) >> a.page_log; };
        auto page_of = [&](uint32_t t) { return gld<int32_t>(table + page_number(t)); };
        auto place = [&](uint32_t t, int32_t page) {  // of key t; a page out of range is read as page 0
            if ((uint32_t)page >= a.c.count) bad = min(bad, t), page = 0;
            return (size_t)page * a.c.ps + (size_t)(t - page_number(t) * a.c.page) * a.c.ts + base;
        };
        // keys behind the tile's last are read as that one: none of them is seen
        // a thread takes groups of 8 values, kDirect 16 bytes; PER of a row, LINES rows a wave
        constexpr uint32_t PER = DIRECT ? CH : D / 8, LINES = 64 / PER, ROUNDS = KT * PER / kBlock;
        auto group_row = [&](uint32_t r) { return (r * kBlock + tid) / PER; };
        // kDirect: the rows of a wave's load lie in one page.  Lane r (and r + ROUNDS ..) finds round r's first
        // row and its place, which the round then has for all lanes.
        int32_t pages[DIRECT ? 1 : ROUNDS];
        uint32_t first = 0;    // that row
        uint64_t first_at = 0;  // and its place, in bytes
        auto look = [&](uint32_t k0) {
            if constexpr (DIRECT) {
                first = min(k0 + (lane % ROUNDS * kWaves + wv) * LINES, (end - 1) / LINES * LINES);
                pages[0] = page_of(first);
            } else {
#pragma unroll
                    for (uint32_t r = 0; r < ROUNDS && SRC != kAny; r++) pages[r] = page_of(min(k0 + group_row(r), end - 1));
            }
        };
        auto found = [&] {  // what look() was after
            if constexpr (DIRECT) {
                const bool fine = (uint32_t)pages[0] < a.c.count;
                bad = fine ? bad : min(bad, first);
                const uint32_t in = first - page_number(first) * a.c.page;
                first_at = (uint64_t)(fine ? (uint32_t)pages[0] : 0u) * (uint32_t)(sizeof(T) * a.c.ps) + in * (uint32_t)(sizeof(T) * a.c.ts);
            }
        };
        [[maybe_unused]] const uint8_t *kbase = a.c.k + sizeof(T) * base, *vbase = a.c.v + sizeof(T) * base;
        // What a thread holds of a step meanwhile, as it is in the cache: eight values of K and of V each.
        constexpr bool HELD16 = SRC == F16 || SRC == BF16;
        u4 kw[HELD16 ? ROUNDS : 1], vw[HELD16 ? ROUNDS : 1];
        uint2 kc[SRC == Q8_0 ? ROUNDS : 1], vc[SRC == Q8_0 ? ROUNDS : 1];     // codes
        uint32_t kf[SRC == Q8_0 ? ROUNDS : 1], vf[SRC == Q8_0 ? ROUNDS : 1];  // scales
        auto fetch = [&](uint32_t k0, uint32_t buf, uint32_t r) {
            if constexpr (DIRECT) {
                // 16 bytes a lane from its own address to LDS.  In assembly, as the compiler lets every
                // later LDS read wait for such loads, of whatever buffer; meet() waits for them.  With the move
                // five wait states, as a load needs behind a vector instruction that writes its scalar
                // address (one read back from a spilled lane, which the compiler does not see read here).
                if (r == 0) found();
                const uint32_t line = lane / PER, t = __builtin_amdgcn_readlane(first, r);
                const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(first_at >> 32), r) << 32 |
                                    (uint32_t)__builtin_amdgcn_readlane((uint32_t)first_at, r);
                constexpr bool SAME = turn<CH>(kWaves * LINES) == 0;  // a row's turn in every round
                const uint32_t chunk = 16 * (lane % PER ^ turn<CH>((SAME ? wv : r * kWaves + wv) * LINES + line));
                // rows behind the tile's last are read as that one
                const uint32_t off = min(line, end - 1 - t) * (uint32_t)(sizeof(T) * a.c.ts) + chunk;
#if defined(__HIP_DEVICE_COMPILE__)
                const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds[buf] + (r * kWaves + wv) * 1024;
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(kbase + at) : "memory", "m0");
                asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to + 2 * TILE), "v"(off), "s"(vbase + at) : "memory", "m0");
#else
                (void)at, (void)off;
#endif
            } else {
                const size_t at = place(min(k0 + group_row(r), end - 1), pages[r]);
                const uint32_t d = (r * kBlock + tid) % PER * 8;
                if constexpr (SRC == Q8_0) {
                    const size_t e = at + min(d, dim - 8);
                    kc[r] = gld<uint2>(a.c.k + e);
                    vc[r] = gld<uint2>(a.c.v + e);
                    kf[r] = gld<uint16_t>(a.c.ks + e / 32);
                    vf[r] = gld<uint16_t>(a.c.vs + e / 32);
                    if (d >= dim) kf[r] = vf[r] = 0;
                } else if constexpr (HELD16) {
                    const size_t e = 2 * (at + min(d, dim - 8));
                    kw[r] = gld<u4>(a.c.k + e);
                    vw[r] = gld<u4>(a.c.v + e);
                    if (d >= dim) kw[r] = vw[r] = u4{0, 0, 0, 0};
                }
            }
        };
        // To LDS, as the products take it: part i of PARTS (a round, of Q8_0's codes its K or its V).
        constexpr uint32_t PARTS = DIRECT || SRC == kAny ? 0 : Q8 ? 2 * ROUNDS : ROUNDS;
        auto store_part = [&](uint32_t buf, uint32_t i) {
            if constexpr (PARTS != 0) {
                const uint32_t r = Q8 ? i / 2 : i;
                const uint32_t u = r * kBlock + tid, line = u / PER;
                auto put = [&](const u4* w, uint32_t b) {
#pragma unroll
                    for (uint32_t i = 0; i < (F ? 2 : 1); i++)
                        *reinterpret_cast<u4*>(lds[b] + line * D * sizeof(T) + ((u % PER * (F ? 2 : 1) + i) ^ turn<CH>(line)) * 16) = w[i];
                };
                if constexpr (Q8) {
                    // code + 128 in the low bits of 1024 + 128 + code, less 1152: the code; V's times its
                    // scale, rounded once
                    auto values = [&](uint2 c, auto f) {
                        u4 w;
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const uint32_t x = __builtin_amdgcn_perm(0x64646464u, (j < 2 ? c.x : c.y) ^ 0x80808080u, j & 1 ? 0x07030702u : 0x07010700u);
                            w[j] = __builtin_bit_cast(uint32_t, f(__builtin_bit_cast(h2, x) - h2((_Float16)1152.f)));
                        }
                        return w;
                    };
                    if (i % 2 == 0) {
                        const u4 k = values(kc[r], [](h2 x) { return x; });
                        put(&k, buf);
                        if (u % PER % 4 == 0) scales[buf][u % PER / 4][line] = h2f(kf[r]);
                    } else {
                        const h2 f = h2(__builtin_bit_cast(_Float16, (uint16_t)vf[r]));
                        const u4 v = values(vc[r], [&](h2 x) { return x * f; });
                        put(&v, 2 + buf);
                    }
                } else if constexpr (SRC == Q8_0) {
                    auto one = [&](uint2 c, uint32_t f16, uint32_t b) {
                        u4 w[2];
                        const float f = h2f(f16);
#pragma unroll
                        for (int j = 0; j < 8; j++) w[j / 4][j % 4] = __float_as_uint((float)(int8_t)((j < 4 ? c.x : c.y) >> 8 * (j & 3)) * f);
                        put(w, b);
                    };
                    one(kc[r], kf[r], buf);
                    one(vc[r], vf[r], 2 + buf);
                } else if constexpr (HELD16) {
                    auto one = [&](const u4& h, uint32_t b) {
                        u4 w[2];
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const uint32_t v = j & 1 ? h[j / 2] >> 16 : h[j / 2] & 0xffff;
                            w[j / 4][j % 4] = SRC == F16 ? __float_as_uint(h2f(v)) : v << 16;
                        }
                        put(w, b);
                    };
                    one(kw[r], buf);
                    one(vw[r], 2 + buf);
                }
            }
        };
        auto store = [&](uint32_t buf) {
#pragma unroll
            for (uint32_t i = 0; i < PARTS; i++) store_part(buf, i);
        };
        // kAny: a value at a time, straight to LDS (16-bit rows aligned to 8 values: eight)
        auto bring = [&](uint32_t k0, uint32_t buf) {
#pragma nounroll
            for (uint32_t r = 0; r < ROUNDS; r++) {
                const uint32_t line = group_row(r), t = min(k0 + line, end - 1), d = (r * kBlock + tid) % PER * 8;
                const size_t at = place(t, page_of(t)) + d;
                uint8_t *ko = lds[buf] + line * D * sizeof(T), *vo = lds[2 + buf] + line * D * sizeof(T);
                auto to = [&](uint32_t j) { return ((d + j) * sizeof(T) / 16 ^ turn<CH>(line)) * 16 + (d + j) * sizeof(T) % 16; };
                if (!F && a.kv_wide) {
                    u4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
                    if (d < dim) k = gld<u4>(a.c.k + 2 * at), v = gld<u4>(a.c.v + 2 * at);
                    *reinterpret_cast<u4*>(ko + to(0)) = k;
                    *reinterpret_cast<u4*>(vo + to(0)) = v;
                    continue;
                }
#pragma nounroll
                for (uint32_t j = 0; j < 8; j++) {
                    const bool in = d + j < dim;
                    if constexpr (F) {
                        auto value = [&](const uint8_t* p, const _Float16* sc) {
                            if (!in) return 0.f;
                            return a.c.kind == Q8_0 ? elem<Q8_0>(p, at + j) * (float)gld<_Float16>(sc + (at + j) / 32) : elem_kind(a.c.kind, p, at + j);
                        };
                        *reinterpret_cast<float*>(ko + to(j)) = value(a.c.k, a.c.ks);
                        *reinterpret_cast<float*>(vo + to(j)) = value(a.c.v, a.c.vs);
                    } else {
                        *reinterpret_cast<uint16_t*>(ko + to(j)) = in ? gld<uint16_t>(a.c.k + 2 * (at + j)) : (uint16_t)0;
                        *reinterpret_cast<uint16_t*>(vo + to(j)) = in ? gld<uint16_t>(a.c.v + 2 * (at + j)) : (uint16_t)0;
                    }
                }
            }
        };

        // ---- a step
        // Where the lane reads: of K row n (and 32 on), chunk 2 g + half; of V, by the transposing
        // read, row (lane % 16) / 4 of four at 16 c + 8 e + 4 half, values 4 (lane % 4) .. + 3 of 16 of
        // chunks 4 d .. + 3.  Both chunks are turned by their row, so that g, d and e flip bits.
        const uint32_t k_at = n * D * sizeof(T) + (half ^ turn<CH>(n)) * 16;
        const uint32_t vrow = 4 * half + lane % 16 / 4;
        const uint32_t v_at = F ? 4 * half * D * 4 + n % 4 * 4
                                : vrow * D * 2 + (((lane >> 4 & 1) * 2 + (lane % 4 >> 1)) ^ turn<CH>(vrow)) * 16 + lane % 2 * 8;
        auto step = [&](uint32_t k0, auto masked, auto buf, auto between, auto behind) {
            const uint8_t *kt = lds[buf], *vt = lds[2 + buf];
            f16v sc[NS];
#pragma unroll
            for (uint32_t m = 0; m < NS; m++)
#pragma unroll
                for (int j = 0; j < 16; j++) sc[m][j] = 0.f;
            if constexpr (F) {
#pragma unroll
                for (uint32_t g = 0; g < D / 8; g++) {
                    const f4 x = *reinterpret_cast<const f4*>(kt + (opaque(k_at) ^ g * 32));
#pragma unroll
                    for (uint32_t j = 0; j < 4; j++) sc[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], q[4 * g + j], sc[0], 0, 0, 0);
                    between(g, D / 8);
                }
            } else {
                auto product = [&](const T8& x, const T8& y, const f16v& z) {
                    if constexpr (H) return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, z, 0, 0, 0);
                    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, z, 0, 0, 0);
                };
                auto k_part = [&](uint32_t g, uint32_t m) { return *reinterpret_cast<const T8*>(kt + ((Q8 ? opaque(k_at) : k_at) ^ g * 32) + m * 32 * D * 2); };
                if constexpr (Q8) {
                    // A block's codes are exact, its scale is the score's: taken while the next block's products
                    // run, whose parts and scales were read meanwhile (two prompts behind 12,000 to 15,000 keys 0.67 ->
                    // 0.57 ms).
                    constexpr uint32_t N = NS * ND;
                    T8 x[2][2];
                    f4 f[2][4];
                    f16v y[2];
                    auto read = [&](uint32_t i) {
                        const uint32_t g = i / NS, m = i % NS;
                        x[i % 2][0] = k_part(2 * g, m), x[i % 2][1] = k_part(2 * g + 1, m);
#pragma unroll
                        for (uint32_t j = 0; j < 4; j++) f[i % 2][j] = *reinterpret_cast<const f4*>(&scales[buf][g][32 * m + 8 * j + 4 * half]);
                    };
                    auto scale = [&](uint32_t i) {
#pragma unroll
                        for (uint32_t j = 0; j < 16; j++) sc[i % NS][j] = fmaf(y[i % 2][j], f[i % 2][j / 4][j % 4], sc[i % NS][j]);
                    };
                    read(0);
                    in_order();
#pragma unroll
                    for (uint32_t i = 0; i < N; i++) {
                        y[i % 2] = product(x[i % 2][0], q[2 * (i / NS)], zeros);
                        y[i % 2] = product(x[i % 2][1], q[2 * (i / NS) + 1], y[i % 2]);
                        if (i) scale(i - 1);
                        if (i + 1 < N) read(i + 1);
                        between(i, N);
                        in_order();
                    }
                    scale(N - 1);
                } else {
                    // four parts of K are on their way ahead of a product
                    constexpr uint32_t N = NS * D / 16, AHEAD = 4;
                    T8 x[AHEAD];
#pragma unroll
                    for (uint32_t i = 0; i < AHEAD; i++) x[i] = k_part(i / NS, i % NS);
                    in_order();
#pragma unroll
                    for (uint32_t i = 0; i < N; i++) {
                        sc[i % NS] = product(x[i % AHEAD], q[i / NS], sc[i % NS]);
                        if (i + AHEAD < N) x[i % AHEAD] = k_part((i + AHEAD) / NS, (i + AHEAD) % NS);
                        between(i, N);
                        in_order();
                    }
                }
            }
            auto v_part = [&](uint32_t c, uint32_t d) {
#if defined(__HIP_DEVICE_COMPILE__)
                struct { s4 w[2]; } w;
#pragma unroll
                for (uint32_t e = 0; e < 2; e++) {
                    const uint8_t* v = vt + (v_at ^ (d * 64 ^ e * 32)) + (16 * c + 8 * e) * D * 2;
                    w.w[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)v);
                }
                return __builtin_bit_cast(T8, w);
#else
                return T8{};
#endif
            };
            T8 x[2][F ? 1 : ND];  // V's parts
            if constexpr (!F && !Q8) {
#pragma unroll
                for (uint32_t d = 0; d < ND; d++) x[0][d] = v_part(0, d);
                in_order();
            }
            if constexpr (masked()) {
                // which of the step's keys the row sees, one a bit
                uint64_t sees = ~0ull;
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
                uint32_t found = 0;
                constexpr uint32_t top_bits = F ? 0x7f800000u : H ? 0x7c007c00u : 0x7f807f80u, one = F ? 0x00800000u : H ? 0x04000400u : 0x00800080u;
                for (uint32_t i = lane; i < KT * CH; i += 64) {
                    const u4 x = *reinterpret_cast<const u4*>(vt + i * 16);
#pragma unroll
                    for (int j = 0; j < 4; j++) found |= (x[j] & top_bits) + one;
                }
                if (odd == ~0u && __any((found & (F ? 0x80000000u : 0x80008000u)) != 0)) odd = k0;
            }
            float top[4];
#pragma unroll
            for (int i = 0; i < 4; i++) top[i] = sc[0][i];
#pragma unroll
            for (int j = 4; j < 16 * (int)NS; j++) top[j % 4] = fmaxf(top[j % 4], sc[j / 16][j % 16]);
            const float2 t2 = halves(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
            const float most_here = fmaxf(t2.x, t2.y) * c2 - kUp;
            // the reference follows the maximum only where that is far above it
            if (__any(most_here > M + (F ? 0.f : kAhead))) {
                const float Mn = fmaxf(M, most_here), f = Mn == -INFINITY ? 1.f : exp2_of(M - Mn);
                M = Mn;
                L *= f;
#pragma unroll
                for (uint32_t d = 0; d < ND; d++)
#pragma unroll
                    for (int j = 0; j < 16; j++) o[d][j] *= f;
            }
            const float Mf = M == -INFINITY ? 0.f : M;
            if constexpr (F) {
                float p[16];
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    p[j] = exp2_of(fmaf(sc[0][j], c2, -Mf));
                    L += p[j];
                }
                if (masked() && odd != ~0u) return;
#pragma unroll
                for (uint32_t j = 0; j < 16; j++) {
                    // row 8 (j / 4) + 4 half + j % 4
                    static_assert(!F || CH >= 16, "turn's form");
                    const uint32_t turned = j % 4 << 2 | j / 4 * 2 % 4;  // and half
                    const uint32_t l = opaque(n);  // computed here: one operation a product is free, registers are not
#pragma unroll
                    for (uint32_t d = 0; d < ND; d++) {
                        const float x = *reinterpret_cast<const float*>(vt + v_at + ((8 * d + l / 4) ^ half ^ turned) * 16 + (j / 4 * 8 + j % 4) * D * 4);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[j], o[d], 0, 0, 0);
                    }
                }
            } else {
                constexpr uint32_t C = 2 * NS;
                T8 p[C], rest[TWO ? C : 1];
                // weights 2 i and 2 i + 1 of p[c], and of rest[c] what their rounding left
                auto weights = [&](uint32_t c, uint32_t i) {
                    const uint32_t m = c / 2, j = c % 2 * 8 + 2 * i;
                    const float x = exp2_of(fmaf(sc[m][j], c2, -Mf)), y = exp2_of(fmaf(sc[m][j + 1], c2, -Mf));
                    typedef typename std::conditional<H, h2, b2>::type T2;
                    const T2 z = {(T)x, (T)y};
                    p[c][2 * i] = z[0], p[c][2 * i + 1] = z[1];
                    if constexpr (TWO) {
                        L += x + y;
                        const T2 r = {(T)fmaf((float)z[0], -1.f, x), (T)fmaf((float)z[1], -1.f, y)};
                        rest[c][2 * i] = r[0], rest[c][2 * i + 1] = r[1];
                    } else {
                        L = __builtin_amdgcn_fdot2(z, T2{(T)1.f, (T)1.f}, L, false);
                    }
                };
                if (masked() && odd != ~0u) {
#pragma unroll
                    for (uint32_t i = 0; i < 4 * C; i++) weights(i / 4, i % 4);
                    return;
                }
                auto add = [&](uint32_t d, const T8& v, const T8& w) {
                    if constexpr (H) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w, o[d], 0, 0, 0);
                    else o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, w, o[d], 0, 0, 0);
                };
                // a step of 16 keys: V's parts and the weights of the next between its products
                if constexpr (Q8)
#pragma unroll
                    for (uint32_t d = 0; d < ND; d++) x[0][d] = v_part(0, d);
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) weights(0, i);
                in_order();
                constexpr uint32_t EACH = TWO ? 2 * ND : ND;  // products of 16 keys
#pragma unroll
                for (uint32_t c = 0; c < C; c++)
#pragma unroll
                    for (uint32_t u = 0; u < EACH; u++) {
                        const uint32_t d = u % ND;
                        add(d, x[c % 2][d], u < ND ? p[c] : rest[TWO ? c : 0]);
                        if (c + 1 < C) {
                            if (u < ND) x[(c + 1) % 2][d] = v_part(c + 1, d);
#pragma unroll
                            for (uint32_t i = u * 4 / EACH; i < (u + 1) * 4 / EACH; i++) weights(c + 1, i);
                        }
                        behind(c * EACH + u, C * EACH);
                        in_order();
                    }
            }
        };

        // the wave waits for its own loads to LDS before it meets the others
        auto meet = [&] {
            if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        };
        if (tid == 0) bad_at = ~0u;
        look(lo);
        constexpr uint32_t each = F ? 4 : 8;  // values of a load: 2 each g + each half + ..
        u4 xq[D / 2 / each];
        {
            const size_t at = (size_t)row * a.q.row + (size_t)h * a.q.head;
            if (a.q_wide && a.q.kind == QKIND) {
#pragma unroll
                for (uint32_t g = 0; g < D / 2 / each; g++) {
                    const uint32_t d = (2 * g + half) * each;
                    xq[g] = u4{0, 0, 0, 0};
                    if (mine && d < dim) xq[g] = gld<u4>(a.q.p + (F ? 4 : 2) * (at + d));
                }
            } else {  // through the wave's part of LDS, a value at a time; 16 bits: of the type of the product
                uint8_t* part = lds[wv];
#pragma nounroll
                for (uint32_t i = lane; i < 32 * D; i += 64) {
                    const uint32_t d = i % D;
                    const size_t from = shfl64(at, i / D) + d;
                    const bool in = i / D < rows && d < dim;
                    if constexpr (F) reinterpret_cast<float*>(part)[i] = in ? elem_kind(a.q.kind, a.q.p, from) : 0.f;
                    else reinterpret_cast<uint16_t*>(part)[i] = in ? gld<uint16_t>(a.q.p + 2 * from) : (uint16_t)0;
                }
                settle();
#pragma unroll
                for (uint32_t g = 0; g < D / 2 / each; g++)
                    xq[g] = *reinterpret_cast<const u4*>(part + (n * D + (2 * g + half) * each) * (F ? 4 : 2));
                __syncthreads();  // before K and V go there
            }
        }
        if constexpr (SRC == kAny) bring(lo, 0);
        else {
#pragma unroll
            for (uint32_t r = 0; r < ROUNDS; r++) fetch(lo, 0, r);
        }
        {
            if constexpr (F) {
#pragma unroll
                for (uint32_t i = 0; i < NQ; i++) q[i] = __uint_as_float(xq[i / 4][i % 4]) * a.sign;
            } else {
                const uint32_t flip = a.sign < 0.f ? 0x80008000u : 0u;
#pragma unroll
                for (uint32_t g = 0; g < NQ; g++) xq[g] ^= flip;
                if (a.sign == 0.f) {  // 0 times what is not finite is NaN
                    constexpr uint32_t top = QKIND == F16 ? 0x7c00u : 0x7f80u;
                    auto none = [](uint32_t x) { return (x & top) == top ? 0x7fffu : 0u; };
#pragma unroll
                    for (uint32_t g = 0; g < NQ; g++)
#pragma unroll
                        for (int j = 0; j < 4; j++) xq[g][j] = none(xq[g][j]) | none(xq[g][j] >> 16) << 16;
                }
                if constexpr (Q8) {
                    // bf16 queries as f16, the row's largest finite value in [2^14, 2^15): what lies below 2^-39
                    // of it is lost, what is not finite stays so
                    uint32_t top = 0;
                    auto finite = [](uint32_t x) { return x < 0x7f800000u ? x : 0u; };
#pragma unroll
                    for (uint32_t g = 0; g < NQ; g++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            top = max(top, max(finite(xq[g][j] << 16 & 0x7fff0000u), finite(xq[g][j] & 0x7fff0000u)));
                    top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64)) >> 23;
                    const int up = 141 - (int)top;  // subnormal rows too: they lie below 2^-126
                    // kept where -inf times it is -inf, and 0 times it 0; what leaves that range is no score that
                    // counts (below 2^-80), or one that is past every other (two that differ, by 2^79 at least)
                    c2 = ldexpf(c2, -up);
                    c2 = c2 < kLeast ? kLeast : c2 > kMost && a.c2 <= kMost ? kMost : c2;
#pragma unroll
                    for (uint32_t g = 0; g < NQ; g++) {
#pragma unroll
                        for (int j = 0; j < 8; j++)
                            q[g][j] = (T)ldexpf(__uint_as_float(j & 1 ? xq[g][j / 2] & 0xffff0000u : xq[g][j / 2] << 16), up);
                        in_order();
                    }
                } else {
#pragma unroll
                    for (uint32_t g = 0; g < NQ; g++) q[g] = __builtin_bit_cast(T8, xq[g]);
                }
            }
        }
        store(0);
        look(lo + KT);
        meet();
        // A step and what comes in meanwhile.  Those that all of the workgroup's rows see whole have
        // a loop of their own, without masks, in which a buffer's place is a constant.
        const uint32_t clear = same(min(hi, (a.seen ? s.c0 : s.c0 + run.i * kTileRows / a.group + 1) / KT * KT));
        // between the products of the scores, i of n: the loads of the next step, then the pages of that after it
        auto loads = [&](uint32_t k0, uint32_t buf, uint32_t i, uint32_t n) {
#pragma unroll
            for (uint32_t r = 0; r < ROUNDS; r++)
                if (i == r * n / ROUNDS) fetch(k0 + KT, buf ^ 1, r);
            if (i == n - 1) look(k0 + 2 * KT);
        };
        // Where registers are short (EARLY false) the next step comes in behind the products.
        constexpr bool EARLY = SRC != kAny && !(D == 256 && !DIRECT);
        auto late = [&](uint32_t k0, uint32_t buf) {
            if constexpr (SRC == kAny) bring(k0 + KT, buf ^ 1);
            else if constexpr (!EARLY)
                for (uint32_t i = 0; i < ROUNDS; i++) loads(k0, buf, i, ROUNDS);
        };
        auto both = [&](uint32_t k0, auto buf) {
            step(k0, std::false_type(), buf, [&](uint32_t i, uint32_t n) {
                if constexpr (EARLY) loads(k0, buf, i, n);
            }, [&](uint32_t i, uint32_t n) {
                if constexpr (Q8 && PARTS != 0)
#pragma unroll
                    for (uint32_t j = 0; j < PARTS; j++)
                        if (i == (2 * j + 1) * n / (2 * PARTS)) store_part(buf ^ 1, j);
            });
            late(k0, buf);
            if constexpr (!Q8) store(buf ^ 1);
            meet();
        };
        uint32_t k0 = lo;
        if (rows)
            for (; k0 + 2 * KT <= clear && k0 + 2 * KT < hi; k0 += 2 * KT) {
                both(k0, std::integral_constant<uint32_t, 0>());
                both(k0 + KT, std::integral_constant<uint32_t, 1>());
            }
#pragma nounroll
        for (uint32_t buf = 0; k0 < hi; k0 += KT, buf ^= 1) {
            const bool more = k0 + KT < hi;
            if (EARLY && more)
                for (uint32_t i = 0; i < ROUNDS; i++) loads(k0, buf, i, ROUNDS);
            if (k0 < most) step(k0, std::true_type(), buf, [](uint32_t, uint32_t) {}, [](uint32_t, uint32_t) {});
            if (more) {
                late(k0, buf);
                store(buf ^ 1);
            }
            meet();
        }
        // the steps left out, a key at a time: its row goes through the wave's part of LDS
        float* part = reinterpret_cast<float*>(lds[wv]);
        if (odd != ~0u) {
            // hidden, so that nothing of this is prepared in front of the steps
            if constexpr (F) {
#pragma unroll
                for (uint32_t i = 0; i < NQ; i++) q[i] = __uint_as_float(opaque(__float_as_uint(q[i])));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < NQ; i++) {
                    u4 w = __builtin_bit_cast(u4, q[i]);
#pragma unroll
                    for (int j = 0; j < 4; j++) w[j] = opaque(w[j]);
                    q[i] = __builtin_bit_cast(T8, w);
                }
            }
            auto value = [&](const uint8_t* p, const _Float16* sc, size_t e) {
                return a.c.kind == Q8_0 ? elem<Q8_0>(p, e) * (float)gld<_Float16>(sc + e / 32) : elem_kind(a.c.kind, p, e);
            };
#pragma nounroll
            for (uint32_t t = odd; t < min(hi, most); t++) {
                const size_t at = place(t, page_of(t));
                settle();
                for (uint32_t d = lane; d < D; d += 64) {
                    part[d] = d < dim ? value(a.c.k, a.c.ks, at + d) : 0.f;
                    part[D + d] = d < dim ? value(a.c.v, a.c.vs, at + d) : 0.f;
                    if constexpr (Q8) part[D + d] = (float)(_Float16)part[D + d];  // as in the other steps
                }
                settle();
                float x = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < D / 2; i++) {
                    constexpr uint32_t each = F ? 4 : 8;
                    float y;
                    if constexpr (F) y = q[i];
                    else y = (float)q[i / 8][i % 8];
                    x = fmaf(y, part[i / each * 2 * each + each * half + i % each], x);
                }
                const float2 x2 = halves(x);
                if (a.seen ? t >= s.c0 && !(bits >> (t - s.c0) & 1) : t >= own) continue;
                const float w = exp2_of(fmaf(x2.x + x2.y, c2, M == -INFINITY ? 0.f : -M));
#pragma unroll
                for (uint32_t i = 0; i < D / 2; i++)
                    o[i / 16][i % 16] = fmaf(w, part[D + i / 16 * 32 + i % 16 / 4 * 8 + 4 * half + i % 4], o[i / 16][i % 16]);
            }
            settle();
        }
        if (bad != ~0u) atomicMin(&bad_at, bad);
        __syncthreads();
        const float2 l2 = halves(L);
        L = bad_at < own ? __builtin_nanf("") : l2.x + l2.y;
        // out of the wave's part of LDS, whole rows at a time: chunk c of four values of row n lies at c ^ n % 16 (or % 8)
        const size_t to = whole ? out_at(opaque(n)) : 0;
        const float f = !whole ? 1.f : L == 0.f ? 0.f : 1.f / L;
        constexpr uint32_t W = TILE / 128, FLIP = W / 4 < 16 ? W / 4 - 1 : 15;  // dims at a time
#pragma unroll
        for (uint32_t d0 = 0; d0 < D; d0 += W) {
#pragma unroll
            for (uint32_t d = d0 / 32; d < (d0 + W) / 32; d++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    f4 x = {o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
                    if (whole && L == 0.f) x = f4(0.f);
                    *reinterpret_cast<f4*>(part + n * W + ((8 * d - d0 / 4 + 2 * i + half) ^ (n & FLIP)) * 4) = x * f;
                }
            settle();
            for (uint32_t i = lane; i < 32 * W / 4; i += 64) {
                const uint32_t line = i / (W / 4), c = i % (W / 4);
                const f4 x = *reinterpret_cast<const f4*>(part + line * W + (c ^ (line & FLIP)) * 4);
                const size_t at = shfl64(to, line);
                if (line >= rows) continue;
                if (whole) put_row(a, dim, at, d0 + 4 * c, x);
                else *reinterpret_cast<f4*>(part_o(a, slot) + (wv * 32 + line) * D + d0 + 4 * c) = x;
            }
            settle();
        }
        if (!whole && mine && half == 0) part_ml(a, slot)[wv * 32 + n] = make_float2(M, L);
        __syncthreads();
    } while (run.next(a));
}

// out of the tiles that several workgroups hold parts of: a workgroup for the first
// run that begins inside a tile and 1,024 of its values, four a thread.  The parts: the
// second slot of the run in front, and the first slot of those up to the last.  Bound by
// what it reads, which is in the caches: 9 to 18 us behind a full grid.
__global__ __launch_bounds__(kBlock) void k_page_many_join(PageMany a) {
    const uint32_t D = a.wide, w = blockIdx.x + 1;
    const uint32_t runs = min(*runs_of(a), a.runs);
    if (w >= runs) return;
    const ManyMark m = *mark_of(a, w);
    if (!m.rows || m.rows > kTileRows || m.kv >= a.c.kvheads) return;
    const uint32_t at = (blockIdx.y * kBlock + threadIdx.x) * 4, line = at / D, d = at % D, last = min(m.last, runs - 1);
    if (line >= m.rows) return;
    float M = -INFINITY, L = 0.f;
    f4 O = {0.f, 0.f, 0.f, 0.f};
    constexpr uint32_t kAhead = 4;  // parts on their way
    for (uint32_t p0 = w - 1; p0 <= last; p0 += kAhead) {
        float2 ml[kAhead];
        f4 o[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            const uint32_t p = min(p0 + i, last);
            const size_t slot = (size_t)p * 2 + (p == w - 1);
            ml[i] = part_ml(a, slot)[line];
            o[i] = *reinterpret_cast<const f4*>(part_o(a, slot) + line * D + d);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            if (p0 + i > last) break;
            const float Mn = fmaxf(M, ml[i].x), Mf = Mn == -INFINITY ? 0.f : Mn;
            const float f = exp2_of(M - Mf), e = exp2_of(ml[i].x - Mf);
            M = Mn;
            L = fmaf(ml[i].y, e, L * f);
            // a part without a step has no values
#pragma unroll
            for (int j = 0; j < 4; j++) O[j] = ml[i].x == -INFINITY ? O[j] * f : fmaf(o[i][j], e, O[j] * f);
        }
    }
    const uint32_t r = m.row + line, row = r / a.group;
    if (row >= a.n) return;
    put_row(a, a.c.dim, (size_t)row * a.out.row + (size_t)(m.kv * a.group + r % a.group) * a.out.head, d, L == 0.f ? f4(0.f) : O * (1.f / L));
}

// ---------------------------------------------------------------- launches --
// The type of a call's products and the width of its tiles; what its rows are aligned to.
void page_many_plan(PageMany& a, uint32_t cus) {
    const uint32_t d = a.c.dim, es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2;
    a.group = a.heads / a.c.kvheads;
    a.wide = d <= 64 ? 64 : d <= 128 ? 128 : 256;
    auto aligned = [](const Heads& h, uint32_t bytes) {
        const uint64_t e = h.kind == F32 ? 4 : 2;
        return (((uintptr_t)h.p | h.row * e | h.head * e) % bytes) == 0;
    };
    a.q_wide = d % 8 == 0 && aligned(a.q, 16);
    a.out_wide = aligned(a.out, a.out.kind == F32 ? 16 : 8);
    a.kv_wide = d % 8 == 0 && (((uintptr_t)a.c.k | (uintptr_t)a.c.v | (a.c.ps | a.c.ts | a.c.hs) * es) % std::min(8 * es, 16u)) == 0;
    // Products of 16 bits: of the cache's own type, or of f16 where bf16 queries read Q8_0 (the two
    // prompts over Q8_0 0.545 ms, 2.27 in 32 bits); wider heads' codes and registers do not fit.
    a.narrow = a.q.kind != F32 && a.out.kind != F32 &&
               (a.c.kind == a.q.kind || (a.c.kind == Q8_0 && a.kv_wide && d <= 128 && a.q.kind == BF16 && a.out.kind == BF16));
    // What a tile's start and end cost, in keys: queries in, values out (256 rather than 32: 16,381
    // tokens 3.29 -> 3.23 ms, 24 prompts 0.93 -> 0.69, 48 trees 107 -> 89 us), and the least that a run
    // is worth having (128, of four steps less than one for its start: a tree behind 517 keys 20.6 us,
    // with 64 23.4, with 256 22.2; f32, where a key costs eight times as much, 32, and 16 or 64 take
    // as long: 517 tokens 60 us).
    a.tile_keys = a.narrow ? 256 : 32;
    a.run_keys = a.narrow ? 128 : 32;
    a.one_page = a.c.page % std::max(1024 / (a.wide * es), 1u) == 0 && a.c.ps * es >> 32 == 0 && (unsigned __int128)a.c.page * a.c.ts * es >> 32 == 0;
    // t / page for t < 2^31: 2 t * ceil(2^(31 + log) / page) >> 32 + log
    a.page_log = 0;
    while ((1ull << a.page_log) < a.c.page) a.page_log++;
    a.page_mul = (uint32_t)(((1ull << (31 + a.page_log)) + a.c.page - 1) / a.c.page);
    a.sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f;
    a.c2 = a.scale == 0.f ? 1.f : std::max(std::fabs(a.scale) * kLog2e, kLeast);
    const uint64_t tiles = ((uint64_t)a.n * a.group / kTileRows + a.r.batch) * a.c.kvheads;
    const uint64_t most = tiles * (a.r.most / a.run_keys + 2);
    // A run for each workgroup that is there at once: two a unit by registers (one: 16,381 tokens 3.23 ->
    // 4.04 ms, 24 prompts 0.69 -> 0.90), and one of the kernels with 256 values, or Q8_0's codes of 128, whose
    // registers leave room for one (two, one behind the other: 48 trees of 256 values 194 -> 212 us, Q8_0 0.545 ->
    // 0.559 ms; 24 prompts of 256 1.68 either way).
    const bool alone = a.wide == 256 || (a.narrow && a.c.kind == Q8_0 && a.wide == 128);
    a.runs = (uint32_t)std::min<uint64_t>(cus * (alone ? 1 : 2), std::max<uint64_t>(most, 1));
}

template <class T, uint32_t SRC> static void launch_many(const PageMany& a, hipStream_t s) {
    const dim3 grid((a.runs + kXcds - 1) / kXcds * kXcds), block(kBlock);
    if (a.wide == 64) hipLaunchKernelGGL((k_page_many<T, 64, SRC>), grid, block, 0, s, a);
    else if (a.wide == 128) hipLaunchKernelGGL((k_page_many<T, 128, SRC>), grid, block, 0, s, a);
    else if constexpr (SRC == kDirect || SRC == kAny || (SRC == Q8_0 && std::is_same<T, float>::value)) hipLaunchKernelGGL((k_page_many<T, 256, SRC>), grid, block, 0, s, a);
}
void launch_page_many(const PageMany& a, hipStream_t s) {
    // Rows straight to LDS (16,381 tokens 3.23 ms, value by value 4.44; 48 trees 89 us, 121) where a
    // wave's load of them lies in one page, which it finds once.
    const bool direct = a.kv_wide && a.one_page && a.c.dim == a.wide;
    if (a.narrow) {
        if (a.c.kind == Q8_0) launch_many<_Float16, Q8_0>(a, s);
        else if (a.c.kind == F16) direct ? launch_many<_Float16, kDirect>(a, s) : launch_many<_Float16, kAny>(a, s);
        else direct ? launch_many<bf16_t, kDirect>(a, s) : launch_many<bf16_t, kAny>(a, s);
    } else if (a.c.kind == F32 && direct) launch_many<float, kDirect>(a, s);
    else if (a.c.kind == F32 || !a.kv_wide || (a.wide == 256 && a.c.kind != Q8_0)) launch_many<float, kAny>(a, s);
    else if (a.c.kind == F16) launch_many<float, F16>(a, s);
    else if (a.c.kind == BF16) launch_many<float, BF16>(a, s);
    else launch_many<float, Q8_0>(a, s);
    if (a.runs > 1)
        hipLaunchKernelGGL(k_page_many_join, dim3(a.runs - 1, kTileRows * a.wide / (4 * kBlock)), dim3(kBlock), 0, s, a);
}

}  // namespace qh
