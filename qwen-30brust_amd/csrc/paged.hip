// The key-value cache in pages: appending tokens (per-head RMSNorm and NeoX
// RoPE of q and k on the way) and the attention of one new token per sequence.
//
// A key t of sequence b lies in slot t % page of page table[b][t / page].
// Page ids come from the caller's device memory: every one is compared with the
// pool's size before it is used.  A sequence whose length or page ids are out
// of range gets NaN from the attention, and an append to such a page is left
// out.
#include <algorithm>
#include <type_traits>

#include "page_runs.hpp"
#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

// ------------------------------------------------------------------ append --
// For every token and head (q's heads, then k's, then v's):
//   y = x / sqrt(sum x^2 / dim + eps) * w              (q and k, with weights)
//   (y_i, y_j) = (y_i cos - y_j sin, y_j cos + y_i sin), j = i + dim / 2
// in 32 bits, rounded once to the type it is stored in.  Q8_0: per 32 values
// d = f16(max |y| / 127) and codes round(y / d), the blocks of GGML's format with
// codes and scales each in an array of their own.  GGML's own quantiser multiplies
// by the inverse of the unrounded scale and takes ties away from 0: its codes can be
// one off from these, which are the nearest to y in the scale that is stored.
// A token outside the table of angles becomes NaN.

// Where token i goes: into place t of sequence b, or nowhere.  By a wave.
struct Place {
    uint32_t b;
    int32_t t;
    bool live;
};
__device__ __forceinline__ Place place_of(const PageAppend& a, uint32_t i) {
    const uint32_t lane = threadIdx.x & 63;
    Place p{i, 0, true};
    int32_t at = 0, count = 1;  // the token's number in its sequence, and of how many
    if (a.first) {
        // the last sequence whose first token is not behind it
        uint32_t before = 0;
        for (uint32_t j = 0; j <= a.r.batch; j += 64) {
            const bool le = j + lane <= a.r.batch && gld<int32_t>(a.first + min(j + lane, a.r.batch)) <= (int32_t)i;
            before += __popcll(__ballot(le));
        }
        p.live = before > 0 && before <= a.r.batch;
        p.b = p.live ? before - 1 : 0;
        const int32_t f = gld<int32_t>(a.first + p.b);
        at = (int32_t)i - f;
        count = gld<int32_t>(a.first + p.b + 1) - f;
    }
    const int32_t len = p.live ? length_of(a.r, p.b) : -1;
    p.t = len - count + at;
    p.live = p.live && p.t >= 0 && p.t < len;
    return p;
}
// The cache's page of a place, or -1.
__device__ __forceinline__ int32_t page_of(const PageAppend& a, const Place& p) {
    const int32_t page = gld<int32_t>(a.r.table + p.b * a.r.stride + (uint32_t)p.t / a.c.page);
    return page < 0 || (uint32_t)page >= a.c.count ? -1 : page;
}
__device__ __forceinline__ size_t slot_of(const PageAppend& a, const Place& p, int32_t page, uint32_t g) {
    return (size_t)page * a.c.ps + (size_t)((uint32_t)p.t % a.c.page) * a.c.ts + g * a.c.hs;
}

typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef bf16_t b4 __attribute__((ext_vector_type(4)));
typedef uint16_t u4h __attribute__((ext_vector_type(4)));

// Elements i .. i + 3 of p, aligned so.
__device__ __forceinline__ f4 four(uint32_t kind, const uint8_t* p, size_t i) {
    if (kind == F32) return gld<f4>(p + 4 * i);
    if (kind == F16) return __builtin_convertvector(gld<h4>(p + 2 * i), f4);
    const u4h u = gld<u4h>(p + 2 * i);
    f4 x;
    for (int j = 0; j < 4; j++) x[j] = __uint_as_float((uint32_t)u[j] << 16);
    return x;
}
__device__ __forceinline__ void put_four(uint32_t kind, uint8_t* p, size_t i, f4 x) {
    if (kind == F32) *reinterpret_cast<f4*>(p + 4 * i) = x;
    else if (kind == F16) *reinterpret_cast<h4*>(p + 2 * i) = __builtin_convertvector(x, h4);
    else *reinterpret_cast<b4*>(p + 2 * i) = __builtin_convertvector(x, b4);
}
// The Q8_0 code of a value: fine, whether its block is finite, f the block's scale.
// Of 11 bits of f the middle between two codes is an f32 value, and the quotient
// of any other, rounded to the nearest, stays on its side of the middle.
__device__ __forceinline__ int32_t code_of(float x, bool fine, float f) {
    return fine && f > 0.f ? (int32_t)fminf(fmaxf(rintf(x / f), -127.f), 127.f) : 0;
}

// Heads of 8 L values, all rows aligned to four elements: a wave takes 64 / L
// heads of a token, a lane four values of the first half and the four they turn
// with, so nothing is exchanged but the norm's sum and, in Q8_0, a block's maximum
// (8 lanes).  Bound by memory where there are many tokens: 2,001 tokens of 32 + 2 x 4
// heads of 128 from f32 into f16 take 16 us (79 MB, 4.9 TB/s), 48 with a wave a head; 64
// tokens of a decode step 4.5 us, the four dependent look-ups of a place.
template <uint32_t L> __global__ __launch_bounds__(kBlock) void k_page_append(PageAppend a, uint32_t groups) {
    constexpr uint32_t D = 8 * L;
    const uint32_t lane = threadIdx.x & 63, l = lane % L;
    const uint32_t unit = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const uint32_t i = a.from + unit / groups, h = unit % groups * (64 / L) + lane / L;
    if (i >= a.n) return;
    const bool mine = h < a.heads + 2 * a.c.kvheads;
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.c.kvheads;
    const uint32_t g = !mine ? 0 : is_q ? h : is_k ? h - a.heads : h - a.heads - a.c.kvheads;
    const Heads& src = is_q ? a.q : is_k ? a.k : a.v;
    const size_t from = i * src.row + g * src.head + 4 * l;
    f4 x = four(src.kind, src.p, from), y = four(src.kind, src.p, from + D / 2);
    const Place p = place_of(a, i);
    if (!p.live || !mine) return;
    const float* w = is_q ? a.qw : is_k ? a.kw : nullptr;
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
#pragma unroll
        for (uint32_t s = 1; s < L; s <<= 1) ss += __shfl_xor(ss, s, 64);
        const float s = 1.f / sqrtf(ss / (float)D + a.eps);
        x = x * s * gld<f4>(w + 4 * l);
        y = y * s * gld<f4>(w + D / 2 + 4 * l);
    }
    if (a.rope && (is_q || is_k)) {
        const int32_t at = a.pos ? gld<int32_t>(a.pos + i) : p.t;
        const bool in = at >= 0 && (uint32_t)at < a.rope_rows;
        const float* row = reinterpret_cast<const float*>(a.rope + (size_t)(in ? at : 0) * (D / 2)) + 8 * l;
        const f4 c0 = gld<f4>(row), c1 = gld<f4>(row + 4);
        const f4 c = {c0.x, c0.z, c1.x, c1.z}, s = {c0.y, c0.w, c1.y, c1.w};
        const f4 turned = x * c - y * s;
        y = y * c + x * s;
        x = turned;
        if (!in) x = y = __builtin_nanf("");
    }
    if (is_q) {
        const size_t o = i * a.qo.row + g * a.qo.head + 4 * l;
        put_four(a.qo.kind, a.qo.p, o, x);
        put_four(a.qo.kind, a.qo.p, o + D / 2, y);
        return;
    }
    const int32_t page = page_of(a, p);
    if (page < 0) return;
    const size_t o = slot_of(a, p, page, g) + 4 * l;
    uint8_t* to = is_k ? a.c.k : a.c.v;
    if (a.c.kind != Q8_0) {
        put_four(a.c.kind, to, o, x);
        put_four(a.c.kind, to, o + D / 2, y);
        return;
    }
    _Float16* scale = is_k ? a.c.ks : a.c.vs;
#pragma unroll
    for (uint32_t half = 0; half < 2; half++) {
        const f4 z = half ? y : x;
        float m = 0.f;
        bool fine = true;
#pragma unroll
        for (int j = 0; j < 4; j++) m = fmaxf(m, fabsf(z[j])), fine &= finite_f(z[j]);
        m = fine ? m : __builtin_inff();  // one that is not finite gives its block a scale of NaN
#pragma unroll
        for (uint32_t s = 1; s < 8; s <<= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
        fine = finite_f(m);
        const _Float16 dq = fine ? (_Float16)(m / 127.f) : (_Float16)__builtin_nanf("");
        uint32_t codes = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) codes |= (uint32_t)(code_of(z[j], fine, (float)dq) & 255) << 8 * j;
        const size_t e = o + half * (D / 2);
        *reinterpret_cast<uint32_t*>(to + e) = codes;
        if (l % 8 == 0) scale[e / 32] = dq;
    }
}

// Any other width up to 256 and alignment: a wave per token and head, every 64th
// value to a lane.  2,001 tokens of 32 + 2 x 4 heads of 96 take 47 us.
__global__ __launch_bounds__(kBlock) void k_page_append_any(PageAppend a) {
    constexpr uint32_t E = kPageMaxDim / 64;
    __shared__ float turn[kWaves][kPageMaxDim];
    const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6, d = a.c.dim;
    const uint32_t slots = a.heads + 2 * a.c.kvheads;
    const uint32_t unit = blockIdx.x * kWaves + wv;
    const uint32_t i = min(a.from + unit / slots, a.n - 1);
    const uint32_t h = unit % slots;
    const Place p = place_of(a, i);
    const bool live = p.live && a.from + unit / slots < a.n;
    const bool is_q = h < a.heads, is_k = !is_q && h < a.heads + a.c.kvheads;
    const uint32_t g = is_q ? h : is_k ? h - a.heads : h - a.heads - a.c.kvheads;
    const Heads& src = is_q ? a.q : is_k ? a.k : a.v;
    float x[E];
#pragma unroll
    for (uint32_t j = 0; j < E; j++) {
        const uint32_t e = lane + 64 * j;
        x[j] = live && e < d ? elem_kind(src.kind, src.p, i * src.row + g * src.head + e) : 0.f;
    }
    const float* w = is_q ? a.qw : is_k ? a.kw : nullptr;
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < E; j++) ss = fmaf(x[j], x[j], ss);
        const float s = 1.f / sqrtf(wave_sum(ss) / (float)d + a.eps);
#pragma unroll
        for (uint32_t j = 0; j < E; j++) {
            const uint32_t e = lane + 64 * j;
            if (e < d) x[j] = x[j] * s * gld<float>(w + e);
        }
    }
    if (a.rope && (is_q || is_k)) {
        const int32_t at = live ? (a.pos ? gld<int32_t>(a.pos + i) : p.t) : 0;
        const bool in = at >= 0 && (uint32_t)at < a.rope_rows;
        const float2* row = a.rope + (size_t)(in ? at : 0) * (d / 2);
#pragma unroll
        for (uint32_t j = 0; j < E; j++) turn[wv][lane + 64 * j] = x[j];
        // the row is this wave's own
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (uint32_t j = 0; j < E; j++) {
            const uint32_t e = lane + 64 * j;
            if (e < d) {
                const bool low = e < d / 2;
                const float2 cs = gld<float2>(row + (low ? e : e - d / 2));
                const float y = turn[wv][low ? e + d / 2 : e - d / 2];
                const float r = low ? x[j] * cs.x - y * cs.y : y * cs.y + x[j] * cs.x;
                x[j] = in ? r : __builtin_nanf("");
            }
        }
    }
    if (!live) return;
    if (is_q) {
#pragma unroll
        for (uint32_t j = 0; j < E; j++)
            if (lane + 64 * j < d) put_kind(a.qo.kind, a.qo.p, i * a.qo.row + g * a.qo.head + lane + 64 * j, x[j]);
        return;
    }
    const int32_t page = page_of(a, p);
    if (page < 0) return;
    const size_t o = slot_of(a, p, page, g);
    uint8_t* to = is_k ? a.c.k : a.c.v;
    if (a.c.kind != Q8_0) {
#pragma unroll
        for (uint32_t j = 0; j < E; j++)
            if (lane + 64 * j < d) put_kind(a.c.kind, to, o + lane + 64 * j, x[j]);
        return;
    }
    _Float16* scale = is_k ? a.c.ks : a.c.vs;
#pragma unroll
    for (uint32_t j = 0; j < E; j++) {
        // 32 lanes hold a block; one that is not finite gets a scale of NaN
        float m = fabsf(x[j]);
        bool fine = finite_f(x[j]);
#pragma unroll
        for (uint32_t s = 1; s < 32; s <<= 1) {
            m = fmaxf(m, __shfl_xor(m, s, 64));
            fine &= (bool)__shfl_xor((int)fine, s, 64);
        }
        const uint32_t e = lane + 64 * j;
        if (e >= d) continue;
        const _Float16 dq = fine ? (_Float16)(m / 127.f) : (_Float16)__builtin_nanf("");
        reinterpret_cast<int8_t*>(to)[o + e] = (int8_t)code_of(x[j], fine, (float)dq);
        if (lane % 32 == 0) scale[(o + e) / 32] = dq;
    }
}

// Whether a run of heads, or the cache, is aligned to four elements in every row.
static bool by_four(const void* p, size_t row, size_t head, size_t es) {
    return ((uintptr_t)p % (4 * es) | row % 4 | head % 4) == 0;
}
static bool by_four(const Heads& h) { return !h.p || by_four(h.p, h.row, h.head, h.kind == F32 ? 4 : 2); }

// f(args, waves) for ranges of tokens, `each` waves a token: a launch has fewer than
// 2^32 threads.
constexpr uint32_t kAppendWaves = 1u << 25;
template <class F> static void by_tokens(PageAppend a, uint32_t each, F f) {
    const uint32_t n = a.n, most = kAppendWaves / each;  // heads <= 65535 and as many KV heads twice
    for (uint32_t done = 0; done < n; done = a.n) {
        a.from = done;
        a.n = std::min(n, done + most);
        f(a, dim3(((a.n - done) * each + kWaves - 1) / kWaves));
    }
}

void launch_page_append(const PageAppend& args, hipStream_t s) {
    const uint32_t slots = args.heads + 2 * args.c.kvheads, d = args.c.dim;
    const size_t es = args.c.kind == F32 ? 4 : args.c.kind == Q8_0 ? 1 : 2;
    const uintptr_t floats = (uintptr_t)args.qw | (uintptr_t)args.kw | (uintptr_t)args.rope;
    const dim3 block(kBlock);
    if ((d == 64 || d == 128 || d == 256) && by_four(args.q) && by_four(args.qo) && by_four(args.k) && by_four(args.v) &&
        by_four(args.c.k, args.c.ts, args.c.hs, es) && by_four(args.c.v, args.c.ps, 0, es) && floats % 16 == 0) {
        const uint32_t per = 512 / d, groups = (slots + per - 1) / per;
        by_tokens(args, groups, [&](const PageAppend& a, dim3 grid) {
            if (d == 64) hipLaunchKernelGGL(k_page_append<8>, grid, block, 0, s, a, groups);
            else if (d == 128) hipLaunchKernelGGL(k_page_append<16>, grid, block, 0, s, a, groups);
            else hipLaunchKernelGGL(k_page_append<32>, grid, block, 0, s, a, groups);
        });
        return;
    }
    by_tokens(args, slots, [&](const PageAppend& a, dim3 grid) { hipLaunchKernelGGL(k_page_append_any, grid, block, 0, s, a); });
}

// --------------------------------------------------------------- attention --
//   s_t = scale * log2(e) * q . k_t,  m = max s_t,  l = sum 2^(s_t - m),
//   o = sum 2^(s_t - m) v_t / l
// over the keys of one sequence, everything in 32 bits.  A row with no keys, or
// whose scores are all -inf, is zeros.
//
// Work is counted in steps of 32 keys of a unit (a sequence, one of its KV heads
// and `per` of that head's query heads), a sequence without keys as one, and
// kUnitCost more for its start and end.  All units' steps, one behind the other,
// are dealt to the workgroups in equal runs (page_runs.hpp), whatever the lengths: a
// ragged batch and one long sequence both fill the chip.  A run may hold several
// units; one that it holds whole goes straight to out, and at most the first and the
// last it holds in part: their (m, l, o) go to the workgroup's two slots, and
// k_page_join folds them.  Lengths are known on the device only, so every workgroup
// finds its run from them (a wave per 64 lengths and pass).  It reads them more than
// once: lengths that change meanwhile give a wrong result, but every loop ends with
// the batch, and the join takes its slots from the noted steps, in range.
constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kStep = 32;     // keys
constexpr uint32_t kPerMost = 8;   // query heads of a unit
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32

__device__ __forceinline__ uint32_t steps_of(int32_t len) {
    return (len <= 0 ? 1u : ((uint32_t)len + kStep - 1) / kStep) + kUnitCost;
}
// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ uint32_t same(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t same64(uint64_t v) { return (uint64_t)same((uint32_t)(v >> 32)) << 32 | same((uint32_t)v); }
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) { return __shfl((unsigned long long)v, lane, 64); }

// The steps of sequences [0, end), by a wave.
__device__ __forceinline__ uint64_t steps_before(const PageAttn& a, uint32_t end) {
    uint64_t n = 0;
    for (uint32_t j = threadIdx.x & 63; j < end; j += 64) n += steps_of(length_of(a.r, j));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor((unsigned long long)n, o, 64);
    return same64(n);
}
// A workgroup's run: unit u (of a.units) of sequence b, from step r of its
// `steps`; `left` steps to go.  Of a unit in hand: key(), the first key, and
// end(), behind the last.
struct Run {
    uint32_t b, u, r, steps;
    int32_t len;
    uint64_t x, left;  // the step's number
    __device__ __forceinline__ bool start(const PageAttn& a) {
        const uint32_t lane = threadIdx.x & 63;
        const uint64_t total = a.units * steps_before(a, a.r.batch), runs = runs_of(total, a.runs);
        if (blockIdx.x >= runs) return false;
        x = run_begin(total, runs, blockIdx.x);
        left = run_begin(total, runs, blockIdx.x + 1) - x;
        if (blockIdx.x == 0 && threadIdx.x == 0) a.begin[a.r.batch] = total;
        uint64_t base = 0;
        for (uint32_t j = 0;; j += 64) {
            if (j >= a.r.batch) return false;  // only where lengths changed meanwhile
            const uint32_t n = j + lane < a.r.batch ? steps_of(length_of(a.r, j + lane)) : 0;
            uint64_t sum = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint64_t t = __shfl_up((unsigned long long)sum, o, 64);
                if (lane >= (uint32_t)o) sum += t;
            }
            const uint64_t past = __ballot(a.units * (base + sum) > x);
            if (past) {
                const int at = __ffsll((unsigned long long)past) - 1;
                b = same(j + at);
                steps = same(__shfl(n, at, 64));
                const uint64_t rest = same64(x - a.units * (base + shfl64(sum - n, at)));
                u = (uint32_t)div64(rest, steps);
                r = (uint32_t)(rest - (uint64_t)u * steps);
                break;
            }
            base += same64(shfl64(sum, 63));
        }
        len = (int32_t)same(length_of(a.r, b));
        note(a);
        return true;
    }
    // for k_page_join
    __device__ __forceinline__ void note(const PageAttn& a) const {
        if (u == 0 && r == 0 && threadIdx.x == 0) a.begin[b] = x;
    }
    // steps of the unit in hand
    __device__ __forceinline__ uint32_t here() const { return (uint32_t)min((uint64_t)(steps - r), left); }
    __device__ __forceinline__ uint32_t key() const { return (max(r, kUnitCost) - kUnitCost) * kStep; }
    __device__ __forceinline__ uint32_t end() const {
        const uint32_t n = len < 0 ? 0u : (uint32_t)len, s = max(r + here(), kUnitCost) - kUnitCost;
        return r + here() == steps ? n : min(n, s * kStep);
    }
    __device__ __forceinline__ bool none() const { return r + here() <= kUnitCost; }  // no step of its own
    __device__ __forceinline__ bool head() const { return r <= kUnitCost; }           // its first step
    __device__ __forceinline__ bool whole() const { return head() && r + here() == steps; }
    __device__ __forceinline__ bool next(const PageAttn& a) {
        x += here();
        left -= here();
        if (left == 0) return false;
        r = 0;
        if (++u == a.units) {
            u = 0;
            if (++b == a.r.batch) return false;  // as in start()
            len = (int32_t)same(length_of(a.r, b));
            steps = steps_of(len);
            note(a);
        }
        return true;
    }
};

// Where head n of a unit goes: a whole unit to out, a part to a slot of the
// workgroup (0: a part that starts inside its unit, 1: one that starts with it).
__device__ __forceinline__ void store_part(const PageAttn& a, const Run& w, uint32_t h, uint32_t n, uint32_t j, float M,
                                           float L, float O) {
    if (w.whole()) {
        put_kind(a.out.kind, a.out.p, w.b * a.out.row + h * a.out.head + j, L == 0.f ? 0.f : O / L);
        if (a.sum && j == 0) a.sum[(size_t)w.b * a.heads + h] = make_float2(M, L);
        return;
    }
    const size_t slot = ((size_t)blockIdx.x * 2 + w.head()) * a.per + n;
    a.o[slot * a.c.dim + j] = O;
    if (j == 0) a.ml[slot] = make_float2(M, L);
}

// Elements e .. e + 3 of a row of d at p + at; `one`: aligned to four, d too.
template <uint32_t K> __device__ __forceinline__ f4 row4(const uint8_t* p, size_t at, uint32_t e, uint32_t d, bool one) {
    if (one) {
        if constexpr (K == Q8_0) {
            const uint32_t w = gld<uint32_t>(p + at + e);
            return f4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)((int32_t)w >> 24)};
        } else {
            return four(K, p, at + e);
        }
    }
    f4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (uint32_t c = 0; c < 4; c++)
        if (e + c < d) x[c] = elem<K>(p, at + e + c);
    return x;
}

// One query head, any head width up to 8 E: eight lanes share a key, with every
// eighth four elements of its row each, and keep the (m, l, o) of their own keys, so
// there is no barrier before the merge at the end.  Every query head reads its keys
// again, from L2: 48 ragged histories of up to 4,096 keys of width 96, eight heads a KV
// head, 316 us in bf16 (2.5 times that with an element a load), some seven times what
// k_page_attn16 takes for width 128.
template <uint32_t K, int E>
__global__ __launch_bounds__(kBlock) void k_page_attn_any(PageAttn a) {
    __shared__ float red[kWaves][8 * E], rm[kWaves], rl[kWaves];
    const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6, kl = lane >> 3, p = lane & 7, d = a.c.dim;
    constexpr size_t ES = K == F32 ? 4 : K == Q8_0 ? 1 : 2;
    const bool one = (d % 4 | ((uintptr_t)a.c.k | (uintptr_t)a.c.v) % (4 * ES) | (a.c.ps | a.c.ts | a.c.hs) % 4) == 0;
    Run w;
    if (!w.start(a)) return;
    do {
        const uint32_t h = w.u, b = w.b, g = h / (a.heads / a.c.kvheads);
        const uint32_t k0 = w.key(), k1 = w.end();
        if (w.none()) continue;
        constexpr int N = E / 4;
        f4 q[N], o[N];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t e = 4 * (p + 8 * i);
#pragma unroll
            for (uint32_t c = 0; c < 4; c++)
                q[i][c] = e + c < d ? elem_kind(a.q.kind, a.q.p, b * a.q.row + h * a.q.head + e + c) : 0.f;
            o[i] = f4{0.f, 0.f, 0.f, 0.f};
        }
        bool bad = w.len < 0;
        for (uint32_t t = k0 + 8 * wv + kl; t - kl < k1; t += 8 * kWaves) {  // wave-uniform
            const uint32_t tt = min(t, k1 - 1);
            int32_t page = gld<int32_t>(a.r.table + b * a.r.stride + tt / a.c.page);
            if (page < 0 || (uint32_t)page >= a.c.count) {
                bad = true;
                page = 0;
            }
            const size_t at = (size_t)page * a.c.ps + (size_t)(tt % a.c.page) * a.c.ts + g * a.c.hs;
            f4 kr[N], vr[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const uint32_t e = 4 * (p + 8 * i);
                kr[i] = vr[i] = f4{0.f, 0.f, 0.f, 0.f};
                if (e < d) {
                    kr[i] = row4<K>(a.c.k, at, e, d, one);
                    vr[i] = row4<K>(a.c.v, at, e, d, one);
                    if constexpr (K == Q8_0) {
                        kr[i] *= (float)gld<_Float16>(a.c.ks + (at + e) / 32);
                        vr[i] *= (float)gld<_Float16>(a.c.vs + (at + e) / 32);
                    }
                }
            }
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) s = fmaf(q[i][c], kr[i][c], s);
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) s += __shfl_xor(s, x, 64);
            s *= a.scale * kLog2e;
            if (t >= k1) continue;  // not 0 times the value of a key past the end
            if (a.score && p == 0) a.score[((size_t)b * a.heads + h) * a.score_row + t] = s;
            const float M = fmaxf(m, s), Mf = M == -INFINITY ? 0.f : M;
            const float alpha = exp2_of(m - Mf), e = exp2_of(s - Mf);
            m = M;
            l = fmaf(l, alpha, e);
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) o[i][c] = fmaf(e, vr[i][c], o[i][c] * alpha);
        }
        if (bad) l = __builtin_nanf("");
        // the wave's eight lane groups, then the waves
        float M = m;
#pragma unroll
        for (int x = 8; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
        const float e = exp2_of(m - (M == -INFINITY ? 0.f : M));
        l *= e;
#pragma unroll
        for (int i = 0; i < N; i++) o[i] *= e;
#pragma unroll
        for (int x = 8; x < 64; x <<= 1) {
            l += __shfl_xor(l, x, 64);
#pragma unroll
            for (int i = 0; i < E; i++) o[i / 4][i % 4] += __shfl_xor(o[i / 4][i % 4], x, 64);
        }
        __syncthreads();  // the unit before has been stored
        if (kl == 0) {
#pragma unroll
            for (int i = 0; i < E; i++) red[wv][4 * (p + 8 * (i / 4)) + i % 4] = o[i / 4][i % 4];
        }
        if (lane == 0) {
            rm[wv] = M;
            rl[wv] = l;
        }
        __syncthreads();
        float Ma = -INFINITY, L = 0.f;
        for (int x = 0; x < kWaves; x++) Ma = fmaxf(Ma, rm[x]);
        const float Mf = Ma == -INFINITY ? 0.f : Ma;
        for (int x = 0; x < kWaves; x++) L = fmaf(rl[x], exp2_of(rm[x] - Mf), L);
        for (uint32_t j = threadIdx.x; j < d; j += kBlock) {
            float O = 0.f;
            for (int x = 0; x < kWaves; x++) O = fmaf(red[x][j], exp2_of(rm[x] - Mf), O);
            store_part(a, w, h, 0, j, Ma, L, O);
        }
    } while (w.next(a));
}

// -------------------------------------------- attention on the matrix cores --
// A wave takes 32 keys a step and up to eight query heads of one KV head, and
// keeps K, V, scores, weights and sums in its registers:
//   S^T = K Q^T      v_mfma_f32_16x16x32: rows are 16 keys, columns the heads
//                    (twice: column n and n + 8 hold head n);
//   O^T = V^T P^T    the same instruction: rows are 16 dims, the 32 k slots the
//                    step's keys.
// Lane (g = lane / 16, n = lane % 16) gets the scores of keys 4 g + r and 16 +
// 4 g + r of its head, which are the k slots 8 g .. 8 g + 7 that the second
// product wants of it when the slots' keys are numbered that way: the weights
// need no exchange between lanes, and the row of dims 8 n .. 8 n + 7 of each of
// those eight keys, one 16-byte load, gives the lane the eight A tiles by a
// transposition of pairs of registers (v_perm_b32).
// Weights go in as two parts of 16 bits, p = hi + lo: the hi parts in columns 0
// to 7, the lo parts in columns 8 to 15, so that the second part costs no
// instruction; their sums are added at the end.  (Where a value is not finite
// the hi column alone says so.)  That leaves 2^-17 (bf16) or 2^-23 (f16) of a
// weight off; one part would leave 2^-8 or 2^-11.  Outputs of 16 bits are rounded by
// more; those of 32 bits take k_page_attn32.  f16's lo part is 2^11 times the rest, so
// that it is as large as the hi part and holds weights down to 2^-43 of the largest (the
// rest as it is would end at 2^-32, and keys that together count beside one that much
// heavier would be lost: one whose value is 0 above 8,191 others).
// The running reference m moves only when a score is kRoom above it, to 8 - kRoom
// above that score: nearly never, so the sums are rarely rescaled.  Weights of f16
// reach 2^15 (kRoom 15; a sum of 2^31 f16 values is far from 32 bits' end), those of
// bf16 and of 32-bit products 1 (kRoom 0): a value near the end of its range comes
// out as it is as long as the values' sum is in range.
// Q8_0: codes are exact in f16 (byte | 0x6400 is 1024 + byte), a block's scale
// multiplies its 32-dim product in 32 bits, and code * scale of V goes in as two
// f16 parts (the product and its rounding error, by a fused multiply-add);
// values past f16's range come out not finite.  Queries then are f16, scaled by a
// power of two of each head's own so that its largest element is just in range.
// The keys' rows come through LDS: every window of kWindow keys is looked up in
// the page table once (any page size), as 32-bit offsets of 16 bytes.
// Bound by memory: two histories of 65,537 f16 keys (268 MB) 51 us, 5.3 TB/s; 48
// ragged ones of up to 4,096 bf16 keys (201 MB) 41, and 52 where the scores are
// kept.  Q8_0 by the codes' conversions, some 500 vector operations a step: 96
// ragged histories (217 MB) 67 us.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

template <int N> struct Words { typedef uint32_t type __attribute__((ext_vector_type(N))); };
template <int N> using words = typename Words<N>::type;
// A load of what no other workgroup reads (3 us of 61 less for 268 MB of rows).
template <typename T> __device__ __forceinline__ T once(const uint8_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_nontemporal_load((gptr<T>)p);
#else
    return *reinterpret_cast<const T*>(p);  // host pass: never executed
#endif
}

constexpr uint32_t kWindow = 512;

template <uint32_t C> __device__ __forceinline__ f4 mfma32(u4 a, u4 b, f4 c) {
    if constexpr (C == BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
// (lo, hi) 16-bit values of the product's type, to the nearest.
template <uint32_t C> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (C == BF16) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{(bf16_t)lo, (bf16_t)hi});
    } else {
        return __builtin_bit_cast(uint32_t, h2{(_Float16)lo, (_Float16)hi});
    }
}
template <uint32_t C> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (C == BF16) return {__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)};
    const h2 h = __builtin_bit_cast(h2, w);
    return {(float)h.x, (float)h.y};
}
// Two f16 codes from a word of 0x6400 | code + 128 each.
__device__ __forceinline__ h2 codes2(uint32_t w) {
    return __builtin_bit_cast(h2, w) - h2{(_Float16)1152, (_Float16)1152};
}
// Value i of 16.
__device__ __forceinline__ float scale_of(const u4 (&w)[2], int i) {
    const uint32_t pair = w[i / 8][i % 8 / 2];
    return (float)__builtin_bit_cast(h2, pair)[i % 2];
}
__device__ __forceinline__ uint32_t bits_of(h2 h) { return __builtin_bit_cast(uint32_t, h); }

// Offsets (16 bytes) of keys [t0, t0 + kWindow) into off, keys past k1 as the
// last, by a wave.  True where a page id is out of range.
__device__ __forceinline__ bool window_offsets(const PageAttn& a, uint32_t b, uint32_t t0, uint32_t k1, uint32_t bytes,
                                               uint32_t* off) {
    const uint32_t end = min(kWindow, (k1 - t0 + kStep - 1) / kStep * kStep);
    bool bad = false;
    __syncthreads();  // off is still read (one wave: an order for the compiler)
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < end; i += 64) {
        const uint32_t t = min(t0 + i, k1 - 1), at = t / a.c.page;
        uint32_t page = (uint32_t)gld<int32_t>(a.r.table + b * a.r.stride + at);
        if (page >= a.c.count) {
            bad = true;
            page = 0;
        }
        off[i] = (uint32_t)((page * a.c.ps + (t - at * a.c.page) * a.c.ts) * bytes / 16);
    }
    __syncthreads();
    return __any(bad);
}

template <uint32_t K> struct Four;  // four elements as they lie, and as floats
template <> struct Four<F32> {
    typedef words<4> type;
    static __device__ __forceinline__ f4 widen(type w) { return __builtin_bit_cast(f4, w); }
};
template <> struct Four<F16> {
    typedef words<2> type;
    static __device__ __forceinline__ f4 widen(type w) {
        const float2 a = unpack2<F16>(w.x), b = unpack2<F16>(w.y);
        return f4{a.x, a.y, b.x, b.y};
    }
};
template <> struct Four<BF16> {
    typedef words<2> type;
    static __device__ __forceinline__ f4 widen(type w) {
        const float2 a = unpack2<BF16>(w.x), b = unpack2<BF16>(w.y);
        return f4{a.x, a.y, b.x, b.y};
    }
};
template <> struct Four<Q8_0> {
    typedef uint32_t type;
    static __device__ __forceinline__ f4 widen(type w) {
        return f4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)((int32_t)w >> 24)};
    }
};

// f(integral constant of the kind): the code of one branch.
template <class F> __device__ __forceinline__ void with_kind(uint32_t kind, F f) {
    if (kind == F32) f(std::integral_constant<uint32_t, F32>());
    else if (kind == F16) f(std::integral_constant<uint32_t, F16>());
    else f(std::integral_constant<uint32_t, BF16>());
}
// Whether four elements at a multiple of four are one access.
__device__ __forceinline__ bool fours(const Heads& h) {
    const size_t es = h.kind == F32 ? 4 : 2;
    return (((uintptr_t)h.p | h.row * es | h.head * es) & (4 * es - 1)) == 0;
}
template <uint32_t K> __device__ __forceinline__ f4 load4(const uint8_t* p, size_t i, bool one) {
    if (one) return Four<K>::widen(gld<typename Four<K>::type>(p + i * (K == F32 ? 4 : 2)));
    return f4{elem<K>(p, i), elem<K>(p, i + 1), elem<K>(p, i + 2), elem<K>(p, i + 3)};
}
template <uint32_t K> __device__ __forceinline__ void put4(uint8_t* p, size_t i, f4 x, bool one) {
    if (one) {
        if constexpr (K == F32) *reinterpret_cast<f4*>(p + 4 * i) = x;
        else *reinterpret_cast<words<2>*>(p + 2 * i) = words<2>{pack2<K>(x[0], x[1]), pack2<K>(x[2], x[3])};
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) put<K>(p, i + k, x[k]);
}

// store_part for head n, of which the lane has dims (4 g + r) D / 16 + t.
template <int D>
__device__ __forceinline__ void store_head(const PageAttn& a, const Run& w, uint32_t h, uint32_t n, uint32_t g, float M,
                                           float L, const f4 (&o)[D / 16]) {
    constexpr int NT = D / 16;
    if (!w.whole()) {
        const size_t slot = ((size_t)blockIdx.x * 2 + w.head()) * a.per + n;
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < NT; t += 4)
                *reinterpret_cast<f4*>(a.o + slot * D + (4 * g + r) * NT + t) = f4{o[t][r], o[t + 1][r], o[t + 2][r], o[t + 3][r]};
        if (g == 0) a.ml[slot] = make_float2(M, L);
        return;
    }
    const size_t at = w.b * a.out.row + h * a.out.head + 4 * g * NT;
    const bool one = fours(a.out);
    with_kind(a.out.kind, [&](auto k) {
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int t = 0; t < NT; t += 4) {
                const f4 x = {o[t][r], o[t + 1][r], o[t + 2][r], o[t + 3][r]};
                put4<k>(a.out.p, at + r * NT + t, L == 0.f ? f4{0.f, 0.f, 0.f, 0.f} : x / L, one);
            }
    });
    if (a.sum && g == 0) a.sum[(size_t)w.b * a.heads + h] = make_float2(M, L);
}

template <uint32_t C, int D>
__global__ __launch_bounds__(64, 2) void k_page_attn16(PageAttn a) {
    constexpr int NC = D / 32, NT = D / 16;             // 32-dim steps of S, 16-dim tiles of O
    constexpr uint32_t ES = C == Q8_0 ? 1 : 2;
    constexpr int KW = 2 * ES, VW = D / 64 * ES;         // words of a K load (8 dims) and of a V load (D / 16 dims)
    constexpr float kLo = C == BF16 ? 1.f : 2048.f;      // of a weight's lo part
    constexpr float kRoom = C == BF16 ? 0.f : 15.f;
    __shared__ uint32_t off[kWindow];
    __shared__ __align__(16) uint16_t ksl[kStep][NC], vsl[NC][kStep];  // the step's scales (Q8_0)
    const uint32_t lane = threadIdx.x, g = lane >> 4, n = lane & 15;
    const float part = n < 8 ? 1.f : kLo, rest = n < 8 ? 0.f : -kLo;  // x part + hi rest: x, or its lo part
    const uint32_t G = a.heads / a.c.kvheads;
    Run run;
    if (!run.start(a)) return;
    do {
        const uint32_t kv = run.u / a.groups, in = run.u % a.groups * a.per, h0 = kv * G + in, nh = min(a.per, G - in);
        const uint32_t b = run.b, k0 = run.key(), k1 = run.end();
        if (run.none()) continue;
        // queries: lane (g, n) holds dims 32 c + 8 g .. + 7 of head n % 8
        u4 q[NC];
        float qs = a.scale * kLog2e;
        {
            const uint32_t h = h0 + min(n & 7, nh - 1);
            const bool on = (n & 7) < nh;
            const uint8_t* row = a.q.p + 2 * (b * a.q.row + h * a.q.head + 8 * g);
            const bool whole = (((uintptr_t)a.q.p | 2 * a.q.row | 2 * a.q.head) & 15) == 0;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                u4 w;
                if (whole) {
                    w = gld<u4>(row + 64 * c);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        w[i] = gld<uint16_t>(row + 64 * c + 4 * i) | (uint32_t)gld<uint16_t>(row + 64 * c + 4 * i + 2) << 16;
                }
                q[c] = on ? w : u4{0u, 0u, 0u, 0u};
            }
            if constexpr (C == Q8_0) {
                float x[NC][8], top = 0.f;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 y = a.q.kind == BF16 ? unpack2<BF16>(q[c][i]) : unpack2<F16>(q[c][i]);
                        x[c][2 * i] = y.x;
                        x[c][2 * i + 1] = y.y;
                        top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));
                    }
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                // The largest goes to [2^14, 2^15), and the power's inverse to the scores: f16
                // queries keep all their bits, bf16 ones down to 2^-31 of the largest, and what
                // is smaller is off by 2^-39 of it at most
                const uint32_t f23 = min(268 - (__float_as_uint(top) >> 23), 253u);
                const float f = __uint_as_float(f23 << 23);
                qs *= __uint_as_float((254 - f23) << 23);
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int i = 0; i < 4; i++) q[c][i] = pack2<F16>(x[c][2 * i] * f, x[c][2 * i + 1] * f);
            }
        }
        f4 o[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) o[t] = f4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        bool bad = run.len < 0;
        const uint8_t* kb = a.c.k + kv * a.c.hs * ES + 8 * ES * g;
        const uint8_t* vb = a.c.v + kv * a.c.hs * ES + (D / 16) * ES * n;
        // lane l fetches scales l % 2 * NC / 2 .. of key l / 2
        const uint8_t* ksb = reinterpret_cast<const uint8_t*>(a.c.ks) + kv * a.c.hs / 16 + (lane & 1) * NC;
        const uint8_t* vsb = reinterpret_cast<const uint8_t*>(a.c.vs) + kv * a.c.hs / 16 + (lane & 1) * NC;
        for (uint32_t w0 = k0; w0 < k1; w0 += kWindow) {
            if (window_offsets(a, b, w0, k1, ES, off)) {
                bad = true;
                break;
            }
            const uint32_t end = min(k1, w0 + kWindow);
            words<KW> kr[2][NC];
            words<VW> vr[8];
            typename std::conditional<NC == 4, uint32_t, uint16_t>::type ksr, vsr;  // half a key's scales
            auto load_k = [&](uint32_t t0) {
                const uint32_t* of = off + (t0 - w0);
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    const uint8_t* row = kb + (size_t)of[16 * kt + n] * 16;
#pragma unroll
                    for (int c = 0; c < NC; c++) kr[kt][c] = once<words<KW>>(row + 16 * KW * c);
                }
                if constexpr (C == Q8_0) ksr = gld<decltype(ksr)>(ksb + of[lane / 2]);
            };
            auto load_v = [&](uint32_t t0) {
                const uint32_t* of = off + (t0 - w0);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    vr[j] = once<words<VW>>(vb + (size_t)of[(j & 4) * 4 + 4 * g + (j & 3)] * 16);
                }
                if constexpr (C == Q8_0) vsr = gld<decltype(vsr)>(vsb + of[lane / 2]);
            };
            f4 s[2];
            auto scores = [&](uint32_t t0) {
                u4 kq[2][2];  // scales of keys 16 kt + 4 g .. + 3
                if constexpr (C == Q8_0) {
                    __syncthreads();  // those of the step before are still read
                    __builtin_memcpy(&ksl[lane / 2][(lane & 1) * NC / 2], &ksr, NC);
                    __syncthreads();
#pragma unroll
                    for (int kt = 0; kt < 2; kt++)
                        __builtin_memcpy(&kq[kt], __builtin_assume_aligned(&ksl[16 * kt + 4 * g][0], 16), 8 * NC);
                }
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    s[kt] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < NC; c++) {
                        if constexpr (C == Q8_0) {
                            u4 k16;
#pragma unroll
                            for (int i = 0; i < 2; i++) {
                                const uint32_t x = kr[kt][c][i] ^ 0x80808080u;
                                k16[2 * i] = bits_of(codes2(__builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)));
                                k16[2 * i + 1] = bits_of(codes2(__builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)));
                            }
                            const f4 acc = mfma32<F16>(k16, q[c], f4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                            for (int r = 0; r < 4; r++)
                                s[kt][r] = fmaf(acc[r], scale_of(kq[kt], r * NC + c), s[kt][r]);
                        } else {
                            s[kt] = mfma32<C>(kr[kt][c], q[c], s[kt]);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; r++) s[kt][r] *= qs;
                }
            };
            auto sums = [&](uint32_t t0, auto last) {
                if constexpr (last) {  // no weight, and no value, past the end
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const bool past = t0 + (j & 4) * 4 + 4 * g + (j & 3) >= k1;
                        if (past) s[j / 4][j % 4] = -INFINITY;
#pragma unroll
                        for (int i = 0; i < VW; i++) vr[j][i] = past ? 0u : vr[j][i];
                    }
                    if constexpr (C == Q8_0) vsr = t0 + lane / 2 >= k1 ? 0 : vsr;
                }
                float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                                  fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
                if (__any(top > m + kRoom)) {
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float M = fmaxf(m, top + (8.f - kRoom)), alpha = M == -INFINITY ? 1.f : exp2_of(m - M);
                    m = M;
                    l *= alpha;
#pragma unroll
                    for (int t = 0; t < NT; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) o[t][r] *= alpha;
                }
                const float mf = m == -INFINITY ? 0.f : m;
                u4 p;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = exp2_of(s[i / 2][2 * (i % 2)] - mf), y = exp2_of(s[i / 2][2 * (i % 2) + 1] - mf);
                    l += x + y;
                    const float2 hi = unpack2<C>(pack2<C>(x, y));
                    p[i] = pack2<C>(fmaf(hi.x, rest, x * part), fmaf(hi.y, rest, y * part));
                }
                if constexpr (C == Q8_0) {
                    // scales of the lane's block and keys, in pairs
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < NC / 2; i++)
                        vsl[(lane & 1) * NC / 2 + i][lane / 2] = (uint16_t)((uint32_t)vsr >> (16 * i));
                    __syncthreads();
                    const uint16_t* vl = vsl[D / 16 * n / 32];
                    h2 d[4];
                    __builtin_memcpy(d, __builtin_assume_aligned(vl + 4 * g, 8), 8);
                    __builtin_memcpy(d + 2, __builtin_assume_aligned(vl + 16 + 4 * g, 8), 8);
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        u4 hi, lo;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t sel = 0x0c000c00u | (uint32_t)(t % 4) | (uint32_t)(4 + t % 4) << 16;
                            const h2 c = codes2(__builtin_amdgcn_perm(vr[2 * i + 1][t / 4], vr[2 * i][t / 4], sel) ^ 0x64806480u);
                            const h2 v = c * d[i];
                            hi[i] = bits_of(v);
                            lo[i] = bits_of(__builtin_elementwise_fma(c, d[i], -v));
                        }
                        o[t] = mfma32<F16>(hi, p, o[t]);
                        o[t] = mfma32<F16>(lo, p, o[t]);
                    }
                } else {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        u4 v;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            v[i] = __builtin_amdgcn_perm(vr[2 * i + 1][t / 2], vr[2 * i][t / 2], t & 1 ? 0x07060302u : 0x05040100u);
                        o[t] = mfma32<C>(v, p, o[t]);
                    }
                }
            };
            auto step = [&](uint32_t t0, auto last) {
                load_k(t0);
                load_v(t0);
                __builtin_amdgcn_sched_barrier(0);  // V is requested before K is waited for
                scores(t0);
                sums(t0, last);
                if (a.score && n < nh) {  // behind the products: a store waits for the loads of other waves
#pragma unroll
                    for (int kt = 0; kt < 2; kt++)  // the row holds whole steps
                        *reinterpret_cast<f4*>(a.score + ((size_t)b * a.heads + h0 + n) * a.score_row + t0 + 16 * kt + 4 * g) = s[kt];
                }
            };
            uint32_t t0 = w0;
            for (; t0 + kStep <= end; t0 += kStep) step(t0, std::false_type());
            if (t0 < end) step(t0, std::true_type());
        }
        if (bad) l = __builtin_nanf("");
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) {  // the lo parts' sums, from column n + 8
                const float lo = __shfl_xor(o[t][r], 8, 64);
                if (finite_f(o[t][r])) o[t][r] = fmaf(lo, 1.f / kLo, o[t][r]);
            }
        if (n < nh) store_head<D>(a, run, h0 + n, n, g, m, l, o);
    } while (run.next(a));
}

// The same for 32-bit queries or outputs, or queries and caches of different types: every
// product in 32 bits on v_mfma_f32_16x16x4_f32, K and V widened as they arrive.
// Sixteen keys a round; k slot g of step (c, i) of the first product is dim 16 c
// + 4 g + i, of step r of the second key 4 g + r, so that the scores again are
// the weights' operand as they come.  An eighth of the 16-bit products' rate, and
// half of each instruction idle with eight heads or fewer: still under the time
// that memory takes for the rows (2,048 matrix-core cycles for 16 KB of f32 rows,
// which take a compute unit's share of the bandwidth about 8,000).  One history of
// 517 f32 keys takes 10 us, the latency of its look-ups and rows; 48 ragged ones of
// up to 4,096 keys 72 us (403 MB, 5.6 TB/s), f32 queries over f16 or bf16 65, over
// Q8_0 67.  16-bit queries with a 32-bit output 70 us where k_page_attn16 takes 46, 75
// over Q8_0 against 48 (whole calls).  Heads of 256 take one wave a SIMD for their
// registers: the same 48 histories 155 us in f32 (805 MB), 138 in bf16, where the
// products bound it (nine times that on k_page_attn_any).
template <uint32_t K, int D>
__global__ __launch_bounds__(64, D == 256 ? 1 : 2) void k_page_attn32(PageAttn a) {
    constexpr int NC = D / 16, NV = D / 64;  // 16-dim loads of a key, 64-dim loads of a value
    constexpr uint32_t ES = K == F32 ? 4 : K == Q8_0 ? 1 : 2;
    typedef typename Four<K>::type four;
    __shared__ uint32_t off[kWindow];
    const uint32_t lane = threadIdx.x, g = lane >> 4, n = lane & 15;
    const uint32_t G = a.heads / a.c.kvheads;
    Run run;
    if (!run.start(a)) return;
    do {
        const uint32_t kv = run.u / a.groups, in = run.u % a.groups * a.per, h0 = kv * G + in, nh = min(a.per, G - in);
        const uint32_t b = run.b, k0 = run.key(), k1 = run.end();
        if (run.none()) continue;
        f4 q[NC];  // dims 16 c + 4 g .. + 3 of head n
        {
            const size_t row = b * a.q.row + (h0 + min(n, nh - 1)) * a.q.head + 4 * g;
            const float scale = a.scale * kLog2e;
            const bool one = fours(a.q);
            with_kind(a.q.kind, [&](auto k) {
#pragma unroll
                for (int c = 0; c < NC; c++) q[c] = load4<k>(a.q.p, row + 16 * c, one);
            });
#pragma unroll
            for (int c = 0; c < NC; c++) q[c] = n < nh ? q[c] * scale : f4{0.f, 0.f, 0.f, 0.f};
        }
        f4 o[4 * NV];  // tile 4 c + i: dims 64 c + 4 (4 g + r) + i
#pragma unroll
        for (int t = 0; t < 4 * NV; t++) o[t] = f4{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, l = 0.f;
        bool bad = run.len < 0;
        const uint8_t* kb = a.c.k + kv * a.c.hs * ES + 4 * ES * g;
        const uint8_t* vb = a.c.v + kv * a.c.hs * ES + 4 * ES * n;
        const uint8_t* ksb = reinterpret_cast<const uint8_t*>(a.c.ks) + kv * a.c.hs / 16;
        const uint8_t* vsb = reinterpret_cast<const uint8_t*>(a.c.vs) + kv * a.c.hs / 16 + n / 8 * 2;
        for (uint32_t w0 = k0; w0 < k1; w0 += kWindow) {
            if (window_offsets(a, b, w0, k1, ES, off)) {
                bad = true;
                break;
            }
            const uint32_t end = min(k1, w0 + kWindow);
            auto round = [&](uint32_t t0, auto last) {
                const uint32_t* of = off + (t0 - w0);
                four kr[NC], vr[4][NV];
                _Float16 ks[NC / 2], vs[4][NV];
                const uint32_t ok = of[n];
#pragma unroll
                for (int c = 0; c < NC; c++) kr[c] = once<four>(kb + (size_t)ok * 16 + 16 * ES * c);
                if constexpr (K == Q8_0) {
#pragma unroll
                    for (int c = 0; c < NC / 2; c++) ks[c] = gld<_Float16>(ksb + ok + 2 * c);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t ov = of[4 * g + r];
#pragma unroll
                    for (int c = 0; c < NV; c++) {
                        vr[r][c] = once<four>(vb + (size_t)ov * 16 + 64 * ES * c);
                        if constexpr (K == Q8_0) vs[r][c] = gld<_Float16>(vsb + ov + 4 * c);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);  // V is requested before K is waited for
                f4 s2[2] = {f4{0.f, 0.f, 0.f, 0.f}, f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    f4 k = Four<K>::widen(kr[c]);
                    if constexpr (K == Q8_0) k *= (float)ks[c / 2];
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s2[i & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i], q[c][i], s2[i & 1], 0, 0, 0);
                }
                f4 s = s2[0] + s2[1];
                const f4 all = s;
                if constexpr (last) {  // no weight past the end
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (t0 + 4 * g + r >= k1) s[r] = -INFINITY;
                }
                float top = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
                if (__any(top > m)) {  // no weight above 1, as in bf16 above
                    top = fmaxf(top, __shfl_xor(top, 16, 64));
                    top = fmaxf(top, __shfl_xor(top, 32, 64));
                    const float M = fmaxf(m, top + 8.f), alpha = M == -INFINITY ? 1.f : exp2_of(m - M);
                    m = M;
                    l *= alpha;
#pragma unroll
                    for (int t = 0; t < 4 * NV; t++) o[t] *= alpha;
                }
                const float mf = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float p = exp2_of(s[r] - mf);
                    l += p;
#pragma unroll
                    for (int c = 0; c < NV; c++) {
                        f4 v = Four<K>::widen(vr[r][c]);
                        if constexpr (K == Q8_0) v *= (float)vs[r][c];
                        if constexpr (last) {  // and no value
                            if (t0 + 4 * g + r >= k1) v = f4{0.f, 0.f, 0.f, 0.f};
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            o[4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i], p, o[4 * c + i], 0, 0, 0);
                    }
                }
                if (a.score && n < nh)  // the row holds whole steps
                    *reinterpret_cast<f4*>(a.score + ((size_t)b * a.heads + h0 + n) * a.score_row + t0 + 4 * g) = all;
            };
            uint32_t t0 = w0;
            for (; t0 + 16 <= end; t0 += 16) round(t0, std::false_type());
            if (t0 < end) round(t0, std::true_type());
        }
        if (bad) l = __builtin_nanf("");
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (n >= nh) continue;
        const bool whole = run.whole(), one = fours(a.out);
        const size_t slot = ((size_t)blockIdx.x * 2 + run.head()) * a.per + n;
        auto each = [&](auto f) {  // f(dim, its four values)
#pragma unroll
            for (int c = 0; c < NV; c++)
#pragma unroll
                for (int r = 0; r < 4; r++)
                    f(64 * c + 16 * g + 4 * r, f4{o[4 * c][r], o[4 * c + 1][r], o[4 * c + 2][r], o[4 * c + 3][r]});
        };
        if (!whole) {
            each([&](uint32_t j, f4 x) { *reinterpret_cast<f4*>(a.o + slot * D + j) = x; });
        } else {
            const size_t at = b * a.out.row + (h0 + n) * a.out.head;
            with_kind(a.out.kind, [&](auto k) {
                each([&](uint32_t j, f4 x) { put4<k>(a.out.p, at + j, l == 0.f ? f4{0.f, 0.f, 0.f, 0.f} : x / l, one); });
            });
        }
        if (g == 0) {
            if (!whole) a.ml[slot] = make_float2(m, l);
            else if (a.sum) a.sum[(size_t)b * a.heads + h0 + n] = make_float2(m, l);
        }
    } while (run.next(a));
}

// out of the units that several workgroups hold parts of: a workgroup per `heads`
// heads of a unit, with V dims of a head (4, or 1 where a head's width is no multiple of 4) a
// thread and its parts dealt to `groups` threads.  The parts of a unit: the
// second slot of the workgroup whose run it begins in, and the first slot of
// those behind.  Bound by latency: 5 us for one unit's parts, 6 to 7 for hundreds.
constexpr uint32_t kJoinMost = 1024, kJoinAhead = 8;  // threads; parts in flight
static_assert(kPerMost * kPageMaxDim / 4 <= kJoinMost / 2 && kPageMaxDim <= kJoinMost / 2, "a thread each, whatever V");
template <int V>
__global__ __launch_bounds__(kJoinMost) void k_page_join(PageAttn a, uint32_t heads, uint32_t wide) {
    __shared__ float red[kJoinMost][V + 2];
    const uint32_t u = blockIdx.x, b = blockIdx.y, d = a.c.dim, tid = threadIdx.x, groups = blockDim.x / wide;
    const uint32_t G = a.heads / a.c.kvheads, in = u % a.groups * a.per, nh = min(a.per, G - in), z = blockIdx.z * heads;
    if (z >= nh) return;
    const uint32_t items = min(heads, nh - z) * d / V;
    const uint64_t total = gld<uint64_t>(a.begin + a.r.batch);
    const Parts held = parts_of(total, a.runs, gld<uint64_t>(a.begin + b), gld<uint64_t>(a.begin + b + 1), a.units, u);
    const uint64_t first = held.first;
    const uint32_t parts = held.count;
    if (parts <= 1) return;  // whole in its workgroup
    const uint32_t item = min(tid % wide, items - 1), n = z + item * V / d, j = item * V % d;
    float M = -INFINITY, L = 0.f, O[V];
#pragma unroll
    for (int k = 0; k < V; k++) O[k] = 0.f;
    for (uint32_t i0 = tid / wide; i0 < parts; i0 += kJoinAhead * groups) {
        float2 ml[kJoinAhead];
        float o[kJoinAhead][V];
#pragma unroll
        for (uint32_t k = 0; k < kJoinAhead; k++) {
            const uint32_t i = min(i0 + k * groups, parts - 1);
            const size_t slot = ((first + i) * 2 + (i == 0)) * a.per + n;
            ml[k] = gld<float2>(a.ml + slot);
            if constexpr (V == 4) {
                const float4 t = gld<float4>(a.o + slot * d + j);
                o[k][0] = t.x, o[k][1] = t.y, o[k][2] = t.z, o[k][3] = t.w;
            } else {
                o[k][0] = gld<float>(a.o + slot * d + j);
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < kJoinAhead; k++) {
            if (i0 + k * groups >= parts) break;
            const float Mn = fmaxf(M, ml[k].x), Mf = Mn == -INFINITY ? 0.f : Mn;
            const float f = exp2_of(M - Mf), e = exp2_of(ml[k].x - Mf);
            M = Mn;
            L = fmaf(ml[k].y, e, L * f);
#pragma unroll
            for (int c = 0; c < V; c++) O[c] = fmaf(o[k][c], e, O[c] * f);
        }
    }
    red[tid][V] = M;
    red[tid][V + 1] = L;
#pragma unroll
    for (int c = 0; c < V; c++) red[tid][c] = O[c];
    __syncthreads();
    if (tid >= wide || tid >= items) return;
    float Ma = M;
    for (uint32_t i = 1; i < groups; i++) Ma = fmaxf(Ma, red[i * wide + tid][V]);
    const float Mf = Ma == -INFINITY ? 0.f : Ma, f0 = exp2_of(M - Mf);
    L *= f0;
#pragma unroll
    for (int c = 0; c < V; c++) O[c] *= f0;
    for (uint32_t i = 1; i < groups; i++) {
        const float* t = red[i * wide + tid];
        const float f = exp2_of(t[V] - Mf);
        L = fmaf(t[V + 1], f, L);
#pragma unroll
        for (int c = 0; c < V; c++) O[c] = fmaf(t[c], f, O[c]);
    }
    const uint32_t h = u / a.groups * G + in + n;
#pragma unroll
    for (int c = 0; c < V; c++)
        put_kind(a.out.kind, a.out.p, b * a.out.row + h * a.out.head + j + c, L == 0.f ? 0.f : O[c] / L);
    if (a.sum && j == 0) a.sum[(size_t)b * a.heads + h] = make_float2(Ma, L);
}

// wout[b][g][t] = win[b][g][t] + sum over g's query heads of 2^(s - m) / l: four
// keys a thread.  In the heads' order, so the same bits on every call.  5.6 us for
// 48 histories of up to 4,096 keys (13 MB of scores).
__global__ __launch_bounds__(kBlock) void k_page_weights(PageAttn a) {
    const uint32_t g = blockIdx.y, b = blockIdx.z, G = a.heads / a.c.kvheads, t = (blockIdx.x * kBlock + threadIdx.x) * 4;
    const int32_t len = length_of(a.r, b);
    if ((int64_t)t >= len) return;
    float w[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t i = 0; i < G; i++) {
        const size_t h = (size_t)b * a.heads + g * G + i;
        const float2 ml = gld<float2>(a.sum + h);
        const float4 s = gld<float4>(a.score + h * a.score_row + t);
        const float Mf = ml.x == -INFINITY ? 0.f : ml.x, inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
        w[0] = fmaf(exp2_of(s.x - Mf), inv, w[0]);
        w[1] = fmaf(exp2_of(s.y - Mf), inv, w[1]);
        w[2] = fmaf(exp2_of(s.z - Mf), inv, w[2]);
        w[3] = fmaf(exp2_of(s.w - Mf), inv, w[3]);
    }
    const float* in = a.win ? a.win + b * a.win_row + g * a.win_head + t : nullptr;
    float* out = a.wout + b * a.wout_row + g * a.wout_head + t;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++)
        if ((int64_t)t + i < len) out[i] = in ? w[i] + gld<float>(in + i) : w[i];
}

// The kernel of a call.  The matrix-core kernels want rows aligned to 16 bytes
// within 64 GiB; k_page_attn16 takes heads of 64 or 128, 16-bit queries of the
// cache's type (or over Q8_0) and a 16-bit output, whose rounding hides that of the
// weights; k_page_attn32 those heads with other types and heads of 256.
uint32_t page_attn_kernel(const PageAttn& a) {
    const bool q8 = a.c.kind == Q8_0;
    if (a.c.dim != 64 && a.c.dim != 128 && a.c.dim != 256) return 0;
    const uint64_t es = q8 ? 1 : a.c.kind == F32 ? 4 : 2, all = a.c.ps | a.c.ts | a.c.hs;
    if (((uintptr_t)a.c.k | (uintptr_t)a.c.v | all * es) % 16) return 0;
    // a key's scales lie together
    if (q8 && (all % a.c.dim || ((uintptr_t)a.c.ks | (uintptr_t)a.c.vs) % (a.c.dim / 16))) return 0;
    if (((a.c.count - 1) * a.c.ps + (a.c.page - 1) * a.c.ts) * es >= (uint64_t)1 << 36) return 0;
    return a.c.dim != 256 && a.q.kind != F32 && a.out.kind != F32 && (q8 || a.c.kind == a.q.kind) ? 16 : 32;
}

// At most kPageMaxRuns workgroups, and no more than there may be runs of work.
void page_attn_plan(PageAttn& a, uint32_t kernel, uint32_t cus) {
    const uint32_t G = a.heads / a.c.kvheads;
    a.kernel = kernel;
    a.groups = kernel ? (G + kPerMost - 1) / kPerMost : G;
    a.per = (G + a.groups - 1) / a.groups;
    a.units = a.c.kvheads * a.groups;
    const uint64_t steps = std::max<uint64_t>(1, ((uint64_t)a.r.most + kStep - 1) / kStep) + kUnitCost;
    // k_page_attn16 over 48 ragged histories of bf16 keys: 1,024 waves 52.5 us, 1,536 and
    // 2,048 53.5 and 54.4, and the join 2 more.  Over 96 of Q8_0 keys whole calls of 1,024
    // and 2,048 waves: 128 wide 74 and 76, 64 wide 52.5 and 50, f32 queries 143 and 128
    const uint64_t fill = std::min<uint64_t>((uint64_t)cus * (kernel && a.c.kind == Q8_0 ? 8 : 4), kPageMaxRuns);
    a.runs = (uint32_t)std::min<uint64_t>(fill, (a.units * steps * a.r.batch + kRunMin - 1) / kRunMin);
    a.score_row = ((uint64_t)a.r.most + 63) / 64 * 64;
}

// The slots, and with weights every score and every head's (m, l).
static size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }
size_t page_attn_bytes(const PageAttn& a, bool weights) {
    const size_t slots = (size_t)a.runs * 2 * a.per, heads = (size_t)a.r.batch * a.heads;
    return round16(slots * a.c.dim * 4) + round16(slots * 8) + round16((a.r.batch + 1) * 8) + (weights ? heads * a.score_row * 4 + heads * 8 : 0);
}
void page_attn_place(PageAttn& a, void* work, bool weights) {
    const size_t slots = (size_t)a.runs * 2 * a.per, heads = (size_t)a.r.batch * a.heads;
    uint8_t* p = static_cast<uint8_t*>(work);
    a.o = reinterpret_cast<float*>(p);
    p += round16(slots * a.c.dim * 4);
    a.ml = reinterpret_cast<float2*>(p);
    p += round16(slots * 8);
    a.begin = reinterpret_cast<uint64_t*>(p);
    p += round16((a.r.batch + 1) * 8);
    a.score = weights ? reinterpret_cast<float*>(p) : nullptr;
    a.sum = weights ? reinterpret_cast<float2*>(p + heads * a.score_row * 4) : nullptr;
}

template <uint32_t K> static void launch_any(const PageAttn& a, hipStream_t s) {
    const dim3 grid(a.runs), block(kBlock);
    if (a.c.dim <= 64) hipLaunchKernelGGL((k_page_attn_any<K, 8>), grid, block, 0, s, a);
    else if (a.c.dim <= 128) hipLaunchKernelGGL((k_page_attn_any<K, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_page_attn_any<K, 32>), grid, block, 0, s, a);
}
template <uint32_t C> static void launch_matrix(const PageAttn& a, hipStream_t s) {
    if constexpr (C != F32) {
        if (a.kernel == 16 && a.c.dim == 64) hipLaunchKernelGGL((k_page_attn16<C, 64>), dim3(a.runs), dim3(64), 0, s, a);
        else if (a.kernel == 16) hipLaunchKernelGGL((k_page_attn16<C, 128>), dim3(a.runs), dim3(64), 0, s, a);
        if (a.kernel == 16) return;
    }
    if (a.c.dim == 256) hipLaunchKernelGGL((k_page_attn32<C, 256>), dim3(a.runs), dim3(64), 0, s, a);
    else if (a.c.dim == 64) hipLaunchKernelGGL((k_page_attn32<C, 64>), dim3(a.runs), dim3(64), 0, s, a);
    else hipLaunchKernelGGL((k_page_attn32<C, 128>), dim3(a.runs), dim3(64), 0, s, a);
}
template <uint32_t C> static void launch_attn(const PageAttn& a, hipStream_t s) {
    if (a.kernel) launch_matrix<C>(a, s);
    else launch_any<C>(a, s);
}

void launch_page_attn(const PageAttn& a, hipStream_t s) {
    if (a.c.kind == F32) launch_attn<F32>(a, s);
    else if (a.c.kind == F16) launch_attn<F16>(a, s);
    else if (a.c.kind == BF16) launch_attn<BF16>(a, s);
    else launch_attn<Q8_0>(a, s);
    if (a.runs > 1) {
        const uint32_t v = a.c.dim % 4 ? 1 : 4;
        // few units hold many parts each (65,537 keys: 64), and a workgroup of
        // 1,024 threads takes one of their heads, else 512 threads a unit's
        const bool few = (uint64_t)a.units * a.r.batch < 128;
        const uint32_t heads = few ? 1 : a.per;
        uint32_t wide = 16;
        while (wide < heads * a.c.dim / v) wide *= 2;  // at most 512: eight heads of 256, or one in single dims
        const dim3 grid(a.units, a.r.batch, few ? a.per : 1), block(few ? kJoinMost : kJoinMost / 2);
        if (v == 4) hipLaunchKernelGGL(k_page_join<4>, grid, block, 0, s, a, heads, wide);
        else hipLaunchKernelGGL(k_page_join<1>, grid, block, 0, s, a, heads, wide);
    }
    if (a.score && a.r.most)
        hipLaunchKernelGGL(k_page_weights, dim3((a.r.most + 4 * kBlock - 1) / (4 * kBlock), a.c.kvheads, a.r.batch),
                           dim3(kBlock), 0, s, a);
}

}  // namespace qh
