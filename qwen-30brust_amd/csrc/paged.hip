// The key-value cache in pages: appending tokens (per-head RMSNorm and NeoX
// RoPE of q and k on the way) and the attention of one new token per sequence.
//
// A key t of sequence b lies in slot t % page of page table[b][t / page].
// Page ids come from the caller's device memory: every one is compared with the
// pool's size before it is used.  A sequence whose length or page ids are out
// of range gets NaN from the attention, and an append to such a page is left
// out.
#include <algorithm>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

// ------------------------------------------------------------------ append --
// A wave per token and head (q's heads, then k's, then v's):
//   y = x / sqrt(sum x^2 / dim + eps) * w              (q and k, with weights)
//   (y_i, y_j) = (y_i cos - y_j sin, y_j cos + y_i sin), j = i + dim / 2
// in 32 bits, rounded once to the type it is stored in.  Q8_0: per 32 values
// d = f16(max |y| / 127) and codes round(y / d), as GGML lays them out, but
// codes and scales each in an array of their own.
// A token outside the table of angles becomes NaN.
__global__ __launch_bounds__(kBlock) void k_page_append(PageAppend a) {
    constexpr uint32_t E = kPageMaxDim / 64;
    __shared__ float turn[kWaves][kPageMaxDim];
    const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6, d = a.c.dim;
    const uint32_t slots = a.heads + 2 * a.c.kvheads;
    const uint64_t unit = (uint64_t)blockIdx.x * kWaves + wv;
    const uint32_t i = (uint32_t)min(unit / slots, (uint64_t)a.n - 1);
    const uint32_t h = (uint32_t)(unit % slots);
    // the token's sequence: the last whose first token is not behind it
    uint32_t b = i;
    int32_t at = 0, count = 1;  // the token's number in its sequence, and of how many
    bool live = unit / slots < a.n;
    if (a.first) {
        uint32_t before = 0;
        for (uint32_t j = 0; j <= a.r.batch; j += 64) {
            const bool le = j + lane <= a.r.batch && gld<int32_t>(a.first + min(j + lane, a.r.batch)) <= (int32_t)i;
            before += __popcll(__ballot(le));
        }
        live = live && before > 0 && before <= a.r.batch;
        b = live ? before - 1 : 0;
        const int32_t f = gld<int32_t>(a.first + b);
        at = (int32_t)i - f;
        count = gld<int32_t>(a.first + b + 1) - f;
    }
    const int32_t len = live ? length_of(a.r, b) : -1;
    const int32_t t = len - count + at;
    live = live && t >= 0 && t < len;
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
        const int32_t p = live ? (a.pos ? gld<int32_t>(a.pos + i) : t) : 0;
        const bool in = p >= 0 && (uint32_t)p < a.rope_rows;
        const float2* row = a.rope + (size_t)(in ? p : 0) * (d / 2);
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
    const int32_t page = gld<int32_t>(a.r.table + b * a.r.stride + (uint32_t)t / a.c.page);
    if (page < 0 || (uint32_t)page >= a.c.count) return;
    const size_t o = (size_t)page * a.c.ps + (size_t)((uint32_t)t % a.c.page) * a.c.ts + g * a.c.hs;
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
        const float f = (float)dq;
        const float code = fine && f > 0.f ? fminf(fmaxf(rintf(x[j] / f), -127.f), 127.f) : 0.f;
        reinterpret_cast<int8_t*>(to)[o + e] = (int8_t)code;
        if (lane % 32 == 0) scale[(o + e) / 32] = dq;
    }
}

void launch_page_append(const PageAppend& a, hipStream_t s) {
    const uint64_t units = (uint64_t)a.n * (a.heads + 2 * a.c.kvheads);
    hipLaunchKernelGGL(k_page_append, dim3((uint32_t)((units + kWaves - 1) / kWaves)), dim3(kBlock), 0, s, a);
}

// --------------------------------------------------------------- attention --
//   s_t = scale * log2(e) * q . k_t,  m = max s_t,  l = sum 2^(s_t - m),
//   o = sum 2^(s_t - m) v_t / l
// over the keys of one sequence, in parts of `span` keys whose (m, l, o) are
// folded by k_page_join; everything in 32 bits.  A row with no keys, or whose
// scores are all -inf, is zeros.
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32

// One head and part per workgroup, any head width up to 8 E: eight lanes share
// a key, with E elements of its row each, and keep the (m, l, o) of their own
// keys, so there is no barrier before the merge at the end.
template <uint32_t K, int E>
__global__ __launch_bounds__(kBlock) void k_page_attn_any(PageAttn a) {
    __shared__ float red[kWaves][8 * E], rm[kWaves], rl[kWaves];
    const uint32_t h = blockIdx.x, part = blockIdx.y, b = blockIdx.z, d = a.c.dim;
    const uint32_t g = h / (a.heads / a.c.kvheads);
    const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6, kl = lane >> 3, p = lane & 7;
    const int32_t len = length_of(a.r, b);
    const uint32_t n = len < 0 ? 0u : (uint32_t)len, k0 = part * a.span;
    if (part && k0 >= n) return;  // k_page_join does not read it
    const uint32_t k1 = min(n, k0 + a.span);
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < E; i++) {
        const uint32_t e = p + 8 * i;
        q[i] = e < d ? elem_kind(a.q.kind, a.q.p, b * a.q.row + h * a.q.head + e) : 0.f;
        o[i] = 0.f;
    }
    bool bad = len < 0;
    for (uint32_t t = k0 + 8 * wv + kl; t - kl < k1; t += 8 * kWaves) {  // wave-uniform
        const uint32_t tt = min(t, k1 - 1);
        int32_t page = gld<int32_t>(a.r.table + b * a.r.stride + tt / a.c.page);
        if (page < 0 || (uint32_t)page >= a.c.count) {
            bad = true;
            page = 0;
        }
        const size_t at = (size_t)page * a.c.ps + (size_t)(tt % a.c.page) * a.c.ts + g * a.c.hs;
        float kr[E], vr[E];
#pragma unroll
        for (int i = 0; i < E; i++) {
            const uint32_t e = p + 8 * i;
            kr[i] = vr[i] = 0.f;
            if (e < d) {
                kr[i] = elem<K>(a.c.k, at + e);
                vr[i] = elem<K>(a.c.v, at + e);
                if constexpr (K == Q8_0) {
                    kr[i] *= (float)gld<_Float16>(a.c.ks + (at + e) / 32);
                    vr[i] *= (float)gld<_Float16>(a.c.vs + (at + e) / 32);
                }
            }
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; i++) s = fmaf(q[i], kr[i], s);
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
        for (int i = 0; i < E; i++) o[i] = fmaf(e, vr[i], o[i] * alpha);
    }
    if (bad) l = __builtin_nanf("");
    // the wave's eight lane groups, then the waves
    float M = m;
#pragma unroll
    for (int x = 8; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
    const float e = exp2_of(m - (M == -INFINITY ? 0.f : M));
    l *= e;
#pragma unroll
    for (int i = 0; i < E; i++) o[i] *= e;
#pragma unroll
    for (int x = 8; x < 64; x <<= 1) {
        l += __shfl_xor(l, x, 64);
#pragma unroll
        for (int i = 0; i < E; i++) o[i] += __shfl_xor(o[i], x, 64);
    }
    if (kl == 0) {
#pragma unroll
        for (int i = 0; i < E; i++) red[wv][p + 8 * i] = o[i];
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
    const size_t slot = ((size_t)b * a.heads + h) * a.splits + part;
    for (uint32_t j = threadIdx.x; j < d; j += kBlock) {
        float O = 0.f;
        for (int x = 0; x < kWaves; x++) O = fmaf(red[x][j], exp2_of(rm[x] - Mf), O);
        if (a.ml) a.o[slot * d + j] = O;
        else put_kind(a.out.kind, a.out.p, b * a.out.row + h * a.out.head + j, L == 0.f ? 0.f : O / L);
    }
    if (a.ml && threadIdx.x == 0) {
        a.ml[2 * slot] = Ma;
        a.ml[2 * slot + 1] = L;
    }
}

// The waves' parts of heads h0 .. h0 + nh - 1 folded: to the part's slot, or,
// where it is the only one, to out.  After a barrier.
template <int H, int D>
__device__ __forceinline__ void merge_waves(const PageAttn& a, uint32_t b, uint32_t h0, uint32_t nh, uint32_t part,
                                            const float (*red)[H][D + 4], const float (*rm)[H], const float (*rl)[H]) {
    for (uint32_t i = threadIdx.x; i < nh * D; i += kBlock) {
        const uint32_t n = i / D, j = i % D;
        float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
        for (int x = 0; x < kWaves; x++) M = fmaxf(M, rm[x][n]);
        const float Mf = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int x = 0; x < kWaves; x++) {
            const float f = exp2_of(rm[x][n] - Mf);
            L = fmaf(rl[x][n], f, L);
            O = fmaf(red[x][n][j], f, O);
        }
        if (!a.ml) {
            put_kind(a.out.kind, a.out.p, b * a.out.row + (h0 + n) * a.out.head + j, L == 0.f ? 0.f : O / L);
            continue;
        }
        const size_t slot = ((size_t)b * a.heads + h0 + n) * a.splits + part;
        a.o[slot * D + j] = O;
        if (j == 0) {
            a.ml[2 * slot] = M;
            a.ml[2 * slot + 1] = L;
        }
    }
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
// the hi column alone says so.)  That leaves 2^-18 (bf16) or 2^-23 (f16) of a
// weight's bits off; one part would leave 2^-9.
// The running maximum moves only when a score is 15 above it (2^15 fits f16),
// to 7 below the new one: nearly never, so the sums are rarely rescaled.
// Q8_0: codes are exact in f16 (byte | 0x6400 is 1024 + byte), a block's scale
// multiplies its 32-dim product in 32 bits, and code * scale of V goes in as two
// f16 parts (the product and its rounding error, by a fused multiply-add);
// values past f16's range become infinite.  Queries then are f16, scaled by a
// power of two of their own.
// The keys' rows come through LDS: every window of kWindow keys is looked up in
// the page table once (any page size), as 32-bit offsets of 16 bytes.
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kWindow = 1024;

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
// Two f16 codes from the words whose bytes 0 and 2 are code + 128.
__device__ __forceinline__ h2 codes2(uint32_t w) {
    return __builtin_bit_cast(h2, w) - h2{(_Float16)1152, (_Float16)1152};
}
__device__ __forceinline__ uint32_t bits_of(h2 h) { return __builtin_bit_cast(uint32_t, h); }

// Offsets (16 bytes) of keys [t0, t0 + kWindow) into off, keys past k1 as the
// last; a barrier.  True where a page id is out of range.
__device__ __forceinline__ bool window_offsets(const PageAttn& a, uint32_t b, uint32_t t0, uint32_t k1, uint32_t bytes,
                                               uint32_t* off) {
    int bad = 0;
    for (uint32_t i = threadIdx.x; i < kWindow && t0 + i < (k1 + 31) / 32 * 32; i += kBlock) {
        const uint32_t t = min(t0 + i, k1 - 1), at = t / a.c.page;
        uint32_t page = (uint32_t)gld<int32_t>(a.r.table + b * a.r.stride + at);
        if (page >= a.c.count) {
            bad = 1;
            page = 0;
        }
        off[i] = (uint32_t)((page * a.c.ps + (t - at * a.c.page) * a.c.ts) * bytes / 16);
    }
    return __syncthreads_or(bad);
}

template <uint32_t C, int D>
__global__ __launch_bounds__(kBlock, 2) void k_page_attn16(PageAttn a) {
    constexpr int NC = D / 32, NT = D / 16;             // 32-dim steps of S, 16-dim tiles of O
    constexpr uint32_t ES = C == Q8_0 ? 1 : 2;
    constexpr int KW = 2 * ES, VW = D / 64 * ES;         // words of a K load (8 dims) and of a V load (D / 16 dims)
    __shared__ uint32_t off[kWindow];
    __shared__ float red[kWaves][8][D + 4], rm[kWaves][8], rl[kWaves][8];
    const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6, g = lane >> 4, n = lane & 15;
    const uint32_t kv = blockIdx.x / a.groups, G = a.heads / a.c.kvheads, part = blockIdx.y, b = blockIdx.z;
    const uint32_t in = blockIdx.x % a.groups * a.per, h0 = kv * G + in, nh = min(a.per, G - in);
    const int32_t len = length_of(a.r, b);
    const uint32_t len0 = len < 0 ? 0u : (uint32_t)len, k0 = part * a.span, k1 = min(len0, k0 + a.span);
    if (part && k0 >= len0) return;  // k_page_join does not read it
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
            // 2^-exponent of the largest; its inverse goes to the scores
            const uint32_t e = __float_as_uint(top) >> 23;
            const bool scaled = e > 1 && e < 253;
            const float f = scaled ? __uint_as_float((254 - e) << 23) : 1.f;
            qs *= scaled ? __uint_as_float(e << 23) : 1.f;
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
    bool bad = len < 0;
    const uint8_t* kb = a.c.k + kv * a.c.hs * ES + 8 * ES * g;
    const uint8_t* vb = a.c.v + kv * a.c.hs * ES + (D / 16) * ES * n;
    const uint8_t* ksb = reinterpret_cast<const uint8_t*>(a.c.ks) + kv * a.c.hs / 16;
    const uint8_t* vsb = reinterpret_cast<const uint8_t*>(a.c.vs) + kv * a.c.hs / 16 + (D / 16 * n / 32) * 2;
    for (uint32_t w0 = k0; w0 < k1; w0 += kWindow) {
        if (w0 != k0) __syncthreads();  // off is still read
        if (window_offsets(a, b, w0, k1, ES, off)) {
            bad = true;
            break;
        }
        const uint32_t end = min(k1, w0 + kWindow);
        for (uint32_t t0 = w0 + 32 * wv; t0 < end; t0 += 32 * kWaves) {
            const uint32_t* of = off + (t0 - w0);
            // every load of the step, K first
            uint32_t kr[2][NC][KW], vr[8][VW];
            uint32_t vs[8];
            uint64_t ksc[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const uint8_t* row = kb + (size_t)of[16 * kt + n] * 16;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    if constexpr (KW == 4) {
                        const u4 w = gld<u4>(row + 64 * c);
                        kr[kt][c][0] = w.x, kr[kt][c][1] = w.y, kr[kt][c][2] = w.z, kr[kt][c][3] = w.w;
                    } else {
                        const uint2 w = gld<uint2>(row + 32 * c);
                        kr[kt][c][0] = w.x, kr[kt][c][1] = w.y;
                    }
                }
            }
            uint32_t vo[8];
#pragma unroll
            for (int j = 0; j < 8; j++) vo[j] = of[(j & 4) * 4 + 4 * g + (j & 3)];
            if constexpr (C == Q8_0) {
#pragma unroll
                for (int j = 0; j < 8; j++) {  // of the keys that the lane's scores belong to
                    if constexpr (NC == 4) ksc[j / 4][j % 4] = gld<uint64_t>(ksb + vo[j]);
                    else ksc[j / 4][j % 4] = gld<uint32_t>(ksb + vo[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint8_t* row = vb + (size_t)vo[j] * 16;
                if constexpr (VW == 4) {
                    const u4 w = gld<u4>(row);
                    vr[j][0] = w.x, vr[j][1] = w.y, vr[j][2] = w.z, vr[j][3] = w.w;
                } else if constexpr (VW == 2) {
                    const uint2 w = gld<uint2>(row);
                    vr[j][0] = w.x, vr[j][1] = w.y;
                } else {
                    vr[j][0] = gld<uint32_t>(row);
                }
                if constexpr (C == Q8_0) vs[j] = gld<uint16_t>(vsb + vo[j]);
            }
            f4 s[2];
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
                            s[kt][r] = fmaf(acc[r], (float)__builtin_bit_cast(_Float16, (uint16_t)(ksc[kt][r] >> (16 * c))),
                                            s[kt][r]);
                    } else {
                        s[kt] = mfma32<C>(u4{kr[kt][c][0], kr[kt][c][1], kr[kt][c][2], kr[kt][c][3]}, q[c], s[kt]);
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; r++) s[kt][r] *= qs;
            }
            if (a.score && n < nh) {  // nh is at most 8; the row holds whole steps
#pragma unroll
                for (int kt = 0; kt < 2; kt++)
                    *reinterpret_cast<f4*>(a.score + ((size_t)b * a.heads + h0 + n) * a.score_row + t0 + 16 * kt + 4 * g) = s[kt];
            }
            if (t0 + 32 > k1) {  // no weight, and no value, past the end
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const bool past = t0 + (j & 4) * 4 + 4 * g + (j & 3) >= k1;
                    if (past) s[j / 4][j % 4] = -INFINITY;
#pragma unroll
                    for (int i = 0; i < VW; i++) vr[j][i] = past ? 0u : vr[j][i];
                    if constexpr (C == Q8_0) vs[j] = past ? 0u : vs[j];
                }
            }
            float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                              fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            if (__any(top > m + 15.f)) {
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float M = fmaxf(m, top - 7.f), alpha = M == -INFINITY ? 1.f : exp2_of(m - M);
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
                const uint32_t hi = pack2<C>(x, y);
                const float2 back = unpack2<C>(hi);
                const uint32_t lo = pack2<C>(x - back.x, y - back.y);
                p[i] = n < 8 ? hi : lo;
            }
            if constexpr (C == Q8_0) {
                h2 d[4];
#pragma unroll
                for (int i = 0; i < 4; i++) d[i] = __builtin_bit_cast(h2, vs[2 * i] | vs[2 * i + 1] << 16);
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int i = 0; i < VW; i++) vr[j][i] ^= 0x80808080u;
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    u4 hi, lo;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t sel = 0x0c000c00u | (uint32_t)(t % 4) | (uint32_t)(4 + t % 4) << 16;
                        const h2 c = codes2(__builtin_amdgcn_perm(vr[2 * i + 1][t / 4], vr[2 * i][t / 4], sel) | 0x64006400u);
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
        }
    }
    if (bad) l = __builtin_nanf("");
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) {  // the lo parts' sums, from column n + 8
            const float lo = __shfl_xor(o[t][r], 8, 64);
            if (finite_f(o[t][r])) o[t][r] += lo;
        }
    if (n < 8) {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) red[wv][n][(4 * g + r) * NT + t] = o[t][r];
        if (g == 0) {
            rm[wv][n] = m;
            rl[wv][n] = l;
        }
    }
    __syncthreads();
    merge_waves<8, D>(a, b, h0, nh, part, red, rm, rl);
}

// The parts in use of a sequence of n keys (one where it has none).
__device__ __forceinline__ uint32_t parts_of(const PageAttn& a, int32_t len) {
    return len <= 0 ? 1u : ((uint32_t)len + a.span - 1) / a.span;
}

// (max, sum) of head h's parts, by one wave.
__device__ __forceinline__ float2 fold_parts(const PageAttn& a, uint32_t b, uint32_t h, uint32_t parts, uint32_t lane) {
    const float* ml = a.ml + 2 * ((size_t)b * a.heads + h) * a.splits;
    float M = -INFINITY, L = 0.f;
    for (uint32_t i = lane; i < parts; i += 64) M = fmaxf(M, gld<float>(ml + 2 * i));
    M = wave_max(M);
    if (M == -INFINITY) M = 0.f;
    for (uint32_t i = lane; i < parts; i += 64) L += gld<float>(ml + 2 * i + 1) * exp2_of(gld<float>(ml + 2 * i) - M);
    L = wave_sum(L);
    return {M, L};
}

// out[b][h] from its parts: a workgroup per sequence and head.
__global__ __launch_bounds__(kBlock) void k_page_join(PageAttn a) {
    const uint32_t h = blockIdx.x, b = blockIdx.y, d = a.c.dim, parts = parts_of(a, length_of(a.r, b));
    const float2 mi = fold_parts(a, b, h, parts, threadIdx.x & 63);
    const size_t slot = ((size_t)b * a.heads + h) * a.splits;
    for (uint32_t j = threadIdx.x; j < d; j += kBlock) {
        float O = 0.f;
        for (uint32_t i = 0; i < parts; i++)
            O = fmaf(gld<float>(a.o + (slot + i) * d + j), exp2_of(gld<float>(a.ml + 2 * (slot + i)) - mi.x), O);
        put_kind(a.out.kind, a.out.p, b * a.out.row + h * a.out.head + j, mi.y == 0.f ? 0.f : O / mi.y);
    }
}

// wout[b][g][t] = win[b][g][t] + sum over g's query heads of exp(s - m) / l:
// a workgroup per kBlock keys of a sequence and KV head.  In the heads' order,
// so the same bits on every call.
__global__ __launch_bounds__(kBlock) void k_page_weights(PageAttn a) {
    const uint32_t g = blockIdx.y, b = blockIdx.z, G = a.heads / a.c.kvheads;
    const int32_t len = length_of(a.r, b);
    if ((int32_t)(blockIdx.x * kBlock) >= len) return;
    const uint32_t t = blockIdx.x * kBlock + threadIdx.x, parts = parts_of(a, len);
    float w = 0.f;
    for (uint32_t i = 0; i < G; i++) {
        const uint32_t h = g * G + i;
        const float2 mi = fold_parts(a, b, h, parts, threadIdx.x & 63);
        if ((int32_t)t < len && mi.y != 0.f)
            w += exp2_of(gld<float>(a.score + ((size_t)b * a.heads + h) * a.score_row + t) - mi.x) / mi.y;
    }
    if ((int32_t)t >= len) return;
    if (a.win) w += gld<float>(a.win + b * a.win_row + g * a.win_head + t);
    a.wout[b * a.wout_row + g * a.wout_head + t] = w;
}

// Whether k_page_attn16 takes the call: 16-bit queries of the cache's type (or
// over Q8_0), heads of 64 or 128, rows aligned to 16 bytes within 64 GiB.
static bool fits16(const PageAttn& a) {
    const bool q8 = a.c.kind == Q8_0;
    if (a.q.kind == F32 || (!q8 && a.c.kind != a.q.kind) || (a.c.dim != 64 && a.c.dim != 128)) return false;
    const uint64_t es = q8 ? 1 : 2, all = a.c.ps | a.c.ts | a.c.hs;
    if (((uintptr_t)a.c.k | (uintptr_t)a.c.v | all * es) % 16) return false;
    // a key's scales are one load
    if (q8 && (all % a.c.dim || ((uintptr_t)a.c.ks | (uintptr_t)a.c.vs) % (a.c.dim / 16))) return false;
    return ((a.c.count - 1) * a.c.ps + (a.c.page - 1) * a.c.ts) * es < (uint64_t)1 << 36;
}

// Parts of at least 128 keys, and as many as give the chip about 1,024
// workgroups of eight query heads.
size_t page_attn_plan(PageAttn& a, bool weights) {
    const uint32_t G = a.heads / a.c.kvheads;
    a.groups = (G + 7) / 8;
    a.per = (G + a.groups - 1) / a.groups;
    const uint64_t most = std::max<uint32_t>(a.r.most, 1), blocks = (uint64_t)a.r.batch * a.c.kvheads * a.groups;
    const uint64_t units = (uint64_t)a.r.batch * a.heads;
    uint64_t span = (most * blocks / 1024 + 127) / 128 * 128;
    span = std::max<uint64_t>(span, ((most + kPageMaxSplits - 1) / kPageMaxSplits + 127) / 128 * 128);
    span = std::min<uint64_t>(std::max<uint64_t>(span, 128), (most + 127) / 128 * 128);
    a.span = (uint32_t)span;
    a.splits = (uint32_t)((most + span - 1) / span);
    a.score_row = (most + 63) / 64 * 64;
    if (a.splits == 1 && !weights) return 0;
    const uint64_t slots = units * a.splits;
    return (slots * (2 + a.c.dim) + (weights ? units * a.score_row : 0)) * 4 + 64;
}

void page_attn_place(PageAttn& a, void* work, bool weights) {
    a.ml = a.o = a.score = nullptr;
    if (a.splits == 1 && !weights) return;
    const uint64_t units = (uint64_t)a.r.batch * a.heads, slots = units * a.splits;
    a.o = static_cast<float*>(work);
    if (weights) a.score = a.o + (slots * a.c.dim + 3) / 4 * 4;
    a.ml = weights ? a.score + units * a.score_row : a.o + (slots * a.c.dim + 3) / 4 * 4;
}

template <uint32_t K> static void launch_any(const PageAttn& a, hipStream_t s) {
    const dim3 grid(a.heads, a.splits, a.r.batch), block(kBlock);
    if (a.c.dim <= 64) hipLaunchKernelGGL((k_page_attn_any<K, 8>), grid, block, 0, s, a);
    else if (a.c.dim <= 128) hipLaunchKernelGGL((k_page_attn_any<K, 16>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_page_attn_any<K, 32>), grid, block, 0, s, a);
}

template <uint32_t C> static void launch16(const PageAttn& a, hipStream_t s) {
    const dim3 grid(a.c.kvheads * a.groups, a.splits, a.r.batch), block(kBlock);
    if (a.c.dim == 64) hipLaunchKernelGGL((k_page_attn16<C, 64>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_page_attn16<C, 128>), grid, block, 0, s, a);
}

void launch_page_attn(const PageAttn& a, hipStream_t s) {
    if (fits16(a)) {
        if (a.c.kind == F16) launch16<F16>(a, s);
        else if (a.c.kind == BF16) launch16<BF16>(a, s);
        else launch16<Q8_0>(a, s);
    } else if (a.c.kind == F32) launch_any<F32>(a, s);
    else if (a.c.kind == F16) launch_any<F16>(a, s);
    else if (a.c.kind == BF16) launch_any<BF16>(a, s);
    else launch_any<Q8_0>(a, s);
    if (!a.ml) return;
    hipLaunchKernelGGL(k_page_join, dim3(a.heads, a.r.batch), dim3(kBlock), 0, s, a);
    if (a.score && a.r.most)
        hipLaunchKernelGGL(k_page_weights, dim3((a.r.most + kBlock - 1) / kBlock, a.c.kvheads, a.r.batch), dim3(kBlock),
                           0, s, a);
}

}  // namespace qh
