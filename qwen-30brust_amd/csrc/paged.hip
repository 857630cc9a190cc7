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
//   s_t = scale * q . k_t,  m = max s_t,  l = sum exp(s_t - m),
//   o = sum exp(s_t - m) v_t / l
// over the keys of one sequence, in parts of `span` keys whose (m, l, o) are
// folded by k_page_join; everything in 32 bits.  A row with no keys, or whose
// scores are all -inf, is zeros.

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
        s *= a.scale;
        if (t >= k1) continue;  // not 0 times the value of a key past the end
        if (a.score && p == 0) a.score[((size_t)b * a.heads + h) * a.score_row + t] = s;
        const float M = fmaxf(m, s), Mf = M == -INFINITY ? 0.f : M;
        const float alpha = expf(m - Mf), e = expf(s - Mf);
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
    const float e = expf(m - (M == -INFINITY ? 0.f : M));
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
    for (int x = 0; x < kWaves; x++) L = fmaf(rl[x], expf(rm[x] - Mf), L);
    const size_t slot = ((size_t)b * a.heads + h) * a.splits + part;
    for (uint32_t j = threadIdx.x; j < d; j += kBlock) {
        float O = 0.f;
        for (int x = 0; x < kWaves; x++) O = fmaf(red[x][j], expf(rm[x] - Mf), O);
        if (a.ml) a.o[slot * d + j] = O;
        else put_kind(a.out.kind, a.out.p, b * a.out.row + h * a.out.head + j, L == 0.f ? 0.f : O / L);
    }
    if (a.ml && threadIdx.x == 0) {
        a.ml[2 * slot] = Ma;
        a.ml[2 * slot + 1] = L;
    }
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
    for (uint32_t i = lane; i < parts; i += 64) L += gld<float>(ml + 2 * i + 1) * expf(gld<float>(ml + 2 * i) - M);
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
            O = fmaf(gld<float>(a.o + (slot + i) * d + j), expf(gld<float>(a.ml + 2 * (slot + i)) - mi.x), O);
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
            w += expf(gld<float>(a.score + ((size_t)b * a.heads + h) * a.score_row + t) - mi.x) / mi.y;
    }
    if ((int32_t)t >= len) return;
    if (a.win) w += gld<float>(a.win + b * a.win_row + g * a.win_head + t);
    a.wout[b * a.wout_row + g * a.wout_head + t] = w;
}

// Parts of at least 128 keys, and as many as give the chip about 1,024
// workgroups.
size_t page_attn_plan(PageAttn& a, bool weights) {
    const uint64_t most = std::max<uint32_t>(a.r.most, 1), units = (uint64_t)a.r.batch * a.heads;
    uint64_t span = (most * units / 1024 + 127) / 128 * 128;
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

void launch_page_attn(const PageAttn& a, hipStream_t s) {
    if (a.c.kind == F32) launch_any<F32>(a, s);
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
