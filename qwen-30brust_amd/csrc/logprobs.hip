// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits, with the padding-vocabulary mask of src/main.rs:262-266 (masked
// ids read as f32::MIN, as the sampler reads them):
//   m = max x,  S = sum exp(x - m),  log p_t = x_t - m - log S,
//   U = sum (x - m) exp(x - m),  H = log S - U / S
// in 32 bits.  The alternatives are in descending total order, the lower id on
// ties.  A row that holds NaN or +inf gives NaN; one of -inf alone gives -inf
// and no entropy; a target outside the vocabulary gives NaN.
//
// One pass over the logits, in batches of 1,024 of a row.  All rows' batches, one
// behind the other, are dealt to waves in equal runs, as many as fill the chip: a
// single row and hundreds of them both do.  A row that one wave holds whole is
// done there; of others every wave that holds a part leaves its (m, S, U) and its
// top keys in one of its two slots (0: a part that starts inside its row, 1: one
// that starts with it), and k_logprobs_join folds them.  Every lane keeps the (m,
// S, U) of its own logits; a new maximum m' takes S to a S and U to a (U + (m -
// m') S), a = exp(m - m').
// The alternatives: a wave keeps its part's top keys (a logit's order and its id,
// so that no two are alike) in its lanes' registers, in descending order.  Only
// logits above the top-th of them can get in (one that equals it has a higher id);
// of a batch with many such, as the first, only those that the top-th largest of
// its loads' maxima lets through.  A key is put in its place by counting the keys
// above it and moving the others up a lane: about a hundred cycles, and a part of
// n batches of random logits has some top (1 + ln n) of them.
//
// 777 rows of 151,936 f32 logits (472 MB): 81 us for the sums alone, memory's rate
// (5.9 TB/s; 88 without the next batch under way); with 20 alternatives 122 us and
// 11 for the join: finding and placing some 90 keys a wave, half of it hidden behind
// the loads (a list in LDS filled with atomics took 157 us).  With 128
// alternatives, two keys a lane, 399 and 37.  One such row: 9 and 8 us,
// latency.
#include <algorithm>
#include <cfloat>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr uint32_t kLpLane = 16;                     // logits of a lane and batch
constexpr uint32_t kLpBatch = 64 * kLpLane;
constexpr uint32_t kLpMany = 32;                     // lanes that hold logits of a batch above the bound
constexpr uint32_t kLpRuns = 4096;                   // waves that fill the chip

__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_key(x) << 32 | (uint32_t)~i; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // v_exp_f32

// (m, S, U) of some logits, m in units of log 2 and U with it: t = x log2(e) - m
// is one fused multiply-add, of which a large x loses nothing, S = sum 2^t, U =
// sum t 2^t, log p = (t - log2 S) ln 2.  m is rounded and the product in t is
// not, so that t reaches half a step of m, 1 for an x of 2^24: a row whose maximum
// lies past that either way, or just above -2^24 with logits below it, is far, and m
// is the maximum itself (slow_sums).
struct Sums {
    float m = -INFINITY, S = 0.f, U = 0.f;
    __device__ __forceinline__ void move(float M) {  // to a maximum M >= m
        const float a = m == -INFINITY ? 0.f : exp2_of(m - M);
        U = a > 0.f ? a * fmaf(m - M, S, U) : 0.f;
        S *= a;
        m = M;
    }
    __device__ __forceinline__ void add(Sums o) {
        const float M = fmaxf(m, o.m);
        move(M);
        o.move(M);
        S += o.S;
        U += o.U;
    }
};

// The largest order key of the upper 20 bits (11 of a mantissa) that at least n of
// the wave's R keys a lane reach (0 where there are fewer).
template <uint32_t R> __device__ __forceinline__ uint32_t nth_of(const uint32_t (&v)[R], uint32_t n) {
    uint32_t found = 0;
#pragma unroll 4
    for (int bit = 31; bit >= 12; bit--) {
        const uint32_t t = found | 1u << bit;
        uint32_t reach = 0;
#pragma unroll
        for (uint32_t k = 0; k < R; k++) reach += __popcll(__ballot(v[k] >= t));
        if (reach >= n) found = t;
    }
    return found;
}

// The largest 64 R keys that came, in descending order: the i-th in lane i % 64 of
// key[i / 64]; 0: none.
template <uint32_t R> struct Best {
    uint64_t key[R] = {};
    __device__ __forceinline__ static uint64_t up(uint64_t v, uint64_t in) {  // a lane up, `in` into lane 0
        const uint32_t lo = __builtin_amdgcn_update_dpp((uint32_t)in, (uint32_t)v, 0x138, 0xf, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp((uint32_t)(in >> 32), (uint32_t)(v >> 32), 0x138, 0xf, 0xf, false);
        return (uint64_t)hi << 32 | lo;
    }
    __device__ __forceinline__ static uint64_t of_lane(uint64_t v, uint32_t l) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), l) << 32 |
               (uint32_t)__builtin_amdgcn_readlane((uint32_t)v, l);
    }
    __device__ __forceinline__ uint64_t at(uint32_t i) const {
        uint64_t v = of_lane(key[0], i & 63);
        if constexpr (R == 2) v = i < 64 ? v : of_lane(key[1], i & 63);
        return v;
    }
    // c, the same in every lane.
    __device__ __forceinline__ void put(uint64_t c) {
        const uint32_t lane = threadIdx.x;
        uint64_t spill = 0;  // what leaves lane 63 of a row
#pragma unroll
        for (uint32_t r = 0; r < R; r++) {
            const uint32_t above = __popcll(__ballot(key[r] > c));  // a row of larger keys stays
            const uint64_t last = of_lane(key[r], 63), moved = up(key[r], spill);
            const uint64_t in = r && spill ? spill : c;
            const uint32_t place = r && spill ? 0 : above;
            key[r] = lane < place ? key[r] : lane == place ? in : moved;
            spill = place < 64 ? last : 0;
            if (place < 64 && last == 0) break;
        }
    }
};

// The wave's Sums, in every lane.
__device__ __forceinline__ Sums fold(Sums s) {
    s.move(wave_max(s.m));
    s.S = wave_sum(s.S);
    s.U = wave_sum(s.U);
    return s;
}

// What a row's logits hold, besides: NaN or +inf; finite maxima past 2^24.  A lane
// whose logits of a batch all lie below -2^24 leaves them out of its sums (kLpLow):
// they have no weight where the row's maximum lies kLpClear above, e^-256, and a row
// whose maximum does not is far too.
enum : uint32_t { kLpBad = 1, kLpHigh = 2, kLpLow = 4 };
constexpr float kLpFar = 16777216.f, kLpClear = 256.f;
__device__ __forceinline__ uint32_t any_of(uint32_t flags) {
    uint32_t r = 0;
#pragma unroll
    for (uint32_t f = 1; f <= kLpLow; f *= 2) r |= __any(flags & f) ? f : 0;
    return r;
}

__device__ __forceinline__ float logp_of(float x, const Sums& s, bool far, bool bad) {
    if (bad) return __builtin_nanf("");
    if (x == -INFINITY) return x;
    const float t = far ? (x - s.m) * kLog2e : fmaf(x, kLog2e, -s.m);
    if (t == -INFINITY) return far ? x - s.m : x - s.m * kLn2;  // f32::MIN among other logits
    return (t - log2f(s.S)) * kLn2;
}

// The Sums of row r about its maximum, by a wave.
template <uint32_t K> __device__ __forceinline__ Sums slow_sums(const Logprobs& a, uint32_t r) {
    auto logit = [&](uint32_t i) {
        const bool masked = a.valid && !gld<uint8_t>(a.valid + i);
        return masked ? -FLT_MAX : elem<K>(static_cast<const uint8_t*>(a.x), r * a.stride + i);
    };
    Sums s;
    float m = -INFINITY;
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < a.vocab; i += 64) m = fmaxf(m, logit(i));
    s.m = wave_max(m);
#pragma unroll 8
    for (uint32_t i = threadIdx.x; i < a.vocab; i += 64) {
        const float t = (logit(i) - s.m) * kLog2e, e = exp2_of(t);
        s.S += e;
        s.U = fmaf(fmaxf(t, -200.f), e, s.U);
    }
    s.S = wave_sum(s.S);
    s.U = wave_sum(s.U);
    return s;
}

// The target's logit of row r, on its way while the sums are folded.
struct Target {
    bool in = false;
    float x = 0.f;
    template <uint32_t K> static __device__ __forceinline__ Target load(const Logprobs& a, uint32_t r) {
        Target t;
        if (!a.logp) return t;
        const uint32_t id = (uint32_t)gld<int32_t>(a.target + r);
        t.in = id < a.vocab;
        if (t.in) {
            t.x = elem<K>(static_cast<const uint8_t*>(a.x), r * a.stride + id);
            if (a.valid && !gld<uint8_t>(a.valid + id)) t.x = -FLT_MAX;
        }
        return t;
    }
};

// A row whose Sums and flags are known: writes its log probability and entropy,
// and gives that of others.
template <uint32_t K> struct Row {
    Sums s;
    bool bad, far;
    __device__ __forceinline__ Row(const Logprobs& a, uint32_t r, const Target& t, Sums sums, uint32_t flags) : s(sums) {
        bad = flags & kLpBad;
        far = !bad && ((flags & kLpHigh) || (flags & kLpLow && s.m < (kLpClear - kLpFar) * kLog2e));
        if (far) {
            s = slow_sums<K>(a, r);
            bad = s.S != s.S;
        }
        if (threadIdx.x) return;
        if (a.logp) a.logp[r] = t.in ? logp(t.x) : __builtin_nanf("");
        if (a.entropy) a.entropy[r] = bad ? __builtin_nanf("") : s.S > 0.f ? (log2f(s.S) - s.U / s.S) * kLn2 : 0.f;
    }
    __device__ __forceinline__ float logp(float x) const { return logp_of(x, s, far, bad); }
    __device__ __forceinline__ void put(const Logprobs& a, uint32_t r, uint32_t rank, uint64_t k) const {
        a.ids[(size_t)r * a.top + rank] = (int32_t) ~(uint32_t)k;
        a.alt[(size_t)r * a.top + rank] = logp(key_value((uint32_t)(k >> 32)));
    }
};

// f(rank, key) for the first `top` keys.
template <uint32_t R, class F> __device__ __forceinline__ void each(const Best<R>& best, uint32_t top, F f) {
#pragma unroll
    for (uint32_t r = 0; r < R; r++)
        if (threadIdx.x + 64 * r < top) f(threadIdx.x + 64 * r, best.key[r]);
}

// Of the batches, `all` a row, the first `more` runs hold len + 1 each, the others
// len.
struct Runs {
    uint32_t all, runs, more;
    uint64_t len;
    static __host__ __device__ uint64_t div(uint64_t a, uint64_t b) {
        return (a | b) >> 32 ? a / b : (uint32_t)a / (uint32_t)b;
    }
    __host__ __device__ uint64_t begin(uint32_t i) const { return i * len + (i < more ? i : more); }
    __host__ __device__ uint64_t with(uint64_t x) const {  // the run of batch x
        const uint64_t head = more * (len + 1);
        return x < head ? div(x, len + 1) : more + div(x - head, len);
    }
};

// The logits and mask bytes of one load: 16 bytes of a row, whatever their
// alignment, so that a wave's loads are whole lines.
template <uint32_t K> struct Load {
    static constexpr uint32_t E = K == F32 ? 4 : 8, kSteps = kLpLane / E, kStep = 64 * E;
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t masks __attribute__((ext_vector_type(E / 4), aligned(1)));
    words w;
    masks valid;
    __device__ __forceinline__ void load(const uint8_t* p, const uint8_t* v) {
#if defined(__HIP_DEVICE_COMPILE__)
        w = __builtin_nontemporal_load((gptr<words>)p);  // read once
#endif
        if (v) valid = gld<masks>(v);
    }
    // Of a row of fewer than E logits.
    __device__ __forceinline__ void few(const uint8_t* p, const uint8_t* v, uint32_t n) {
        w = words(0u);
        valid = masks(0u);
#pragma unroll
        for (uint32_t j = 0; j < E; j++) {
            const uint32_t i = min(j, n - 1);
            if constexpr (K == F32) w[j] = gld<uint32_t>(p + 4 * i);
            else w[j / 2] |= (uint32_t)gld<uint16_t>(p + 2 * i) << 16 * (j % 2);
            if (v) valid[j / 4] |= (uint32_t)gld<uint8_t>(v + i) << 8 * (j % 4);
        }
    }
    // Not 0 where a byte is not 1.
    __device__ __forceinline__ uint32_t masked() const {
        uint32_t off = valid[0] ^ 0x01010101u;
        if constexpr (E == 8) off |= valid[1] ^ 0x01010101u;
        return off;
    }
    __device__ __forceinline__ bool on(uint32_t j) const {
        const uint32_t word = valid[j / 4];
        return word >> (8 * (j % 4)) & 255;
    }
    __device__ __forceinline__ float at(uint32_t j) const {
        if constexpr (K == F32) {
            return __uint_as_float(w[j]);
        } else {
            const uint32_t pair = w[j / 2];
            if constexpr (K == BF16) return __uint_as_float(j % 2 ? pair & 0xffff0000u : pair << 16);
            const uint16_t half = (uint16_t)(j % 2 ? pair >> 16 : pair);
            return (float)__builtin_bit_cast(_Float16, half);
        }
    }
};

// Work: [runs][2] (m, S, U, flags), then [runs][2][top] keys.
__device__ __forceinline__ float4* sums_of(const Logprobs& a) { return static_cast<float4*>(a.work); }
__device__ __forceinline__ uint64_t* keys_of(const Logprobs& a, uint32_t runs) {
    return reinterpret_cast<uint64_t*>(sums_of(a) + 2 * (size_t)runs);
}

template <uint32_t K, uint32_t R> __global__ __launch_bounds__(64, 4) void k_logprobs(Logprobs a, Runs w) {
    const uint32_t lane = threadIdx.x, top = a.top;
    uint64_t at = w.begin(blockIdx.x);
    const uint64_t end = w.begin(blockIdx.x + 1);
    while (at < end) {
        const uint32_t r = (uint32_t)Runs::div(at, w.all), b0 = (uint32_t)(at - (uint64_t)r * w.all);
        const uint32_t b1 = (uint32_t)min((uint64_t)w.all, b0 + (end - at));
        at += b1 - b0;
        const uint8_t* row = static_cast<const uint8_t*>(a.x) + r * a.stride * (K == F32 ? 4 : 2);
        const uint32_t lo = b0 * kLpBatch, hi = min(a.vocab, b1 * kLpBatch);
        Best<R> best;
        Sums s;
        uint32_t flags = 0;
        float bound = -INFINITY;  // logits below it do not get in
        constexpr uint32_t E = Load<K>::E, kSteps = Load<K>::kSteps, kStep = Load<K>::kStep;
        // Lane's loads k of a batch: logits i .. i + E - 1, i = b + kStep k + lane E; the
        // last ones of a row end with it, and hold some again that other loads hold
        Load<K> raw[kSteps];
        auto request = [&](uint32_t b) {
            const uint32_t last = b + kLpBatch <= hi ? ~0u : hi - min(hi, E);
#pragma unroll
            for (uint32_t k = 0; k < kSteps; k++) {
                const uint32_t i = min(b + kStep * k + lane * E, last);
                if (hi >= E) raw[k].load(row + (size_t)i * (K == F32 ? 4 : 2), a.valid ? a.valid + i : nullptr);
                else raw[k].few(row, a.valid, hi);
            }
        };
        request(lo);
        for (uint32_t b = lo; b < hi; b += kLpBatch) {
            const bool whole = b + kLpBatch <= hi;
            auto at_of = [&](uint32_t k) { return b + kStep * k + lane * E; };
            auto from_of = [&](uint32_t k) { return whole ? at_of(k) : min(at_of(k), hi - min(hi, E)); };
            float x[kSteps][E], M[kSteps], most = -INFINITY;
#pragma unroll
            for (uint32_t k = 0; k < kSteps; k++)
#pragma unroll
                for (uint32_t j = 0; j < E; j++) x[k][j] = raw[k].at(j);
            if (a.valid) {
                uint32_t off = 0;
#pragma unroll
                for (uint32_t k = 0; k < kSteps; k++) off |= raw[k].masked();
                if (__any(off)) {
#pragma unroll
                    for (uint32_t k = 0; k < kSteps; k++)
#pragma unroll
                        for (uint32_t j = 0; j < E; j++) x[k][j] = raw[k].on(j) ? x[k][j] : -FLT_MAX;
                }
            }
            // the next batch is on its way while this one is worked on
            __builtin_amdgcn_sched_barrier(0);
            if (b + kLpBatch < hi) request(b + kLpBatch);
            __builtin_amdgcn_sched_barrier(0);
            if (!whole) {
#pragma unroll
                for (uint32_t k = 0; k < kSteps; k++)
#pragma unroll
                    for (uint32_t j = 0; j < E; j++) {
                        const uint32_t i = from_of(k) + j;
                        x[k][j] = i >= at_of(k) && i < hi ? x[k][j] : -INFINITY;
                    }
            }
#pragma unroll
            for (uint32_t k = 0; k < kSteps; k++) {
                M[k] = x[k][0];
#pragma unroll
                for (uint32_t j = 1; j < E; j++) M[k] = fmaxf(M[k], x[k][j]);  // NaN only if all are
                most = fmaxf(most, M[k]);
            }
            if (most >= -kLpFar && most * kLog2e > s.m) s.move(most * kLog2e);
            const float m = s.m == -INFINITY ? 0.f : s.m;
            float S = 0.f, U = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < kSteps; k++)
#pragma unroll
                for (uint32_t j = 0; j < E; j++) {
                    const float t = fmaf(x[k][j], kLog2e, -m), e = exp2_of(t);
                    S += e;
                    U = fmaf(fmaxf(t, -200.f), e, U);  // 0, not NaN, for -inf
                }
            s.S += S;
            s.U += U;
            if (fabsf(most) > kLpFar && most != -INFINITY) flags |= most == INFINITY ? kLpBad : most > 0.f ? kLpHigh : kLpLow;
            if (S != S) flags |= kLpBad;  // of finite logits, however large, no term is NaN
            if (!top) continue;
            const uint64_t some = __ballot(!(most < bound)), bad = __ballot(flags & kLpBad);
            if (!(some | bad)) continue;
            float low = bound;
            if (__popcll(some) > kLpMany) {
                uint32_t mine[kSteps];
#pragma unroll
                for (uint32_t k = 0; k < kSteps; k++) mine[k] = at_of(k) < hi ? order_key(M[k]) : 0;
                const uint32_t t = nth_of(mine, top);
                if (t && key_value(t) > low) low = key_value(t);
            }
#pragma unroll
            for (uint32_t k = 0; k < kSteps; k++) {
                if (!(__ballot(!(M[k] < low)) | bad)) continue;
                const uint32_t at = at_of(k), i = from_of(k);
#pragma unroll
                for (uint32_t j = 0; j < E; j++) {
                    uint64_t who = __ballot(!(x[k][j] < low));
                    if (!whole) who &= __ballot(i + j >= at && i + j < hi);
                    for (; who; who &= who - 1) {
                        const uint32_t l = __ffsll((unsigned long long)who) - 1;
                        const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x[k][j]), l));
                        best.put(key_of(v, __builtin_amdgcn_readlane(i + j, l)));
                    }
                }
            }
            const uint32_t last = (uint32_t)(best.at(top - 1) >> 32);
            if (last) {
                bound = key_value(last);
                if (bound < INFINITY) bound = key_value(last + 1);
            }
        }
        flags = any_of(flags);
        s = fold(s);
        const size_t slot = (size_t)blockIdx.x * 2 + (b0 == 0);
        if (b1 - b0 == w.all) {
            const Row<K> done(a, r, Target::load<K>(a, r), s, flags);
            each(best, top, [&](uint32_t rank, uint64_t k) { done.put(a, r, rank, k); });
        } else {
            if (lane == 0) sums_of(a)[slot] = make_float4(s.m, s.S, s.U, __uint_as_float(flags));
            uint64_t* out = keys_of(a, w.runs) + slot * top;
            each(best, top, [&](uint32_t rank, uint64_t k) { out[rank] = k; });
        }
    }
}

// A row that several waves hold parts of.  Their keys lie in descending order.
// With n = ceil(top / parts), ceil(top / n) parts' n-th keys that reach a bound
// stand for top keys that do, so that only keys that reach the largest such bound
// are looked at, and none of a rank behind one where no part has any.  Bound by
// the look-ups' latency: what does not depend on another is loaded first (11 us
// for a row of 149 parts and 20 alternatives without, 8 with).
template <uint32_t K, uint32_t R> __global__ __launch_bounds__(64) void k_logprobs_join(Logprobs a, Runs w) {
    constexpr uint32_t kAhead = 8;  // keys of a lane in flight
    const uint32_t r = blockIdx.x, lane = threadIdx.x, top = a.top;
    const uint64_t x = (uint64_t)r * w.all, first = w.with(x);
    const uint32_t parts = (uint32_t)(w.with(x + w.all - 1) - first) + 1;
    if (parts == 1) return;  // done in its wave
    auto slot = [&](uint32_t i) { return (first + i) * 2 + (i == 0); };
    const uint64_t* keys = keys_of(a, w.runs);
    const uint32_t n = (top + parts - 1) / parts, all = parts * top;
    // what the first 256 parts left and the target, all under way at once
    uint32_t nth[4] = {};
    float4 sums[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        const uint32_t i = min(lane + 64 * k, parts - 1);
        sums[k] = gld<float4>(sums_of(a) + slot(i));
        if (top) nth[k] = (uint32_t)(gld<uint64_t>(keys + slot(i) * top + n - 1) >> 32);
    }
    const Target target = Target::load<K>(a, r);
    Sums s;
    uint32_t flags = 0;
    auto add = [&](float4 v) {
        Sums o;
        o.m = v.x, o.S = v.y, o.U = v.z;
        s.add(o);
        flags |= __float_as_uint(v.w);
    };
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        if (lane + 64 * k < parts) add(sums[k]);
        else nth[k] = 0;
    }
    for (uint32_t i = lane + 256; i < parts; i += 64) add(gld<float4>(sums_of(a) + slot(i)));
    Best<R> best;
    if (top) {
        uint64_t bound = 1;  // 0: a part of fewer keys
        if (parts <= 256) bound = max((uint64_t)nth_of(nth, (top + n - 1) / n) << 32, (uint64_t)1);
        for (uint32_t i0 = 0; i0 < all; i0 += 64 * kAhead) {
            uint64_t k[kAhead];
#pragma unroll
            for (uint32_t j = 0; j < kAhead; j++) {
                const uint32_t i = i0 + 64 * j + lane, rank = min(i, all - 1) / parts, part = min(i, all - 1) - rank * parts;
                k[j] = gld<uint64_t>(keys + slot(part) * top + rank);  // the parts' first keys first
                if (i >= all) k[j] = 0;
            }
            bool some = parts > 64 * kAhead;
#pragma unroll
            for (uint32_t j = 0; j < kAhead; j++) {
                some |= __any(k[j] >= bound);
                for (uint64_t who = __ballot(k[j] >= bound); who; who &= who - 1) {
                    const uint64_t c = Best<R>::of_lane(k[j], __ffsll((unsigned long long)who) - 1);
                    if (c >= bound) best.put(c);
                }
                bound = max(bound, best.at(top - 1));
            }
            if (!some) break;  // of every part a key, and none reached the bound
        }
    }
    const Row<K> done(a, r, target, fold(s), any_of(flags));
    each(best, top, [&](uint32_t rank, uint64_t k) { done.put(a, r, rank, k); });
}

static Runs lp_runs(uint32_t rows, uint32_t vocab) {
    Runs w{};
    w.all = (vocab + kLpBatch - 1) / kLpBatch;
    const uint64_t total = (uint64_t)rows * w.all;
    w.runs = (uint32_t)std::min<uint64_t>(total, kLpRuns);
    w.len = total / w.runs;
    w.more = (uint32_t)(total % w.runs);
    return w;
}

size_t logprobs_bytes(uint32_t rows, uint32_t vocab, uint32_t top) {
    const Runs w = lp_runs(rows, vocab);
    return (size_t)w.runs * 2 * (16 + 8 * (size_t)top);
}

template <uint32_t K, uint32_t R> static void launch(const Logprobs& a, hipStream_t s) {
    const Runs w = lp_runs(a.rows, a.vocab);
    hipLaunchKernelGGL((k_logprobs<K, R>), dim3(w.runs), dim3(64), 0, s, a, w);
    if (a.rows % w.runs)  // else every run holds whole rows
        hipLaunchKernelGGL((k_logprobs_join<K, R>), dim3(a.rows), dim3(64), 0, s, a, w);
}
template <uint32_t K> static void launch_kind(const Logprobs& a, hipStream_t s) {
    if (a.top <= 64) launch<K, 1>(a, s);
    else launch<K, 2>(a, s);
}

void launch_logprobs(const Logprobs& a, hipStream_t s) {
    if (a.kind == F32) launch_kind<F32>(a, s);
    else if (a.kind == F16) launch_kind<F16>(a, s);
    else launch_kind<BF16>(a, s);
}

}  // namespace qh
