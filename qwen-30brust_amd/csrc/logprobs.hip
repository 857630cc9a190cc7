// Log probabilities of given tokens, entropy and the top alternatives of rows
// of logits, with the padding-vocabulary mask of src/main.rs:262-266 (masked
// ids read as f32::MIN, as the sampler reads them):
//   m = max x,  S = sum exp(x - m),  log p_t = x_t - m - log S,
//   U = sum (x - m) exp(x - m),  H = log S - U / S
// in 32 bits.  The alternatives are in descending total order, the lower id on
// ties.  A row that holds NaN or +inf gives NaN; one of -inf alone gives -inf
// and no entropy; a target outside the vocabulary gives NaN.
//
// One pass over the logits, in batches of 2,048 of a row.  All rows' batches, one
// behind the other, are dealt to waves in equal runs, as many as fill the chip: a
// single row and hundreds of them both do.  A row that one wave holds whole is
// done there; of others every wave that holds a part leaves its (m, S, U) and its
// top keys in one of its two slots (0: a part that starts inside its row, 1: one
// that starts with it), and k_logprobs_join folds them.  Every lane keeps the (m,
// S, U) of its own logits; a new maximum m' takes S to a S and U to a (U + (m -
// m') S), a = exp(m - m').
// The alternatives: of the first batch's 256 maxima of eight logits the top-th is
// a bound that top logits of the part reach, so only logits that reach it (of
// later batches: that are above it, since ties go to the lower id) can be among
// them.  They go to a list in LDS, a few more than top in a batch of random logits;
// it is cut back (cut) at the part's end, or before it could overflow, as rising
// rows make it.  The n-th largest of the lanes' numbers is found bit by bit, by
// counting lanes (nth_of).
#include <cfloat>

#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr uint32_t kLpLanes = 8;                     // logits of a load
constexpr uint32_t kLpStep = 64 * kLpLanes;          // of a wave's load
constexpr uint32_t kLpSteps = 4;                     // loads of a batch
constexpr uint32_t kLpBatch = kLpStep * kLpSteps;
constexpr uint32_t kLpList = 1536;                   // keys of a part's list
constexpr uint32_t kLpJoin = 4096;                   // and of a row's
constexpr uint32_t kLpRuns = 2048;                   // waves that fill the chip

__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return (uint64_t)order_key(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

// (m, S, U) of some logits.
struct Sums {
    float m = -INFINITY, S = 0.f, U = 0.f;
    __device__ __forceinline__ void move(float M) {  // to a maximum M >= m
        const float a = m == -INFINITY ? 0.f : exp_of(m - M);
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

// The largest number that at least n of the wave's R numbers a lane reach (0
// where there are fewer numbers).
template <typename T, uint32_t R> __device__ __forceinline__ T nth_of(const T (&v)[R], uint32_t n) {
    T found = 0;
#pragma unroll 4
    for (int bit = 8 * sizeof(T) - 1; bit >= 0; bit--) {
        const T t = found | (T)1 << bit;
        uint32_t reach = 0;
#pragma unroll
        for (uint32_t k = 0; k < R; k++) reach += __popcll(__ballot(v[k] >= t));
        if (reach >= n) found = t;
    }
    return found;
}

// Keys of one wave in LDS; the count is the same in every lane.
template <uint32_t N> struct List {
    uint64_t* key;
    uint32_t count = 0;
    __device__ __forceinline__ void append(bool on, uint64_t k) {
        const uint64_t who = __ballot(on);
        if (who == 0) return;
        if (on) key[count + __popcll(who & (((uint64_t)1 << (threadIdx.x & 63)) - 1))] = k;
        count += __popcll(who);
    }
    // To at least its top keys, and few more: keys below the top-th largest of 256
    // columns' maxima go.  At most top columns keep some (keys differ), so that a
    // pass halves the list or leaves one key a column.
    __device__ __forceinline__ void cut(uint32_t top) {
        while (count > 64 && count > top) {
            __syncthreads();  // (one wave: an order for the compiler)
            const uint32_t n = count, lane = threadIdx.x;
            uint64_t most[4] = {0, 0, 0, 0};
            for (uint32_t i = 0; i < n; i += 256)
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) {
                    const uint32_t j = i + lane + 64 * k;
                    if (j < n) most[k] = max(most[k], key[j]);
                }
            const uint64_t bound = max(nth_of(most, top), (uint64_t)1);  // 0: no key
            count = 0;
            for (uint32_t i = 0; i < n; i += 64) {  // a key moves forward, never past those still to be read
                const uint64_t k = i + lane < n ? key[i + lane] : 0;
                __syncthreads();
                append(k >= bound, k);
                __syncthreads();
            }
        }
    }
    // f(rank, key) for the top largest keys, each by some lane.
    template <class F> __device__ __forceinline__ void ranked(uint32_t top, F f) {
        cut(top);
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < count; i += 64) {
            const uint64_t k = key[i];
            uint32_t above = 0;
#pragma unroll 8
            for (uint32_t j = 0; j < count; j++) above += key[j] > k;
            if (above < top) f(above, k);
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

__device__ __forceinline__ float logp_of(float x, const Sums& s, bool bad) {
    return bad ? __builtin_nanf("") : x == -INFINITY ? x : x - s.m - logf(s.S);
}

// A row's numbers from its Sums and its list.
template <uint32_t K, uint32_t N>
__device__ __forceinline__ void finish_row(const Logprobs& a, List<N>& L, uint32_t r, const Sums& s, bool bad) {
    if (threadIdx.x == 0) {
        if (a.logp) {
            const uint32_t t = (uint32_t)gld<int32_t>(a.target + r);
            float p = __builtin_nanf("");
            if (t < a.vocab)
                p = logp_of(a.valid && !gld<uint8_t>(a.valid + t) ? -FLT_MAX
                                                                   : elem<K>(static_cast<const uint8_t*>(a.x), r * a.stride + t),
                            s, bad);
            a.logp[r] = p;
        }
        if (a.entropy) a.entropy[r] = bad ? __builtin_nanf("") : s.S > 0.f ? logf(s.S) - s.U / s.S : 0.f;
    }
    if (!a.top) return;
    L.ranked(a.top, [&](uint32_t rank, uint64_t k) {
        a.ids[(size_t)r * a.top + rank] = (int32_t) ~(uint32_t)k;
        a.alt[(size_t)r * a.top + rank] = logp_of(key_value((uint32_t)(k >> 32)), s, bad);
    });
}

// Run i holds batches [total i / runs, total (i + 1) / runs) of `all` a row.
struct Runs {
    uint32_t all, runs;
    uint64_t total;
    __host__ __device__ uint64_t begin(uint64_t i) const { return total * i / runs; }
    __host__ __device__ uint64_t with(uint64_t x) const { return ((x + 1) * runs + total - 1) / total - 1; }  // the run of batch x
};

// Eight logits from p, whatever its alignment.
template <uint32_t K> struct Eight {
    typedef uint32_t words __attribute__((ext_vector_type(K == F32 ? 8 : 4), aligned(K == F32 ? 4 : 2)));
    words w;
    __device__ __forceinline__ void load(const uint8_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
        w = __builtin_nontemporal_load((gptr<words>)p);  // read once
#else
        w = *reinterpret_cast<const words*>(p);  // host pass: never executed
#endif
    }
    __device__ __forceinline__ float at(uint32_t i) const {
        if constexpr (K == F32) {
            return __uint_as_float(w[i]);
        } else {
            const uint32_t pair = w[i / 2];
            if constexpr (K == BF16) return __uint_as_float(i % 2 ? pair & 0xffff0000u : pair << 16);
            return (float)__builtin_bit_cast(_Float16, (uint16_t)(i % 2 ? pair >> 16 : pair));
        }
    }
};

// Eight mask bytes, whatever their alignment.
__device__ __forceinline__ uint64_t eight_bytes(const uint8_t* p) {
    typedef uint32_t words __attribute__((ext_vector_type(2), aligned(1)));
    const words w = gld<words>(p);
    return (uint64_t)w.y << 32 | w.x;
}

// Work: [runs][2] (m, S, U, bad), then [runs][2][top] keys.
__device__ __forceinline__ float4* sums_of(const Logprobs& a) { return static_cast<float4*>(a.work); }
__device__ __forceinline__ uint64_t* keys_of(const Logprobs& a, uint32_t runs) {
    return reinterpret_cast<uint64_t*>(sums_of(a) + 2 * (size_t)runs);
}

template <uint32_t K> __global__ __launch_bounds__(64) void k_logprobs(Logprobs a, Runs w) {
    __shared__ uint64_t keys[kLpList];
    const uint32_t lane = threadIdx.x, top = a.top;
    uint64_t at = w.begin(blockIdx.x);
    const uint64_t end = w.begin(blockIdx.x + 1);
    while (at < end) {
        const uint32_t r = (uint32_t)(at / w.all), b0 = (uint32_t)(at % w.all);
        const uint32_t b1 = (uint32_t)min((uint64_t)w.all, b0 + (end - at));
        at += b1 - b0;
        const uint8_t* row = static_cast<const uint8_t*>(a.x) + r * a.stride * (K == F32 ? 4 : 2);
        const uint32_t lo = b0 * kLpBatch, hi = min(a.vocab, b1 * kLpBatch);
        List<kLpList> L{keys};
        Sums s;
        bool bad = false;
        float bound = -INFINITY;
        Eight<K> next[kLpSteps];
        uint64_t mask[kLpSteps];
        auto load = [&](uint32_t k, uint32_t i) {  // logits i .. i + 7, where all are there
            mask[k] = ~(uint64_t)0;
            if (i + kLpLanes > hi) return;
            next[k].load(row + (size_t)i * (K == F32 ? 4 : 2));
            if (a.valid) mask[k] = eight_bytes(a.valid + i);
        };
#pragma unroll
        for (uint32_t k = 0; k < kLpSteps; k++) load(k, lo + kLpStep * k + lane * kLpLanes);
        for (uint32_t b = lo; b < hi; b += kLpBatch) {
            float x[kLpSteps][kLpLanes], M[kLpSteps];
#pragma unroll
            for (uint32_t k = 0; k < kLpSteps; k++) {
                const uint32_t i = b + kLpStep * k + lane * kLpLanes;
                if (i + kLpLanes <= hi) {
#pragma unroll
                    for (uint32_t j = 0; j < kLpLanes; j++) x[k][j] = mask[k] >> (8 * j) & 255 ? next[k].at(j) : -FLT_MAX;
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < kLpLanes; j++)
                        x[k][j] = i + j >= hi ? -INFINITY : a.valid && !gld<uint8_t>(a.valid + i + j) ? -FLT_MAX : elem<K>(row, i + j);
                }
                load(k, i + kLpBatch);
            }
#pragma unroll
            for (uint32_t k = 0; k < kLpSteps; k++) {
                M[k] = x[k][0];
#pragma unroll
                for (uint32_t j = 1; j < kLpLanes; j++) M[k] = fmaxf(M[k], x[k][j]);  // NaN only if all are
            }
            const float most = fmaxf(fmaxf(M[0], M[1]), fmaxf(M[2], M[3]));
            if (most > s.m) s.move(most);
            const float m = s.m == -INFINITY ? 0.f : s.m;
            float S = 0.f, U = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < kLpSteps; k++)
#pragma unroll
                for (uint32_t j = 0; j < kLpLanes; j++) {
                    const float d = x[k][j] - m, e = exp_of(d);
                    S += e;
                    U = fmaf(fmaxf(d, -1e4f), e, U);  // 0, not NaN, for -inf
                }
            s.S += S;
            s.U += U;
            bad |= most == INFINITY || S != S;
            if (!top) continue;
            const bool first = b == lo;
            if (first) {
                uint32_t mine[kLpSteps];
#pragma unroll
                for (uint32_t k = 0; k < kLpSteps; k++)
                    mine[k] = b + kLpStep * k + lane * kLpLanes < hi ? order_key(M[k]) : 0;
                const uint32_t t = nth_of(mine, top);
                bound = t ? key_value(t) : -INFINITY;
            }
#pragma unroll
            for (uint32_t k = 0; k < kLpSteps; k++) {
                if (!__any(bad || (first ? !(M[k] < bound) : M[k] > bound))) continue;
                if (L.count > kLpList - kLpStep) L.cut(top);
                const uint32_t i = b + kLpStep * k + lane * kLpLanes;
#pragma unroll
                for (uint32_t j = 0; j < kLpLanes; j++)
                    L.append(i + j < hi && (first ? !(x[k][j] < bound) : !(x[k][j] <= bound)), key_of(x[k][j], i + j));
            }
        }
        const bool any = __any(bad);
        s = fold(s);
        if (b1 - b0 == w.all) {
            finish_row<K>(a, L, r, s, any);
        } else {
            const size_t slot = (size_t)blockIdx.x * 2 + (b0 == 0);
            if (lane == 0) sums_of(a)[slot] = make_float4(s.m, s.S, s.U, any ? 1.f : 0.f);
            uint64_t* out = keys_of(a, w.runs) + slot * top;
            for (uint32_t i = hi - lo + lane; i < top; i += 64) out[i] = 0;  // a part may hold fewer
            if (top) L.ranked(top, [&](uint32_t rank, uint64_t k) { out[rank] = k; });
        }
        __syncthreads();
    }
}

// A row that several waves hold parts of, at most kLpJoin / top of them.  Their
// keys lie in descending order.  With n = ceil(top / parts), ceil(top / n) parts'
// n-th keys that reach a bound stand for top keys that do, so that only keys that
// reach the largest such bound go to the list.
template <uint32_t K> __global__ __launch_bounds__(64) void k_logprobs_join(Logprobs a, Runs w) {
    __shared__ uint64_t listed[kLpJoin];
    const uint32_t r = blockIdx.x, lane = threadIdx.x, top = a.top;
    const uint64_t x = (uint64_t)r * w.all, first = w.with(x);
    const uint32_t parts = (uint32_t)(w.with(x + w.all - 1) - first) + 1;
    if (parts == 1) return;  // done in its wave
    auto slot = [&](uint32_t i) { return (first + i) * 2 + (i == 0); };
    Sums s;
    bool bad = false;
    for (uint32_t i = lane; i < parts; i += 64) {
        const float4 v = gld<float4>(sums_of(a) + slot(i));
        Sums o;
        o.m = v.x, o.S = v.y, o.U = v.z;
        s.add(o);
        bad |= v.w != 0.f;
    }
    List<kLpJoin> L{listed};
    if (top) {
        const uint64_t* keys = keys_of(a, w.runs);
        const uint32_t n = (top + parts - 1) / parts;
        uint64_t bound = 1;
        if (parts <= 256) {
            uint64_t nth[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; k++)
                nth[k] = lane + 64 * k < parts ? gld<uint64_t>(keys + slot(lane + 64 * k) * top + n - 1) : 0;
            bound = max(nth_of(nth, (top + n - 1) / n), (uint64_t)1);  // 0: a part of fewer keys
        }
        const uint32_t all = parts * top;
#pragma unroll 8
        for (uint32_t i0 = 0; i0 < all; i0 += 64) {
            const uint32_t i = min(i0 + lane, all - 1);
            const uint64_t k = gld<uint64_t>(keys + slot(i / top) * top + i % top);
            L.append(i0 + lane < all && k >= bound, k);
        }
    }
    finish_row<K>(a, L, r, fold(s), __any(bad));
}

static Runs lp_runs(uint32_t rows, uint32_t vocab, uint32_t top) {
    Runs w{};
    w.all = (vocab + kLpBatch - 1) / kLpBatch;
    w.total = (uint64_t)rows * w.all;
    w.runs = (uint32_t)(w.total < kLpRuns ? w.total : kLpRuns);
    // the list of k_logprobs_join holds the keys of a row's parts: one more may
    // begin in the row than runs fit it
    if (top && kLpJoin / top < w.all + 2) {
        const uint64_t most = (uint64_t)rows * (kLpJoin / top - 2);
        if (w.runs > most) w.runs = (uint32_t)most;
    }
    return w;
}

size_t logprobs_bytes(uint32_t rows, uint32_t vocab, uint32_t top) {
    const Runs w = lp_runs(rows, vocab, top);
    return (size_t)w.runs * 2 * (16 + 8 * (size_t)top);
}

template <uint32_t K> static void launch(const Logprobs& a, hipStream_t s) {
    const Runs w = lp_runs(a.rows, a.vocab, a.top);
    hipLaunchKernelGGL(k_logprobs<K>, dim3(w.runs), dim3(64), 0, s, a, w);
    if (a.rows % w.runs)  // else every run holds whole rows
        hipLaunchKernelGGL(k_logprobs_join<K>, dim3(a.rows), dim3(64), 0, s, a, w);
}

void launch_logprobs(const Logprobs& a, hipStream_t s) {
    if (a.kind == F32) launch<F32>(a, s);
    else if (a.kind == F16) launch<F16>(a, s);
    else launch<BF16>(a, s);
}

}  // namespace qh
