// Pages of the key-value cache given out and taken back on the device: the
// sequences' tables, and the slots and places of their new tokens.
#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

constexpr uint32_t kPlanBlock = 1024, kPlanWaves = kPlanBlock / 64;
// Tokens that k_page_plan itself fills in: a launch less (two plans of 64 sequences 39 us rather
// than 42), but one workgroup (48 prompts of 50,000 tokens 76 us rather than 38).
constexpr uint32_t kPlanHere = 4096;

// What sequence b asks for.
struct Ask {
    int32_t len, grown;     // tokens before and after
    uint32_t held, need;    // pages
    uint32_t claims, gives, tokens;
    bool fine;
};
__device__ __forceinline__ Ask ask_of(const PagePlan& a, uint32_t b) {
    Ask q{};
    if (b >= a.batch) return q;
    const int32_t len = gld<int32_t>(a.length + b), grow = gld<int32_t>(a.grow + b), held = gld<int32_t>(a.held + b);
    const int64_t to = (int64_t)len + grow, most = (int64_t)a.table_pages * a.page;
    q.len = q.grown = len;
    q.held = q.need = (uint32_t)held;
    q.fine = len >= 0 && len <= most && to >= 0 && to <= most && held >= 0 && (uint32_t)held <= a.table_pages;
    if (!q.fine) return q;
    q.grown = (int32_t)to;
    const uint32_t need = (uint32_t)((to + a.page - 1) / a.page);
    if (grow > 0) {
        q.tokens = (uint32_t)grow;
        q.claims = need > q.held ? need - q.held : 0;
    } else {
        q.gives = q.held > need ? q.held - need : 0;
    }
    q.need = grow > 0 ? max(need, q.held) : min(need, q.held);
    return q;
}

// Pages and tokens; neither sum passes 2^48.
struct Sum {
    uint64_t pages, tokens;
};
// Inclusive sums over the workgroup, and in all.
__device__ __forceinline__ Sum scan_block(Sum v, Sum* part, Sum& all) {
    const uint32_t lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t p = __shfl_up((unsigned long long)v.pages, o, 64), t = __shfl_up((unsigned long long)v.tokens, o, 64);
        if (lane >= (uint32_t)o) v.pages += p, v.tokens += t;
    }
    __syncthreads();
    if (lane == 63) part[wv] = v;
    __syncthreads();
    all = {0, 0};
    for (uint32_t i = 0; i < kPlanWaves; i++) {
        if (i == wv) v.pages += all.pages, v.tokens += all.tokens;
        all.pages += part[i].pages, all.tokens += part[i].tokens;
    }
    return v;
}

// What the tokens are filled in from: new lengths, and first, of all sequences; in LDS
// where they are few enough.
struct Filled {
    const int32_t *first, *length;
    bool near;
    __device__ __forceinline__ int32_t first_of(uint32_t b) const { return near ? first[b] : gld<int32_t>(first + b); }
    __device__ __forceinline__ int32_t length_of(uint32_t b) const { return near ? length[b] : gld<int32_t>(length + b); }
};

// Token i's sequence (the last whose first token is not behind it), place and slot;
// position and ancestors of a tree's nodes are its wave's (fill_tree).
__device__ __forceinline__ void fill_token(const PagePlan& a, const Filled& q, uint32_t i) {
    const bool live = a.batch && (int32_t)i < q.first_of(a.batch);
    int32_t b = -1, t = -1;
    int64_t slot = -1;
    if (live) {
        uint32_t lo = 0, hi = a.batch;  // first[lo] <= i < first[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (q.first_of(mid) <= (int32_t)i) lo = mid;
            else hi = mid;
        }
        b = (int32_t)lo;
        t = q.length_of(lo) - q.first_of(lo + 1) + (int32_t)i;
        const uint32_t page = (uint32_t)t / a.page;
        slot = (int64_t)gld<int32_t>(a.table + lo * a.stride + page) * a.page + ((uint32_t)t - page * a.page);
    }
    if (a.sequence) a.sequence[i] = b;
    if (a.slot) a.slot[i] = slot;
    if (a.position && !(a.parent && live)) a.position[i] = t;
    if (a.seen && !live) a.seen[i] = 0;
}

// A sequence's tree by a wave, a node a lane: a node's ancestors are its own bit and
// its parent's ancestors, found by doubling (six times for a path of up to 64).
__device__ __forceinline__ void fill_tree(const PagePlan& a, const Filled& q, uint32_t b) {
    const uint32_t lane = threadIdx.x & 63;
    const int32_t f = q.first_of(b), count = q.first_of(b + 1) - f;
    if (count <= 0) return;
    const int32_t context = q.length_of(b) - count;
    const int32_t parent = (int32_t)lane < count ? gld<int32_t>(a.parent + f + lane) : -1;
    uint64_t bits = 1ull << lane;
    int up = parent >= 0 && parent < (int32_t)lane ? parent : (int)lane;
#pragma unroll
    for (int i = 0; i < 6; i++) {
        bits |= __shfl((unsigned long long)bits, up, 64);
        up = __shfl(up, up, 64);
    }
    if ((int32_t)lane < count) {
        if (a.seen) a.seen[f + lane] = bits;
        if (a.position) a.position[f + lane] = context + __popcll(bits) - 1;
    }
    for (int32_t i = 64 + (int32_t)lane; i < count; i += 64) {
        if (a.seen) a.seen[f + i] = 0;
        if (a.position) a.position[f + i] = context + i;
    }
}

// One workgroup: three passes over the sequences (pages given back, the sums that
// decide who grows, pages claimed), 1,024 of them at a time with a sum over the
// workgroup, the pages themselves dealt to all threads by a search in the sums; then
// the tokens, where they are few.  Bound by latency, each pass waits for its reads: 7.5 us
// for 64 sequences with a token each, 8.4 for 48 with up to 2,100 (k_page_fill 4 more).
__global__ __launch_bounds__(kPlanBlock) void k_page_plan(PagePlan a, uint32_t fill) {
    __shared__ Sum part[kPlanWaves];
    __shared__ uint32_t upto[kPlanBlock];  // pages up to and with each sequence of the chunk
    __shared__ uint32_t from[kPlanBlock];  // the first of them in its table row
    __shared__ int32_t firsts[kPlanBlock + 1], lengths[kPlanBlock];  // of a batch of one chunk
    const uint32_t tid = threadIdx.x;
    const bool near = a.batch <= kPlanBlock;
    const int32_t stored = gld<int32_t>(a.count);
    const Ask own = ask_of(a, tid);
    auto asked_by = [&](uint32_t b) { return b < kPlanBlock ? own : ask_of(a, b); };  // tid's sequence of a chunk
    Sum all, sum;
    uint32_t gives = 0;  // at most what the table holds, below 2^31
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kPlanBlock) {
        const uint32_t mine = asked_by(b0 + tid).gives;
        if (!__syncthreads_or(mine)) continue;
        sum = scan_block({mine, 0}, part, all);
        gives += (uint32_t)all.pages;
    }
    const uint32_t count = (uint32_t)min(max(stored, 0), (int32_t)a.pages), free = min(count + gives, a.pages);
    // f(a page's number among the chunk's, its sequence in the chunk, its place in the table row)
    auto each_page = [&](uint32_t sum, uint32_t total, uint32_t begin, auto f) {
        __syncthreads();
        upto[tid] = sum;
        from[tid] = begin;
        __syncthreads();
        for (uint32_t i = tid; i < total; i += kPlanBlock) {
            uint32_t s = 0;
#pragma unroll
            for (uint32_t step = kPlanBlock / 2; step; step /= 2)
                if (upto[s + step - 1] <= i) s += step;
            f(i, s, from[s] + i - (s ? upto[s - 1] : 0));
        }
    };
    if (gives) {
        uint32_t done = 0;
        for (uint32_t b0 = 0; b0 < a.batch; b0 += kPlanBlock) {
            const Ask q = asked_by(b0 + tid);
            if (!near) sum = scan_block({q.gives, 0}, part, all);
            each_page((uint32_t)sum.pages, (uint32_t)all.pages, q.need, [&](uint32_t i, uint32_t s, uint32_t j) {
                const uint32_t to = count + (gives - 1 - done - i);
                if (to < a.pages) a.free[to] = gld<int32_t>(a.table + (size_t)(b0 + s) * a.stride + j);
            });
            done += (uint32_t)all.pages;
        }
        __syncthreads();
    }
    if (tid == 0) a.first[0] = firsts[0] = 0;
    Sum asked{0, 0}, given{0, 0};
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kPlanBlock) {
        const uint32_t b = b0 + tid;
        Ask q = asked_by(b);
        sum = all = {0, 0};
        if (__syncthreads_or(q.tokens)) {
            sum = scan_block({q.claims, q.tokens}, part, all);
            // the sums only rise, so behind the first that does not fit none does
            const bool late = q.tokens && (asked.pages + sum.pages > free || asked.tokens + sum.tokens > a.n);
            if (late) q.claims = q.tokens = 0, q.grown = q.len, q.need = q.held;
            asked.pages += all.pages, asked.tokens += all.tokens;
            if (__syncthreads_or(late)) sum = scan_block({q.claims, q.tokens}, part, all);
        }
        if (b < a.batch) {
            a.first[b + 1] = (int32_t)(given.tokens + sum.tokens);
            a.new_length[b] = q.grown;
            if (q.fine && q.need != q.held) a.held[b] = (int32_t)q.need;
            if (near) firsts[b + 1] = (int32_t)(given.tokens + sum.tokens), lengths[b] = q.grown;
        }
        const uint32_t top = free - (uint32_t)given.pages;
        if (all.pages) each_page((uint32_t)sum.pages, (uint32_t)all.pages, q.need - q.claims, [&](uint32_t i, uint32_t s, uint32_t j) {
            a.table[(size_t)(b0 + s) * a.stride + j] = gld<int32_t>(a.free + top - 1 - i);
        });
        given.pages += all.pages, given.tokens += all.tokens;
    }
    if (tid == 0) a.count[0] = (int32_t)(free - (uint32_t)given.pages);
    if (!fill) return;
    __syncthreads();
    const Filled q{near ? firsts : a.first, near ? lengths : a.new_length, near};
    for (uint32_t i = tid; i < a.n; i += kPlanBlock) fill_token(a, q, i);
    if (a.parent)
        for (uint32_t b = tid >> 6; b < a.batch; b += kPlanWaves) fill_tree(a, q, b);
}

__global__ __launch_bounds__(kBlock) void k_page_fill(PagePlan a) {
    const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
    const Filled q{a.first, a.new_length, false};
    if (i < a.n) fill_token(a, q, i);
    if (a.parent)
        for (uint32_t b = blockIdx.x * kWaves + (threadIdx.x >> 6); b < a.batch; b += gridDim.x * kWaves) fill_tree(a, q, b);
}

void launch_page_plan(const PagePlan& a, hipStream_t s) {
    const bool here = a.n <= kPlanHere;
    hipLaunchKernelGGL(k_page_plan, dim3(1), dim3(kPlanBlock), 0, s, a, here);
    if (!here) hipLaunchKernelGGL(k_page_fill, dim3((a.n + kBlock - 1) / kBlock), dim3(kBlock), 0, s, a);
}

}  // namespace qh
