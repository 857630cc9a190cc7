// Acceptance of drafted tokens: the walk down each sequence's tree by what the
// model chose, and the move of the accepted nodes' keys and values to the slots
// behind the context.
#include "qh_block.hpp"
#include "serving_device.hpp"

namespace qh {

// A workgroup per sequence, KV head and layer; the walk is short, so each does it
// for itself: lane j of a wave holds node j, and a step is one ballot.  At most 64
// steps, as a child lies behind its parent.  Accepted nodes ascend, so step s goes
// from a slot at or behind s to slot s: a batch of steps is read whole before it is
// written, and no later step's source lies in what an earlier one wrote.
// Latency: three dependent reads (bounds, nodes, pages) and the rows' own: 4.9 us for a
// tree of 16 nodes in two f32 caches, 5.8 for 48 trees in four of bf16.
constexpr uint32_t kMoveAhead = 8;  // units that a thread holds

// Moves steps 1 .. accepted - 1 of `each` units of type T in both arrays.
template <class T, class At>
__device__ __forceinline__ void move_steps(T* k, T* v, uint32_t each, uint32_t accepted, At at) {
    const uint32_t per = 2 * each, steps = max(1u, kMoveAhead * kBlock / per);  // steps of a batch
    for (uint32_t s0 = 1; s0 < accepted; s0 += steps) {
        const uint32_t units = min(steps, accepted - s0) * per;
        T x[kMoveAhead];
        size_t to[kMoveAhead];
#pragma unroll
        for (uint32_t i = 0; i < kMoveAhead; i++) {
            const uint32_t u = threadIdx.x + i * kBlock;
            if (u >= units) continue;
            size_t from;
            at(s0 + u / per, from, to[i]);
            x[i] = gld<T>((u % per < each ? k : v) + from + u % each);
            to[i] += u % each;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < kMoveAhead; i++) {
            const uint32_t u = threadIdx.x + i * kBlock;
            if (u < units) (u % per < each ? k : v)[to[i]] = x[i];
        }
    }
}

__global__ __launch_bounds__(kBlock) void k_page_accept(PageAccept a, uint32_t unit) {
    __shared__ int32_t path[kTreeMost];
    __shared__ size_t slot[kTreeMost];  // the nodes' elements
    __shared__ uint32_t steps;
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = blockIdx.x, layer = blockIdx.y, b = blockIdx.z;
    const int32_t f = gld<int32_t>(a.first + b), e = gld<int32_t>(a.first + b + 1), len = length_of(a.r, b);
    const bool rows = f >= 0 && f <= e && (uint32_t)e <= a.n;
    const uint32_t count = rows ? (uint32_t)(e - f) : 0;
    const bool ok = count > 0 && count <= kTreeMost && len >= 0 && (uint32_t)len >= count;
    const uint32_t c0 = ok ? (uint32_t)len - count : 0;
    const bool first = g == 0 && layer == 0;
    if (tid < 64) {
        const bool mine = ok && lane < count;
        const int32_t parent = mine ? gld<int32_t>(a.parent + f + lane) : -1, token = mine ? gld<int32_t>(a.token + f + lane) : 0;
        const int32_t chosen = mine ? gld<int32_t>(a.chosen + f + lane) : 0;
        const uint32_t t = c0 + lane;
        const int32_t page = mine ? gld<int32_t>(a.r.table + b * a.r.stride + t / a.c.page) : 0;
        const bool bad = !ok || __any((uint32_t)page >= a.c.count);
        slot[lane] = bad ? 0 : (size_t)page * a.c.ps + (size_t)(t % a.c.page) * a.c.ts + g * a.c.hs;
        path[lane] = -1;
        uint32_t n = 0;
        int32_t next = -1;
        if (!bad) {
            for (uint32_t node = 0;;) {
                if (lane == 0) path[n] = (int32_t)node;
                n++;
                next = __shfl(chosen, node, 64);
                const uint64_t child = __ballot(mine && lane > node && parent == (int32_t)node && token == next);
                if (!child) break;
                node = __ffsll((unsigned long long)child) - 1;
            }
        }
        if (lane == 0) {
            steps = n;
            if (first) {
                a.new_length[b] = n ? (int32_t)(c0 + n) : gld<int32_t>(a.r.length + b);
                a.accepted[b] = (int32_t)n;
                a.next[b] = next;
            }
        }
    }
    __syncthreads();
    if (first) {
        for (uint32_t i = tid; i < count; i += kBlock) a.path[f + i] = i < kTreeMost ? path[i] : -1;
        // rows of no sequence
        const int32_t f0 = b == 0 ? gld<int32_t>(a.first) : 0, last = gld<int32_t>(a.first + a.r.batch);
        for (uint32_t i = tid; i < a.n && (int32_t)i < f0; i += kBlock) a.path[i] = -1;
        if (b == a.r.batch - 1)
            for (uint32_t i = (uint32_t)max(last, 0) + tid; i < a.n; i += kBlock) a.path[i] = -1;
    }
    auto move = [&](auto one) {
        typedef decltype(one) T;
        auto& l = a.layer[layer];
        const uint32_t es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2, per = sizeof(T) / es;
        move_steps(reinterpret_cast<T*>(l.k), reinterpret_cast<T*>(l.v), a.c.dim / per, steps,
                   [&](uint32_t s, size_t& from, size_t& to) { from = slot[path[s]] / per, to = slot[s] / per; });
    };
    if (unit == 16) move(uint4());
    else if (unit == 4) move(uint32_t());
    else if (unit == 2) move(uint16_t());
    else move(uint8_t());
    if (a.c.kind == Q8_0)
        move_steps(reinterpret_cast<uint16_t*>(a.layer[layer].ks), reinterpret_cast<uint16_t*>(a.layer[layer].vs),
                   a.c.dim / 32, steps, [&](uint32_t s, size_t& from, size_t& to) { from = slot[path[s]] / 32, to = slot[s] / 32; });
}

void launch_page_accept(const PageAccept& a, hipStream_t s) {
    const uint32_t es = a.c.kind == F32 ? 4 : a.c.kind == Q8_0 ? 1 : 2;
    uintptr_t all = (a.c.dim | a.c.ps | a.c.ts | a.c.hs) * es;
    for (uint32_t i = 0; i < a.layers; i++) all |= (uintptr_t)a.layer[i].k | (uintptr_t)a.layer[i].v;
    hipLaunchKernelGGL(k_page_accept, dim3(a.c.kvheads, a.layers, a.r.batch), dim3(kBlock), 0, s, a, all % 16 ? es : 16);
}

}  // namespace qh
