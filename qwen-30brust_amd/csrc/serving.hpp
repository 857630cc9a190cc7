// Argument blocks and launch helpers of the operators on device tensors
// (paged.hip, evict.hip, prompts.hip, pool.hip, accept.hip, logprobs.hip): a
// key-value cache held in pages and the log probabilities of tokens.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "qh_format.hpp"

namespace qh {

// bfloat16, by its GGML type id; the other element types are F32, F16 and, in
// a cache, Q8_0.
constexpr uint32_t BF16 = 30;
constexpr uint32_t kPageMaxDim = 256;      // widest head of the paged operators
constexpr uint32_t kPageMaxRuns = 2048;    // most workgroups of the attention
constexpr uint32_t kMoveKeys = 64;         // keys per workgroup of k_page_move
constexpr uint32_t kLogprobMaxTop = 128;   // most alternatives of a row

// A cache: element j of head g of slot s of page p is at p * ps + s * ts +
// g * hs + j of k and v (Q8_0: int8 codes, whose f16 scales are at the same
// offset / 32 of ks and vs).
struct Pages {
    uint8_t *k, *v;
    _Float16 *ks, *vs;
    size_t ps, ts, hs;
    uint32_t kind, page, kvheads, dim;
    uint32_t count;  // pages
};

// Sequences: key t of sequence b is in slot t % page of page table[b * stride
// + t / page], t < length[b].
struct Rows {
    const int32_t* table;
    const int32_t* length;
    size_t stride;
    uint32_t batch;
    uint32_t most;  // no length is above it; at most the table row's keys
};

// [rows][heads][dim] in elements of `kind`, dim contiguous.
struct Heads {
    uint8_t* p;
    size_t row, head;
    uint32_t kind;
};

struct PageAppend {
    Pages c;
    Rows r;
    const int32_t* first;  // [batch + 1] tokens before each sequence's, or null: one each
    uint32_t from, n;      // tokens [from, n)
    Heads k, v, q, qo;     // q.p null: no queries
    uint32_t heads;
    const float *qw, *kw;  // RMSNorm weights [dim], or null
    float eps;
    const float2* rope;    // [rope_rows][dim / 2] (cos, sin), or null
    uint32_t rope_rows;
    const int32_t* pos;    // [n] rows of rope, or null: the tokens' places
};
void launch_page_append(const PageAppend& a, hipStream_t s);

// Attention of one token per sequence (paged.hip: runs of work, their slots).
struct PageAttn {
    Pages c;
    Rows r;
    Heads q, out;
    uint32_t heads;
    float scale;
    uint32_t kernel;        // 16: k_page_attn16, 32: k_page_attn32, 0: k_page_attn_any
    uint32_t groups, per;   // a KV head's query heads, `per` to a unit of work
    uint32_t units;         // of a sequence
    uint32_t runs;          // workgroups
    float* o;               // [runs][2][per][dim] weighted values of parts of units
    float2* ml;             // [runs][2][per] and their (max, sum)
    uint64_t* begin;        // [batch + 1] steps of work before each sequence, and in all
    float* score;           // [batch][heads][score_row] scores, or null
    float2* sum;            // [batch][heads] (max, sum), with score
    size_t score_row;
    const float* win;       // softmax weights so far, or null
    float* wout;            // and with this call's added
    size_t win_row, win_head, wout_row, wout_head;
};
uint32_t page_attn_kernel(const PageAttn& a);  // (q and out set)
// The units and runs of a kernel on a GPU of `cus` compute units, then the bytes
// of its workspace and its pointers.
void page_attn_plan(PageAttn& a, uint32_t kernel, uint32_t cus);
size_t page_attn_bytes(const PageAttn& a, bool weights);
void page_attn_place(PageAttn& a, void* work, bool weights);
void launch_page_attn(const PageAttn& a, hipStream_t s);

struct PageEvict {
    Pages c;
    Rows r;
    const float* w;        // weights of the keys
    size_t w_row, w_head;
    uint32_t keep, first, recent;
    const int32_t* to;     // [batch][to_stride] new pages
    size_t to_stride;
    int32_t* kept;         // [batch][kvheads][keep] kept keys, ascending; -1 behind them
    float* wout;           // [batch][kvheads][keep] their weights; 0 behind them
    int32_t* length;       // [batch] keys kept
};
void launch_page_evict(const PageEvict& a, hipStream_t s);

// Attention of several tokens per sequence, packed: sequence b's are rows
// first[b] .. first[b + 1] - 1 of q and out, the last of its keys their own.
struct PageMany {
    Pages c;
    Rows r;
    const int32_t* first;  // [batch + 1]
    uint32_t n;            // rows of q and out
    const uint64_t* seen;  // [n] bit j: the sequence's new token j is seen; null: those up to the token's own
    Heads q, out;
    uint32_t heads;
    float scale;
    // by page_many_plan
    uint32_t group, wide, runs;     // query heads of a KV head, width of the tiles, workgroups
    bool narrow;                    // products of 16 bits, else of 32
    bool one_page;                  // the rows that a wave loads at a time lie in one page
    bool q_wide, out_wide, kv_wide; // rows aligned to what is read and written at a time
    uint32_t tile_keys, run_keys;   // a tile's start and end in keys, keys of a run at least
    uint32_t page_mul, page_log;    // t / page
    float sign, c2;                 // scale * log2 e = sign * c2
    void* work;
};
void page_many_plan(PageMany& a, uint32_t cus);
size_t page_many_bytes(const PageMany& a);  // (aligned to 16)
void launch_page_many(const PageMany& a, hipStream_t s);

// Pages from and to a stack of free ones, and what the new tokens need.
struct PagePlan {
    int32_t *free, *count;  // [pages] ids, the first count[0] of them free
    uint32_t pages, page;
    int32_t* table;
    size_t stride;
    uint32_t table_pages, batch;
    int32_t* held;          // [batch] pages of each table row
    const int32_t *length, *grow;
    int32_t *new_length, *first;
    uint32_t n;             // rows of what follows
    int64_t* slot;          // page * `page` + slot, or null
    int32_t *position, *sequence;  // or null
    const int32_t* parent;  // [n], or null
    uint64_t* seen;         // [n], with parent
};
void launch_page_plan(const PagePlan& a, hipStream_t s);

// The walk down trees of drafted tokens, and the accepted ones' move.
constexpr uint32_t kTreeMost = 64;         // nodes of a tree
constexpr uint32_t kAcceptLayers = 64;     // caches of a launch
struct PageAccept {
    Pages c;  // of every cache, but the pointers
    Rows r;
    const int32_t* first;
    uint32_t n;
    const int32_t *parent, *token, *chosen;
    int32_t *new_length, *accepted, *path, *next;
    uint32_t layers;
    struct {
        uint8_t *k, *v;
        _Float16 *ks, *vs;
    } layer[kAcceptLayers];
};
void launch_page_accept(const PageAccept& a, hipStream_t s);

struct Logprobs {
    const void* x;
    uint32_t kind;
    uint32_t rows, vocab;
    size_t stride;          // elements between rows
    const int32_t* target;  // [rows], or null
    const uint8_t* valid;   // [vocab] 0 = read as f32::MIN, or null
    uint32_t top;
    float *logp, *entropy;  // [rows], or null
    int32_t* ids;           // [rows][top]
    float* alt;             // [rows][top] log probabilities of ids
    void* work;
};
size_t logprobs_bytes(uint32_t rows, uint32_t vocab, uint32_t top);
void launch_logprobs(const Logprobs& a, hipStream_t s);

}  // namespace qh
