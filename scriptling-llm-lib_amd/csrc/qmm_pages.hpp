// A cache of pages for many sequences, its batches, and the kernels' view of them.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <memory>
#include <mutex>
#include <new>
#include <vector>

#include "qmm_internal.hpp"

namespace sllm {

// Rows of a page to copy to another page, in every layer, of K and of V.
struct PageCopy {
    int src, dst, rows;
};

struct PageSeq {
    bool live = false;
    int len = 0;
    // raised whenever rows of the sequence move or end (free, truncate, a copied tail
    // page, compact): a batch begun before that is refused
    uint32_t version = 0;
    std::vector<int> pages;  // ceil(len / page_rows) page ids
};

// The pools [layer][page][kv head][row of the page][d_k], and who holds which page.
struct PageCache {
    int n_layers = 0, n_kv = 0, d_k = 0, page_rows = 0, shift = 0, n_pages = 0, type = 0, device = 0;
    char *k = nullptr, *v = nullptr;
    std::vector<int> refs;          // sequences holding each page
    std::vector<uint64_t> vacant;   // bit per page without holders
    int n_vacant = 0;
    size_t first_word = 0;          // no vacant page in words below
    std::vector<PageSeq> seqs;
    std::vector<int> spare;         // dead sequence ids, the lowest last
    std::mutex mu;

    ~PageCache();
    int elem() const { return type == SLLM_CACHE_F16 ? 2 : 4; }
    bool live(int s) const { return s >= 0 && s < (int)seqs.size() && seqs[(size_t)s].live; }
    int take();           // the lowest vacant page (n_vacant > 0), held once
    void drop(int page);  // one holder less
};

// What the kernels read of a step: one buffer at an address that stays (captured launches
// follow later steps), a header of counts and offsets (in ints) first.
enum {
    kStepRows = 0,     // query rows
    kStepItems = 1,    // pieces
    kStepRowsAt = 2,   // StepRow of every query row (offset in ints)
    kStepSeqs = 3,     // sequences
    kStepSeqsAt = 4,   // the first query row of each, and the number of all (offset)
    kStepOfAt = 5,     // every query row's sequence (offset)
    kStepHeader = 16   // then the pieces (StepItem), query rows of segments, StepRows, tables, the two above, trees
};
// The states of one query row in a segment: of the first piece and q head of the kv head, and the
// distance to those of the next piece; how many pieces the row sees.
struct StepPart {
    int first, step, pieces;
};
constexpr int kMaxParts = 3;  // segments of a row at most
struct StepRow {
    int page, slot;  // where the row's K and V go
    int pos;         // its position
    int direct;      // its one piece writes the output itself
    StepPart parts[kMaxParts];  // (pieces 0 behind the last)
    int end;         // rows of its sequence that precede it, itself included (its position + 1, but of a tree)
    int tree;        // the rows of its tree that it sees (tree_halves), -1 where these are all up to its own
    int parent;      // the query row before it (of a tree: its parent), -1 for none
};
// What a row of a tree sees: a bit for each of its sequence's rows, 16 to an element, from the element with the
// first row of the tree on (rows before the tree are seen); one more element, of zeros, behind them. `tree` counts
// elements from the step's first.
constexpr int kTreeRows = 1024;  // of a sequence's tree at most
inline int tree_halves(int base, int n) { return ((base + n - 1) >> 4) - (base >> 4) + 2; }
// A piece of a segment for a block of its query rows.
struct StepItem {
    int table;     // page ids of the positions from 0 on (offset)
    int p0, p1;    // positions
    int tok, ntok; // the block's query rows: from tok on (kItemRun), or a list there (offset)
    int slot;      // state of its first row
    int lim0;      // positions from here on are not seen by every row (of a tree: the position of its first row)
    int flags;
    int pages[8];  // the first page ids from p0 on: enough for every wave's first rows
};
enum { kItemShape = 3, kItemCausal = 4, kItemDirect = 8, kItemRun = 16, kItemTree = 32 };  // shape: kShapeRows
// The rows of a block of each shape (0: not there), as far as a wave's registers go: rows that all waves take
// together, 16 and 32 rows of each wave's own. By d_k: up to 128, the same with f16 runs that are not whole, up to 192, above.
constexpr int kShapeRows[4][3] = {{32, 64, 128}, {16, 64, 128}, {16, 64, 0}, {0, 64, 0}};
constexpr int shape_class(int d_k, bool f16) {
    return d_k > 192 ? 3 : d_k > 128 ? 2 : f16 && d_k > 64 && d_k != 128 ? 1 : 0;
}

struct PageBatch {
    std::shared_ptr<PageCache> c;
    int n_heads = 0, max_seqs = 0, max_rows = 0;
    std::vector<int> seqs;           // the current step's sequences
    std::vector<uint32_t> versions;  // as they were at its begin
    std::vector<int> counts, bases;  // their rows in the step, and before it
    int rows = 0;
    bool begun = false, captured = false;
    int *dev = nullptr;              // the step: header, rows, tables (device)
    size_t dev_cap = 0;              // bytes
    std::vector<void *> retired;
    float *qrot = nullptr;           // max_rows x n_heads x d_k, then a scale for every head
    float *part = nullptr, *ml = nullptr;  // the pieces' states, slots for every kv head
    int slots = 0;
    int items = 0;
    int rows_at = 0, seqs_at = 0, of_at = 0;  // as in the step's header
    bool wide = false;               // some block of the first shape has more than 16 rows
    int combine = 0;                 // most pieces that a row's states are merged of (0: none has several)
    // staging of a step on the host: a slot is written again when its upload is done
    static constexpr int kSlots = 4;
    char *host[kSlots] = {};
    size_t host_cap[kSlots] = {};
    hipEvent_t done[kSlots] = {};
    int slot = 0;
    std::mutex mu;

    ~PageBatch();
};

// The attention section of one layer for a batch's step.
struct PageAttnArgs {
    const float *q, *k, *v;
    float *out;
    int n_heads, n_kv, d_k, rep, shift;
    const float *q_bias, *k_bias, *v_bias;
    int qb_len, kb_len, vb_len;
    const float *q_norm, *k_norm;
    float eps;
    const float *freqs;
    int half_dim;
    float scale_log2;       // log2(e) / sqrt(d_k)
    char *pool_k, *pool_v;  // this layer
    const int *step;
    int rows_at;            // as in the step's header; -1: as that says, where the step may also have fewer rows than the launch
    float *qrot, *qscale, *part, *ml;
    int slots;
    bool wide;                  // blocks of the first shape may have more than 16 rows
    int items;                  // pieces over all kv heads; -1: as the step says
    int grid_rows, grid_items;  // the step's, or under capture what later ones may have
    int combine;                // most pieces of a row, 0 where none has several
    int type;
};

// A C entry ends with a status, whatever the host's allocations do.
template <class F>
sllm_status guarded(F f) {
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return set_error(SLLM_ERR_OOM, "out of memory");
    } catch (...) {
        return set_error(SLLM_ERR_ARG, "internal error");
    }
}
inline sllm_status on_device(int device) {
    int dev = 0;
    SLLM_HIP(hipGetDevice(&dev));
    if (dev != device) return set_error(SLLM_ERR_ARG, "the page cache is another device's");
    return SLLM_OK;
}
// Whether calls on the batch's step are accepted (under the cache's mutex and the batch's).
inline sllm_status step_stands(const PageBatch &b) {
    if (!b.begun) return set_error(SLLM_ERR_ARG, "the batch has no step: sllm_page_batch_begin first");
    for (size_t i = 0; i < b.seqs.size(); i++)
        if (b.c->seqs[(size_t)b.seqs[i]].version != b.versions[i])
            return set_error(SLLM_ERR_ARG, "a sequence of the step was freed, cut or moved: begin it again");
    return SLLM_OK;
}

sllm_status launch_page_copies(const PageCache &c, const PageCopy *jobs, size_t n, hipStream_t s);
sllm_status launch_page_attention(const PageAttnArgs &a, hipStream_t s);

// Of qmm_api.hip: the library's set-up, and whether a stream is under capture.
sllm_status library_init();
bool stream_capturing(hipStream_t s);
// The stream's workspace, grown to at least `need` bytes (not under capture).
sllm_status stream_workspace(hipStream_t s, size_t need, void **out, size_t *cap);

}  // namespace sllm

struct sllm_page_cache {
    std::shared_ptr<sllm::PageCache> c;
};
struct sllm_page_batch {
    sllm::PageBatch b;
};
