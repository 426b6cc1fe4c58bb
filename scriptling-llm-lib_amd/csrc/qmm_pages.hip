// The page cache of a batch of sequences: who holds which page (host), the copies
// (device), and the C entry points of the cache, its sequences and its batches.
//
// A page is a number of rows (positions) of every kv head of every layer; a sequence is a
// list of pages. Sequences that begin alike hold the same pages (fork); a shared page
// that one of them is to write is copied first, its filled rows alone. All decisions
// are the host's and follow from the calls' order (the lowest vacant page is taken first),
// so a program can foresee them.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstring>
#include <functional>
#include <new>
#include <string>
#include <unordered_map>

#include "qmm_pages.hpp"

struct sllm_page_cache {
    std::shared_ptr<sllm::PageCache> c;
};
struct sllm_page_batch {
    sllm::PageBatch b;
};

namespace sllm {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
constexpr int kCopyJobs = 256;  // copies per launch, by value (kernel arguments: 4 KiB)
struct CopyJobs {
    PageCopy j[kCopyJobs];
};

// One workgroup per (copy, K or V of a layer, kv head): the rows of one head of a page are one
// run of rows x d_k elements (a multiple of 16 bytes). HBM-bound: every byte is read
// and written once, four 16-byte loads of a thread in flight before its first store.
__global__ void __launch_bounds__(256) page_copy_kernel(CopyJobs jobs, char *pool_k, char *pool_v, int n_pages, int n_kv,
                                                        int page_rows, int row_bytes) {
    const PageCopy j = jobs.j[blockIdx.x];
    const int layer = blockIdx.y >> 1, head = blockIdx.z;
    char *pool = blockIdx.y & 1 ? pool_v : pool_k;
    const size_t run = (size_t)page_rows * row_bytes;
    const v4i *src = (const v4i *)(pool + (((size_t)layer * n_pages + j.src) * n_kv + head) * run);
    v4i *dst = (v4i *)(pool + (((size_t)layer * n_pages + j.dst) * n_kv + head) * run);
    const int n = j.rows * row_bytes / 16;
    for (int i = threadIdx.x; i < n; i += 4 * 256) {
        v4i v[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i + 256 * u < n) v[u] = src[i + 256 * u];
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i + 256 * u < n) dst[i + 256 * u] = v[u];
    }
}

// A small step, by value: a copy from staging memory and the event that guards it cost the host more (4 beams' fork,
// rows and end: 22.4 us with it, 20.1 with this; 53 and 30 when each is waited for).
constexpr int kSmallStep = 960;  // ints
struct SmallStep {
    int v[kSmallStep];
};
__global__ void __launch_bounds__(256) page_step_kernel(SmallStep step, int *dev, int n) {
    for (int i = threadIdx.x; i < n; i += 256) dev[i] = step.v[i];
}

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

struct DeviceFree {
    void operator()(void *p) const { (void)hipFree(p); }
};

sllm_status on_device(int device) {
    int dev = 0;
    SLLM_HIP(hipGetDevice(&dev));
    if (dev != device) return set_error(SLLM_ERR_ARG, "the page cache is another device's");
    return SLLM_OK;
}

// The pages that appending rows[i] rows to each sequence takes, and whether there are so
// many; all the memory that `append` needs is taken here.
sllm_status prepare_append(PageCache &c, const int *seqs, const int *rows, int n, std::vector<PageCopy> *copies) {
    std::unordered_map<int, int> lost;  // holders that tail pages lose to copies
    int64_t need = 0;
    for (int i = 0; i < n; i++) {
        const PageSeq &q = c.seqs[(size_t)seqs[i]];
        if (!rows[i]) continue;
        if ((int64_t)q.len + rows[i] > INT32_MAX - 512) return set_error(SLLM_ERR_SHAPE, "sequence too long");
        need += (((int64_t)q.len + rows[i] + c.page_rows - 1) >> c.shift) - (int64_t)q.pages.size();
        if (q.len & (c.page_rows - 1)) {
            int &l = lost[q.pages.back()];
            if (c.refs[(size_t)q.pages.back()] - l > 1) {
                l++;
                need++;
            }
        }
    }
    if (need > c.n_vacant)
        return set_error(SLLM_ERR_OOM, "page cache: " + std::to_string(need) + " pages needed, " +
                                           std::to_string(c.n_vacant) + " vacant");
    copies->reserve(copies->size() + lost.size() + (size_t)n);
    for (int i = 0; i < n; i++) {
        PageSeq &q = c.seqs[(size_t)seqs[i]];
        if (rows[i]) q.pages.reserve((size_t)(((int64_t)q.len + rows[i] + c.page_rows - 1) >> c.shift));
    }
    return SLLM_OK;
}

// The appending: the sequences' tables and lengths, and the copies of shared tail pages.
void append(PageCache &c, const int *seqs, const int *rows, int n, std::vector<PageCopy> *copies) noexcept {
    for (int i = 0; i < n; i++) {
        PageSeq &q = c.seqs[(size_t)seqs[i]];
        if (!rows[i]) continue;
        const int filled = q.len & (c.page_rows - 1);
        if (filled && c.refs[(size_t)q.pages.back()] > 1) {
            const int to = c.take();
            copies->push_back({q.pages.back(), to, filled});
            c.drop(q.pages.back());
            q.pages.back() = to;
            q.version++;
        }
        q.len += rows[i];
        while ((int64_t)q.pages.size() < (((int64_t)q.len + c.page_rows - 1) >> c.shift)) q.pages.push_back(c.take());
    }
}

// `append` undone, with the copies that it asked for: pages that it took are vacant again, shared tail pages held again.
void take_back(PageCache &c, const int *seqs, const int *rows, int n, std::vector<PageCopy> *copies) noexcept {
    for (int i = n - 1; i >= 0; i--) {
        if (!rows[i]) continue;
        PageSeq &q = c.seqs[(size_t)seqs[i]];
        q.len -= rows[i];
        for (; (int64_t)q.pages.size() > (((int64_t)q.len + c.page_rows - 1) >> c.shift); q.pages.pop_back()) c.drop(q.pages.back());
        if (copies->empty() || q.pages.empty() || q.pages.back() != copies->back().dst) continue;
        c.drop(q.pages.back());
        q.pages.back() = copies->back().src;
        c.refs[(size_t)q.pages.back()]++;
        q.version--;
        copies->pop_back();
    }
}

int new_seq(PageCache &c) {
    if (!c.spare.empty()) {
        const int s = c.spare.back();
        c.spare.pop_back();
        c.seqs[(size_t)s].live = true;
        return s;
    }
    c.seqs.emplace_back();
    c.spare.reserve(c.seqs.size());  // ending a sequence does not allocate
    c.seqs.back().live = true;
    return (int)c.seqs.size() - 1;
}

void end_seq(PageCache &c, int s) {
    PageSeq &q = c.seqs[(size_t)s];
    for (int p : q.pages) c.drop(p);
    q.pages.clear();
    q.len = 0;
    q.live = false;
    q.version++;
    c.spare.insert(std::lower_bound(c.spare.begin(), c.spare.end(), s, [](int a, int b) { return a > b; }), s);
}

// ---- a step's segments and pieces ----

struct Segment {
    int first;           // the sequence (of the step) whose table it reads
    int p0, p1;          // positions
    int tok0, ntok;
    int shape = 0, block = 0;  // rows of a block (shape), query rows of a block
    int slot = 0, pieces = 1, piece = 0;
    bool causal = false, lone = false;  // lone: its rows have no other segment
};

struct Plan {
    std::vector<Segment> segs;
    std::vector<int> tok;
    std::vector<std::vector<std::pair<int, int>>> parts;  // per sequence: (segment, number of its first row in it)
};

// Positions that sharing has to save each further sequence for a segment of its own: below,
// reading them once more costs less than another state to merge.
constexpr int kWorthSharing = 128;

// (The plan is made before the step's rows are appended: they change no full page before them.)
// Sequences `who` (of the step) have page p in common for p < from (their segments up to there
// are made); what follows is cut into segments: a run of pages that several hold once for all of these, and so
// on behind it, at most kMaxParts to a sequence. Sequences that go on with the same page are one group; where the run that
// all of it holds is shorter than kWorthSharing, each is on its own, also those that have more in common behind it.
void share(const PageCache &c, const int *seqs, const int *rows, const std::vector<int> &row0, std::vector<int> who, int from,
           int depth, Plan *plan) {
    auto table = [&](int i) -> const std::vector<int> & { return c.seqs[(size_t)seqs[i]].pages; };
    // full pages before the sequence's first new row: every new row sees all of them
    auto full = [&](int i) { return c.seqs[(size_t)seqs[i]].len >> c.shift; };
    auto own = [&](int i) {
        Segment s;
        s.first = i;
        s.p0 = from << c.shift;
        s.p1 = c.seqs[(size_t)seqs[i]].len + rows[i];
        s.tok0 = (int)plan->tok.size();
        s.ntok = rows[i];
        s.causal = rows[i] > 1;
        s.lone = plan->parts[(size_t)i].empty();
        for (int r = 0; r < rows[i]; r++) plan->tok.push_back(row0[(size_t)i] + r);
        plan->parts[(size_t)i].push_back({(int)plan->segs.size(), 0});
        plan->segs.push_back(s);
    };
    // by the next page; those without a further full page are on their own
    auto key = [&](int i) { return full(i) > from ? table(i)[(size_t)from] : -1; };
    std::stable_sort(who.begin(), who.end(), [&](int x, int y) { return key(x) < key(y); });
    for (size_t i = 0; i < who.size();) {
        size_t j = i + 1;
        while (j < who.size() && key(who[j]) == key(who[i])) j++;
        int to = from;
        if (key(who[i]) >= 0 && j - i > 1 && depth + 1 < kMaxParts)
            for (bool same = true; same; to += same) {
                for (size_t k = i; same && k < j; k++)
                    same = full(who[k]) > to && table(who[k])[(size_t)to] == table(who[i])[(size_t)to];
            }
        if (((to - from) << c.shift) < kWorthSharing) {
            for (; i < j; i++) own(who[i]);
            continue;
        }
        Segment s;
        s.first = who[i];
        s.p0 = from << c.shift;
        s.p1 = to << c.shift;
        s.tok0 = (int)plan->tok.size();
        std::vector<int> group(who.begin() + (long)i, who.begin() + (long)j);
        for (int k : group) {
            plan->parts[(size_t)k].push_back({(int)plan->segs.size(), (int)plan->tok.size() - s.tok0});
            for (int r = 0; r < rows[k]; r++) plan->tok.push_back(row0[(size_t)k] + r);
        }
        s.ntok = (int)plan->tok.size() - s.tok0;
        plan->segs.push_back(s);
        share(c, seqs, rows, row0, std::move(group), to, depth + 1, plan);
        i = j;
    }
}

constexpr int kPieceTile = 32;     // positions: pieces are multiples of it
constexpr int kTargetPieces = 512; // workgroups that run at a time (two per CU)
constexpr int kLeastTiles = 4;     // of a piece: one for every wave

constexpr int kSpareStates = 8192; // of a kv head, beyond what a step's rows need in one piece each

// How long a piece takes (us), roughly: a tile's bytes or products at a workgroup's share of what the card reaches
// when all workgroups run, and what a piece costs beside its tiles.
struct PieceCost {
    double tile[3];  // by shape
    double piece = 4.5, merge = 2.5;
    double state;    // one row's state of all kv heads, written and read
    PieceCost(const PageCache &c, const int *most) {
        const double read = 6.0e6, f16 = 0.4e9, f32 = 0.1e9;  // bytes, operations in a us
        for (int i = 0; i < 3; i++) {
            const double bytes = 2.0 * kPieceTile * c.d_k * c.elem(), ops = 4.0 * kPieceTile * c.d_k * most[i];
            tile[i] = std::max(i ? 0.0 : bytes / read, ops / (c.elem() == 2 ? f16 : f32)) * kTargetPieces;
        }
        state = 8.0 * (c.d_k + 2) * c.n_kv / read;
    }
};

// The segments' blocks and pieces: of a few lengths around a share of all the step's tiles the one whose pieces, taken by
// workgroups one after the other, are estimated to end first; and no more states than the batch has room for. Returns
// the number of pieces (for one kv head). (32 / 8 heads of 128; the longest share that all workgroups take at once, and
// so chosen, us: f32, 64 sequences on a prefix of 4000 85.7, 70.8; 16 on 8000 48.8, 44.9; 5 prompts of 211 rows 161,
// 147; f16, the 64 39.3, 35.2; others within 1. A step's begin with all of this takes the host 12 us for 16 sequences, 30 for
// 64 on a prefix of 4000 in pages of 64, 90 on one of 16000 in pages of 16, 105 for 256 on 4000.)
int cut(const PageCache &c, Plan *plan, int rep, int slots) {
    const int *most = kShapeRows[shape_class(c.d_k, c.type == SLLM_CACHE_F16)], n_kv = c.n_kv;
    int64_t all = 0;
    for (Segment &s : plan->segs) {
        const int64_t nv = (int64_t)s.ntok * rep;
        s.shape = nv <= most[0] ? 0 : nv <= most[1] || !most[2] ? 1 : 2;
        s.block = most[s.shape] / rep;
        all += (int64_t)((s.ntok + s.block - 1) / s.block) * ((s.p1 - s.p0 + kPieceTile - 1) / kPieceTile);
    }
    // pieces of up to `tiles` tiles: how many, and their states
    int64_t used = 0;
    auto pieces = [&](int64_t tiles) {
        int64_t items = 0;
        used = 0;
        for (Segment &s : plan->segs) {
            const int64_t n = (s.p1 - s.p0 + kPieceTile - 1) / kPieceTile;
            s.pieces = (int)((n + tiles - 1) / tiles);
            s.piece = (int)((n + s.pieces - 1) / s.pieces) * kPieceTile;
            s.pieces = (int)(((int64_t)s.p1 - s.p0 + s.piece - 1) / s.piece);
            s.slot = (int)used;
            if (!(s.lone && s.pieces == 1)) used += (int64_t)s.pieces * s.ntok * rep;
            items += (int64_t)s.pieces * ((s.ntok + s.block - 1) / s.block);
        }
        return items;
    };
    const int64_t share = std::max<int64_t>(kLeastTiles, (all * n_kv + kTargetPieces - 1) / kTargetPieces);
    const PieceCost cost(c, most);
    std::vector<double> busy;
    auto estimate = [&](int64_t items) {
        // fewer workgroups than CUs have more of the card each; a launch merges states where there are any (one row, 130
        // positions of 9 / 3 heads of 64: 10.0 us in two pieces, 7.9 in one)
        const double x = (double)items * n_kv / kTargetPieces, load = x >= 0.5 ? 1.0 : std::max(0.27, x);
        busy.assign((size_t)std::max(1, kTargetPieces / n_kv), 0.0);  // a heap, the first to be free on top
        double end = 0.0;
        for (const Segment &s : plan->segs)
            for (int i = 0; i < s.pieces; i++) {
                const int at = s.p0 + i * s.piece, n = (std::min(s.p1 - at, s.piece) + kPieceTile - 1) / kPieceTile;
                const double t = cost.piece + n * load * cost.tile[s.shape];
                for (int k = 0; k < s.ntok; k += s.block) {
                    std::pop_heap(busy.begin(), busy.end(), std::greater<>());
                    end = std::max(end, busy.back() += t);
                    std::push_heap(busy.begin(), busy.end(), std::greater<>());
                }
            }
        return end + (used ? cost.merge : 0.0) + (double)used * cost.state;
    };
    int64_t tiles = share;
    double best = -1.0;
    for (const int64_t eighths : {4, 5, 6, 7, 8, 9, 10, 11, 12, 14, 16, 20}) {
        const int64_t t = std::max<int64_t>(kLeastTiles, share * eighths / 8);
        const int64_t n = pieces(t);
        if (used > slots) continue;
        const double e = estimate(n);
        if (best >= 0.0 && e >= best) continue;
        best = e;
        tiles = t;
    }
    int64_t items = pieces(tiles);
    // (with one piece each the states fit: kMaxParts for every row)
    while (used > slots) items = pieces(tiles *= 2);
    return (int)items;
}

}  // namespace

PageCache::~PageCache() {
    if (k) (void)hipFree(k);
    if (v) (void)hipFree(v);
}

int PageCache::take() {
    while (!vacant[first_word]) first_word++;
    const int p = (int)(first_word * 64) + __builtin_ctzll(vacant[first_word]);
    vacant[first_word] &= vacant[first_word] - 1;
    n_vacant--;
    refs[(size_t)p] = 1;
    return p;
}

void PageCache::drop(int page) {
    if (--refs[(size_t)page]) return;
    vacant[(size_t)page / 64] |= 1ull << (page % 64);
    n_vacant++;
    first_word = std::min(first_word, (size_t)page / 64);
}

PageBatch::~PageBatch() {
    for (int i = 0; i < kSlots; i++) {
        if (done[i]) {
            (void)hipEventSynchronize(done[i]);
            (void)hipEventDestroy(done[i]);
        }
        if (host[i]) (void)hipHostFree(host[i]);
    }
    if (dev) (void)hipFree(dev);
    for (void *p : retired) (void)hipFree(p);
    for (float *p : {qrot, part, ml})
        if (p) (void)hipFree(p);
}

sllm_status launch_page_copies(const PageCache &c, const PageCopy *jobs, size_t n, hipStream_t s) {
    CopyJobs j;
    for (size_t at = 0; at < n; at += kCopyJobs) {
        const size_t m = std::min<size_t>(kCopyJobs, n - at);
        std::memcpy(j.j, jobs + at, m * sizeof(PageCopy));
        hipLaunchKernelGGL(page_copy_kernel, dim3((unsigned)m, (unsigned)c.n_layers * 2, (unsigned)c.n_kv), dim3(256), 0, s,
                           j, c.k, c.v, c.n_pages, c.n_kv, c.page_rows, c.d_k * c.elem());
        SLLM_HIP(hipGetLastError());
    }
    return SLLM_OK;
}

}  // namespace sllm

using namespace sllm;

extern "C" {

sllm_status sllm_page_cache_create(int n_layers, int n_kv_heads, int d_k, int page_rows, int n_pages, int type,
                                   sllm_page_cache **out) {
    if (!out) return set_error(SLLM_ERR_ARG, "null pointer");
    *out = nullptr;
    if (n_layers <= 0 || n_kv_heads <= 0 || d_k <= 0 || n_pages <= 0)
        return set_error(SLLM_ERR_ARG, "page cache dimensions must be positive");
    if (d_k % 8 != 0 || d_k > 256) return set_error(SLLM_ERR_SHAPE, "d_k must be a multiple of 8, at most 256");
    if (page_rows < 16 || page_rows > 256 || (page_rows & (page_rows - 1)))
        return set_error(SLLM_ERR_SHAPE, "page_rows must be 16, 32, 64, 128 or 256");
    if (n_layers > 32767 || n_kv_heads > 65535) return set_error(SLLM_ERR_SHAPE, "too many layers or kv heads");
    if (type != SLLM_CACHE_F32 && type != SLLM_CACHE_F16) return set_error(SLLM_ERR_ARG, "unknown cache type");
    // one side of the pool, in 64 bits: each factor is bounded above but the pages
    const double bytes_d = (double)n_layers * n_kv_heads * d_k * page_rows * n_pages * 4;
    if (bytes_d > 1e15) return set_error(SLLM_ERR_OOM, "page cache allocation failed");
    return guarded([&]() -> sllm_status {
        sllm_status st = library_init();
        if (st != SLLM_OK) return st;
        auto c = std::make_shared<PageCache>();
        c->n_layers = n_layers;
        c->n_kv = n_kv_heads;
        c->d_k = d_k;
        c->page_rows = page_rows;
        c->shift = __builtin_ctz((unsigned)page_rows);
        c->n_pages = n_pages;
        c->type = type;
        SLLM_HIP(hipGetDevice(&c->device));
        c->refs.assign((size_t)n_pages, 0);
        c->vacant.assign(((size_t)n_pages + 63) / 64, ~0ull);
        if (n_pages % 64) c->vacant.back() = (1ull << (n_pages % 64)) - 1;
        c->n_vacant = n_pages;
        const size_t bytes = (size_t)n_layers * n_pages * n_kv_heads * page_rows * d_k * c->elem();
        if (hipMalloc(&c->k, bytes) != hipSuccess || hipMalloc(&c->v, bytes) != hipSuccess) {
            (void)hipGetLastError();
            return set_error(SLLM_ERR_OOM, "page cache allocation failed");
        }
        SLLM_HIP(hipMemsetAsync(c->k, 0, bytes, nullptr));
        SLLM_HIP(hipMemsetAsync(c->v, 0, bytes, nullptr));
        SLLM_HIP(hipStreamSynchronize(nullptr));
        *out = new sllm_page_cache{std::move(c)};
        return SLLM_OK;
    });
}

void sllm_page_cache_destroy(sllm_page_cache *pc) { delete pc; }

sllm_status sllm_page_cache_data(const sllm_page_cache *pc, void **k_dev, void **v_dev) {
    if (!pc || !k_dev || !v_dev) return set_error(SLLM_ERR_ARG, "null pointer");
    *k_dev = pc->c->k;
    *v_dev = pc->c->v;
    return SLLM_OK;
}

sllm_status sllm_page_cache_vacant(const sllm_page_cache *pc, int *pages) {
    if (!pc || !pages) return set_error(SLLM_ERR_ARG, "null pointer");
    std::lock_guard<std::mutex> lk(pc->c->mu);
    *pages = pc->c->n_vacant;
    return SLLM_OK;
}

sllm_status sllm_page_seq_add(sllm_page_cache *pc, int *seq) {
    if (!pc || !seq) return set_error(SLLM_ERR_ARG, "null pointer");
    return guarded([&] {
        std::lock_guard<std::mutex> lk(pc->c->mu);
        *seq = new_seq(*pc->c);
        return SLLM_OK;
    });
}

// fork (copies null) and copy: `count` new sequences of the first `rows` rows of `seq`
static sllm_status duplicate(PageCache &c, int seq, int rows, int count, int *out, std::vector<PageCopy> *copies) {
    if (!c.live(seq)) return set_error(SLLM_ERR_ARG, "no such sequence");
    if (count < 0) return set_error(SLLM_ERR_ARG, "count must not be negative");
    if (rows < 0 || rows > c.seqs[(size_t)seq].len) return set_error(SLLM_ERR_ARG, "rows outside 0 .. the sequence's length");
    const int pages = (int)(((int64_t)rows + c.page_rows - 1) >> c.shift);
    if (copies && (int64_t)pages * count > c.n_vacant)
        return set_error(SLLM_ERR_OOM, "page cache: " + std::to_string((int64_t)pages * count) + " pages needed, " +
                                           std::to_string(c.n_vacant) + " vacant");
    if (copies) copies->reserve((size_t)pages * count);
    c.seqs.reserve(c.seqs.size() + (size_t)count);
    int made = 0;
    try {
        for (; made < count; made++) {
            const int s = new_seq(c);
            out[made] = s;
            PageSeq &q = c.seqs[(size_t)s];
            try {
                q.pages.reserve((size_t)pages);
            } catch (...) {
                end_seq(c, s);
                throw;
            }
            q.len = rows;
            for (int i = 0; i < pages; i++) {
                const int p = c.seqs[(size_t)seq].pages[(size_t)i];
                if (copies) {
                    const int to = c.take();
                    copies->push_back({p, to, std::min(c.page_rows, rows - (i << c.shift))});
                    q.pages.push_back(to);
                } else {
                    c.refs[(size_t)p]++;
                    q.pages.push_back(p);
                }
            }
        }
    } catch (...) {
        while (made > 0) end_seq(c, out[--made]);
        throw;
    }
    return SLLM_OK;
}

sllm_status sllm_page_seq_fork(sllm_page_cache *pc, int seq, int rows, int count, int *out) {
    if (!pc || (!out && count > 0)) return set_error(SLLM_ERR_ARG, "null pointer");
    return guarded([&] {
        std::lock_guard<std::mutex> lk(pc->c->mu);
        return duplicate(*pc->c, seq, rows, count, out, nullptr);
    });
}

sllm_status sllm_page_seq_copy(sllm_page_cache *pc, int seq, int rows, int count, int *out, void *stream) {
    if (!pc || (!out && count > 0)) return set_error(SLLM_ERR_ARG, "null pointer");
    return guarded([&]() -> sllm_status {
        PageCache &c = *pc->c;
        std::lock_guard<std::mutex> lk(c.mu);
        sllm_status st = on_device(c.device);
        if (st != SLLM_OK) return st;
        if (stream_capturing((hipStream_t)stream))
            return set_error(SLLM_ERR_ARG, "a page cache's sequences cannot change under capture");
        std::vector<PageCopy> copies;
        if ((st = duplicate(c, seq, rows, count, out, &copies)) != SLLM_OK) return st;
        if ((st = launch_page_copies(c, copies.data(), copies.size(), (hipStream_t)stream)) != SLLM_OK)
            for (int i = count - 1; i >= 0; i--) end_seq(c, out[i]);
        return st;
    });
}

sllm_status sllm_page_seq_extend(sllm_page_cache *pc, int seq, int rows, void *stream) {
    if (!pc) return set_error(SLLM_ERR_ARG, "null pointer");
    return guarded([&]() -> sllm_status {
        PageCache &c = *pc->c;
        std::lock_guard<std::mutex> lk(c.mu);
        if (!c.live(seq)) return set_error(SLLM_ERR_ARG, "no such sequence");
        if (rows < 0) return set_error(SLLM_ERR_ARG, "rows must not be negative");
        sllm_status st = on_device(c.device);
        if (st != SLLM_OK) return st;
        if (stream_capturing((hipStream_t)stream))
            return set_error(SLLM_ERR_ARG, "a page cache's sequences cannot change under capture");
        std::vector<PageCopy> copies;
        if ((st = prepare_append(c, &seq, &rows, 1, &copies)) != SLLM_OK) return st;
        append(c, &seq, &rows, 1, &copies);
        if ((st = launch_page_copies(c, copies.data(), copies.size(), (hipStream_t)stream)) != SLLM_OK)
            take_back(c, &seq, &rows, 1, &copies);
        return st;
    });
}

sllm_status sllm_page_seq_truncate(sllm_page_cache *pc, int seq, int rows) {
    if (!pc) return set_error(SLLM_ERR_ARG, "null pointer");
    PageCache &c = *pc->c;
    std::lock_guard<std::mutex> lk(c.mu);
    if (!c.live(seq)) return set_error(SLLM_ERR_ARG, "no such sequence");
    PageSeq &q = c.seqs[(size_t)seq];
    if (rows < 0 || rows > q.len) return set_error(SLLM_ERR_ARG, "rows outside 0 .. the sequence's length");
    if (rows < q.len) q.version++;
    q.len = rows;
    while ((int64_t)q.pages.size() > (((int64_t)rows + c.page_rows - 1) >> c.shift)) {
        c.drop(q.pages.back());
        q.pages.pop_back();
    }
    return SLLM_OK;
}

sllm_status sllm_page_seq_free(sllm_page_cache *pc, const int *seqs, int count) {
    if (!pc || (!seqs && count > 0)) return set_error(SLLM_ERR_ARG, "null pointer");
    if (count < 0) return set_error(SLLM_ERR_ARG, "count must not be negative");
    return guarded([&]() -> sllm_status {
        PageCache &c = *pc->c;
        std::lock_guard<std::mutex> lk(c.mu);
        std::vector<int> s(seqs, seqs + count);
        std::sort(s.begin(), s.end());
        for (size_t i = 0; i < s.size(); i++) {
            if (!c.live(s[i])) return set_error(SLLM_ERR_ARG, "no such sequence");
            if (i && s[i] == s[i - 1]) return set_error(SLLM_ERR_ARG, "a sequence is named twice");
        }
        for (int q : s) end_seq(c, q);
        return SLLM_OK;
    });
}

sllm_status sllm_page_seq_length(const sllm_page_cache *pc, int seq, int *rows) {
    if (!pc || !rows) return set_error(SLLM_ERR_ARG, "null pointer");
    std::lock_guard<std::mutex> lk(pc->c->mu);
    if (!pc->c->live(seq)) return set_error(SLLM_ERR_ARG, "no such sequence");
    *rows = pc->c->seqs[(size_t)seq].len;
    return SLLM_OK;
}

sllm_status sllm_page_seq_tables(const sllm_page_cache *pc, const int *seqs, int count, int *pages, int width, int *most) {
    if (!pc || (count > 0 && !seqs)) return set_error(SLLM_ERR_ARG, "null pointer");
    if (count < 0 || width < 0 || (width > 0 && count > 0 && !pages)) return set_error(SLLM_ERR_ARG, "bad table size");
    const PageCache &c = *pc->c;
    std::lock_guard<std::mutex> lk(pc->c->mu);
    int longest = 0;
    for (int i = 0; i < count; i++) {
        if (!c.live(seqs[i])) return set_error(SLLM_ERR_ARG, "no such sequence");
        longest = std::max(longest, (int)c.seqs[(size_t)seqs[i]].pages.size());
    }
    if (most) *most = longest;
    if (!width) return SLLM_OK;
    if (width < longest) return set_error(SLLM_ERR_ARG, "width is less than the longest table");
    for (int i = 0; i < count; i++) {
        const std::vector<int> &t = c.seqs[(size_t)seqs[i]].pages;
        int *row = pages + (size_t)i * width;
        std::copy(t.begin(), t.end(), row);
        std::fill(row + t.size(), row + width, -1);
    }
    return SLLM_OK;
}

sllm_status sllm_page_cache_compact(sllm_page_cache *pc, int *used, void *stream) {
    if (!pc) return set_error(SLLM_ERR_ARG, "null pointer");
    return guarded([&]() -> sllm_status {
        PageCache &c = *pc->c;
        std::lock_guard<std::mutex> lk(c.mu);
        sllm_status st = on_device(c.device);
        if (st != SLLM_OK) return st;
        if (stream_capturing((hipStream_t)stream))
            return set_error(SLLM_ERR_ARG, "a page cache's sequences cannot change under capture");
        const int n = c.n_pages - c.n_vacant;
        std::vector<PageCopy> copies;
        std::unordered_map<int, int> to;
        int gap = 0;
        for (int p = n; p < c.n_pages; p++) {
            if (!c.refs[(size_t)p]) continue;
            while (c.refs[(size_t)gap]) gap++;
            copies.push_back({p, gap, c.page_rows});
            to[p] = gap++;
        }
        if ((st = launch_page_copies(c, copies.data(), copies.size(), (hipStream_t)stream)) != SLLM_OK) return st;
        for (const PageCopy &j : copies) {
            c.refs[(size_t)j.dst] = c.refs[(size_t)j.src];
            c.refs[(size_t)j.src] = 0;
            c.vacant[(size_t)j.dst / 64] &= ~(1ull << (j.dst % 64));
            c.vacant[(size_t)j.src / 64] |= 1ull << (j.src % 64);
        }
        c.first_word = 0;
        if (!copies.empty())
            for (PageSeq &q : c.seqs) {
                bool moved = false;
                for (int &p : q.pages) {
                    if (p < n) continue;
                    p = to[p];
                    moved = true;
                }
                q.version += moved;
            }
        if (used) *used = n;
        return SLLM_OK;
    });
}

sllm_status sllm_page_batch_create(sllm_page_cache *pc, int n_heads, int max_seqs, int max_rows, sllm_page_batch **out) {
    if (!out) return set_error(SLLM_ERR_ARG, "null pointer");
    *out = nullptr;
    if (!pc) return set_error(SLLM_ERR_ARG, "null pointer");
    if (max_seqs <= 0 || max_rows <= 0) return set_error(SLLM_ERR_ARG, "max_seqs and max_rows must be positive");
    const PageCache &c = *pc->c;
    if (n_heads <= 0 || n_heads % c.n_kv != 0 || n_heads / c.n_kv > 8)
        return set_error(SLLM_ERR_SHAPE, "n_heads must be a multiple of n_kv_heads, at most 8 times it");
    // the kernels address a row's q, output and states with 32 bits
    if ((int64_t)max_rows * n_heads * c.d_k > (1 << 28))
        return set_error(SLLM_ERR_SHAPE, "max_rows x n_heads x d_k must be at most 2^28");
    // a launch has fewer than 2^32 threads: the merge 256 for every row and head
    if ((int64_t)max_rows * n_heads >= 1 << 24) return set_error(SLLM_ERR_SHAPE, "max_rows x n_heads must be below 2^24");
    return guarded([&]() -> sllm_status {
        sllm_status st = on_device(c.device);
        if (st != SLLM_OK) return st;
        auto b = std::make_unique<sllm_page_batch>();
        b->b.c = pc->c;
        b->b.n_heads = n_heads;
        b->b.max_seqs = max_seqs;
        b->b.max_rows = max_rows;
        b->b.seqs.reserve((size_t)max_seqs);
        b->b.versions.reserve((size_t)max_seqs);
        const int rep = n_heads / c.n_kv;
        b->b.slots = (kMaxParts + 1) * max_rows * rep + kSpareStates;
        const size_t states = (size_t)b->b.slots * c.n_kv;
        if (hipMalloc(&b->b.qrot, (size_t)max_rows * n_heads * (c.d_k + 1) * sizeof(float)) != hipSuccess ||
            hipMalloc(&b->b.part, states * c.d_k * sizeof(float)) != hipSuccess ||
            hipMalloc(&b->b.ml, states * 2 * sizeof(float)) != hipSuccess) {
            (void)hipGetLastError();
            return set_error(SLLM_ERR_OOM, "page batch allocation failed");
        }
        for (hipEvent_t &e : b->b.done) SLLM_HIP(hipEventCreateWithFlags(&e, hipEventDisableTiming));
        *out = b.release();
        return SLLM_OK;
    });
}

void sllm_page_batch_destroy(sllm_page_batch *batch) { delete batch; }

sllm_status sllm_page_batch_begin(sllm_page_batch *batch, const int *seqs, const int *rows, int count, void *stream) {
    if (!batch || (count > 0 && (!seqs || !rows))) return set_error(SLLM_ERR_ARG, "null pointer");
    PageBatch &b = batch->b;
    if (count < 0 || count > b.max_seqs) return set_error(SLLM_ERR_ARG, "count outside 0 .. max_seqs");
    hipStream_t s = (hipStream_t)stream;
    return guarded([&]() -> sllm_status {
        std::lock_guard<std::mutex> lb(b.mu);
        PageCache &c = *b.c;
        std::lock_guard<std::mutex> lk(c.mu);
        int64_t total = 0, pages = 0;
        std::vector<int> sorted(seqs, seqs + count);
        std::sort(sorted.begin(), sorted.end());
        for (int i = 0; i < count; i++) {
            if (!c.live(seqs[i])) return set_error(SLLM_ERR_ARG, "no such sequence");
            if (i && sorted[(size_t)i] == sorted[(size_t)i - 1]) return set_error(SLLM_ERR_ARG, "a sequence is named twice");
            if (rows[i] < 0) return set_error(SLLM_ERR_ARG, "rows must not be negative");
            total += rows[i];
            pages += ((int64_t)c.seqs[(size_t)seqs[i]].len + rows[i] + c.page_rows - 1) >> c.shift;
        }
        if (total > b.max_rows) return set_error(SLLM_ERR_SHAPE, "more rows than max_rows");
        // room for the step on the device and in the next staging slot: header, rows, rows of segments,
        // pieces, tables
        const int64_t most_segs = 2 * (int64_t)count;
        const int64_t most_items = most_segs + kMaxParts * total + 3 * kTargetPieces;
        const int64_t ints = kStepHeader + total * (int64_t)(sizeof(StepRow) / 4 + kMaxParts) + 16 * most_items + pages + 32;
        if (ints > INT32_MAX) return set_error(SLLM_ERR_SHAPE, "the step has too many rows and pages (offsets of 32 bits)");
        const size_t bytes = (size_t)ints * sizeof(int);
        sllm_status st = on_device(c.device);
        if (st != SLLM_OK) return st;
        if (stream_capturing(s)) return set_error(SLLM_ERR_ARG, "a batch's step cannot begin under capture");
        std::vector<PageCopy> copies;
        if ((st = prepare_append(c, seqs, rows, count, &copies)) != SLLM_OK) return st;
        Plan plan;
        plan.parts.resize((size_t)count);
        plan.tok.reserve((size_t)total * kMaxParts);
        std::vector<int> row0((size_t)count), who;
        int r0 = 0;
        for (int i = 0; i < count; i++) {
            row0[(size_t)i] = r0;
            r0 += rows[i];
            if (rows[i]) who.push_back(i);
        }
        const int64_t rep = b.n_heads / c.n_kv;
        share(c, seqs, rows, row0, std::move(who), 0, 0, &plan);
        const int n_items = cut(c, &plan, (int)rep, b.slots);
        std::vector<int> table((size_t)count, -1);  // of the sequences that segments read
        // (a larger buffer takes the old one's place once nothing refuses the step any more: until then the step before
        // it is the batch's, and the old buffer holds it)
        std::unique_ptr<void, DeviceFree> grown;
        size_t dev_cap = b.dev_cap;
        if (dev_cap < bytes) {
            if (b.captured)
                return set_error(SLLM_ERR_SHAPE, "the step has more pages than the batch held when it was captured");
            b.retired.reserve(b.retired.size() + 1);
            void *p = nullptr;
            dev_cap = 2 * bytes + 65536;
            if (hipMalloc(&p, dev_cap) != hipSuccess) {
                (void)hipGetLastError();
                return set_error(SLLM_ERR_OOM, "page batch allocation failed");
            }
            grown.reset(p);
        }
        const int slot = b.slot;
        SLLM_HIP(hipEventSynchronize(b.done[slot]));
        if (b.host_cap[slot] < bytes) {
            if (b.host[slot]) (void)hipHostFree(b.host[slot]);
            b.host[slot] = nullptr;
            b.host_cap[slot] = 0;
            if (hipHostMalloc((void **)&b.host[slot], dev_cap, hipHostMallocDefault) != hipSuccess) {
                (void)hipGetLastError();
                return set_error(SLLM_ERR_OOM, "page batch staging allocation failed");
            }
            b.host_cap[slot] = dev_cap;
        }
        // nothing below allocates memory or refuses the step
        append(c, seqs, rows, count, &copies);
        if ((st = launch_page_copies(c, copies.data(), copies.size(), s)) != SLLM_OK) {
            take_back(c, seqs, rows, count, &copies);
            return st;
        }
        b.begun = false;
        if (grown) {
            if (b.dev) b.retired.push_back(b.dev);
            b.dev = (int *)grown.release();
            b.dev_cap = dev_cap;
        }
        int *h = (int *)b.host[slot];
        int at = kStepHeader;
        auto place = [&](int64_t ints) {
            const int was = at;
            at += (int)((ints + 3) & ~(int64_t)3);
            return was;
        };
        h[kStepRows] = (int)total;
        h[kStepItems] = n_items;
        StepItem *hi = (StepItem *)(h + place(16 * (int64_t)n_items));
        const int tok_at = place((int64_t)plan.tok.size());
        h[kStepRowsAt] = place((int64_t)(sizeof(StepRow) / 4) * total);
        StepRow *hr = (StepRow *)(h + h[kStepRowsAt]);
        b.combine = 0;
        for (int i = 0; i < count; i++) {
            const PageSeq &q = c.seqs[(size_t)seqs[i]];
            const auto &mine = plan.parts[(size_t)i];
            int pieces = 0;
            for (const auto &m : mine) pieces += plan.segs[(size_t)m.first].pieces;
            if (pieces > 1) b.combine = std::max(b.combine, pieces);
            for (int r = 0; r < rows[i]; r++) {
                const int pos = q.len - rows[i] + r;
                StepRow x = {q.pages[(size_t)(pos >> c.shift)], pos & (c.page_rows - 1), pos, pieces == 1, {}};
                for (size_t k = 0; k < mine.size(); k++) {
                    const Segment &s = plan.segs[(size_t)mine[k].first];
                    x.parts[k] = {s.slot + (mine[k].second + r) * (int)rep, s.ntok * (int)rep,
                                  std::min(s.pieces, (pos - s.p0) / s.piece + 1), 0};
                }
                *hr++ = x;
            }
        }
        std::copy(plan.tok.begin(), plan.tok.end(), h + tok_at);
        for (const Segment &s : plan.segs) {
            int &t = table[(size_t)s.first];
            if (t < 0) {
                const std::vector<int> &pg = c.seqs[(size_t)seqs[s.first]].pages;
                t = at;
                at += (int)pg.size();
                std::copy(pg.begin(), pg.end(), h + t);
            }
            const bool direct = s.lone && s.pieces == 1;
            for (int i = 0; i < s.pieces; i++)
                for (int k = 0; k < s.ntok; k += s.block) {
                    StepItem x;
                    x.table = t;
                    x.p0 = s.p0 + i * s.piece;
                    x.p1 = x.p0 + std::min(s.p1 - x.p0, s.piece);
                    x.ntok = std::min(s.block, s.ntok - k);
                    const int *tk = plan.tok.data() + s.tok0 + k;
                    bool run = true;
                    for (int u = 1; u < x.ntok; u++) run &= tk[u] == tk[0] + u;
                    x.tok = run ? tk[0] : tok_at + s.tok0 + k;
                    x.slot = s.slot + (i * s.ntok + k) * (int)rep;
                    // a sequence's own rows: row k of n sees n - 1 - k positions less than the last
                    x.lim0 = s.causal ? std::min(x.p1, s.p1 - (s.ntok - 1 - k)) : x.p1;
                    x.flags = s.shape | (s.causal ? kItemCausal : 0) | (direct ? kItemDirect : 0) | (run ? kItemRun : 0);
                    const std::vector<int> &pg = c.seqs[(size_t)seqs[s.first]].pages;
                    for (int u = 0; u < 8; u++) {
                        const size_t at_page = (size_t)(x.p0 >> c.shift) + (size_t)u;
                        x.pages[u] = at_page < pg.size() ? pg[at_page] : 0;
                    }
                    *hi++ = x;
                }
        }
        b.items = n_items;
        b.wide = false;
        for (const Segment &s : plan.segs) b.wide |= s.shape == 0 && s.ntok * rep > 16;
        b.seqs.assign(seqs, seqs + count);
        b.versions.resize((size_t)count);
        for (int i = 0; i < count; i++) b.versions[(size_t)i] = c.seqs[(size_t)seqs[i]].version;
        b.rows = (int)total;
        st = [&]() -> sllm_status {
            if (at <= kSmallStep) {
                SmallStep small;
                std::memcpy(small.v, h, (size_t)at * sizeof(int));
                hipLaunchKernelGGL(page_step_kernel, dim3(1), dim3(256), 0, s, small, b.dev, at);
                SLLM_HIP(hipGetLastError());
            } else {
                SLLM_HIP(hipMemcpyAsync(b.dev, h, (size_t)at * sizeof(int), hipMemcpyHostToDevice, s));
                b.slot = (slot + 1) % PageBatch::kSlots;
                SLLM_HIP(hipEventRecord(b.done[slot], s));
            }
            return SLLM_OK;
        }();
        if (st != SLLM_OK) take_back(c, seqs, rows, count, &copies);
        b.begun = st == SLLM_OK;
        return st;
    });
}

sllm_status sllm_page_attention_dev(sllm_page_batch *batch, int layer, const sllm_attn_params *p, const float *q,
                                    const float *k, const float *v, float *out, void *stream) {
    if (!batch || !p || !q || !k || !v || !out) return set_error(SLLM_ERR_ARG, "null pointer");
    PageBatch &b = batch->b;
    std::lock_guard<std::mutex> lb(b.mu);
    PageCache &c = *b.c;
    if (layer < 0 || layer >= c.n_layers) return set_error(SLLM_ERR_ARG, "layer out of range");
    if (p->n_heads != b.n_heads || p->n_kv_heads != c.n_kv || p->d_k != c.d_k)
        return set_error(SLLM_ERR_ARG, "n_heads / n_kv_heads / d_k differ from the batch's");
    if (p->rope_half_dim < 0 || 2 * p->rope_half_dim > p->d_k)
        return set_error(SLLM_ERR_ARG, "rope_half_dim outside 0 .. d_k / 2");
    if (p->rope_half_dim > 0 && !p->rope_freqs) return set_error(SLLM_ERR_ARG, "null rope_freqs");
    if (p->q_bias_len < 0 || p->k_bias_len < 0 || p->v_bias_len < 0)
        return set_error(SLLM_ERR_ARG, "negative bias length");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15)
        return set_error(SLLM_ERR_ARG, "q, k, v and out must be 16-byte aligned");
    {
        std::lock_guard<std::mutex> lk(c.mu);
        if (!b.begun) return set_error(SLLM_ERR_ARG, "the batch has no step: sllm_page_batch_begin first");
        for (size_t i = 0; i < b.seqs.size(); i++)
            if (c.seqs[(size_t)b.seqs[i]].version != b.versions[i])
                return set_error(SLLM_ERR_ARG, "a sequence of the step was freed, cut or moved: begin it again");
    }
    sllm_status st = on_device(c.device);
    if (st != SLLM_OK) return st;
    hipStream_t s = (hipStream_t)stream;
    const bool capture = stream_capturing(s);
    if (!b.rows && !capture) return SLLM_OK;
    PageAttnArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.n_heads = b.n_heads;
    a.n_kv = c.n_kv;
    a.d_k = c.d_k;
    a.rep = b.n_heads / c.n_kv;
    a.shift = c.shift;
    a.n_pages = c.n_pages;
    a.q_bias = p->q_bias_len ? p->q_bias : nullptr;
    a.k_bias = p->k_bias_len ? p->k_bias : nullptr;
    a.v_bias = p->v_bias_len ? p->v_bias : nullptr;
    a.qb_len = p->q_bias_len;
    a.kb_len = p->k_bias_len;
    a.vb_len = p->v_bias_len;
    a.q_norm = p->q_norm_w;
    a.k_norm = p->k_norm_w;
    a.eps = p->norm_eps;
    a.freqs = p->rope_freqs;
    a.half_dim = p->rope_half_dim;
    a.scale_log2 = (float)(1.4426950408889634 / __builtin_sqrt((double)c.d_k));
    const size_t loff = (size_t)layer * c.n_pages * c.n_kv * c.page_rows * c.d_k * c.elem();
    a.pool_k = c.k + loff;
    a.pool_v = c.v + loff;
    a.step = b.dev;
    a.qrot = b.qrot;
    a.qscale = b.qrot + (size_t)b.max_rows * b.n_heads * c.d_k;
    a.part = b.part;
    a.ml = b.ml;
    a.slots = b.slots;
    // a captured launch serves later steps of the batch too
    a.grid_rows = capture ? b.max_rows : b.rows;
    a.wide = capture || b.wide;
    a.items = capture ? -1 : b.items * c.n_kv;
    // (workgroups take pieces one after the other where there are more than those of a launch of 2^31 threads)
    a.grid_items = capture ? 2 * kTargetPieces : std::min(b.items * c.n_kv, 1 << 23);
    a.combine = capture ? INT32_MAX : b.combine;
    a.type = c.type;
    b.captured |= capture;
    return launch_page_attention(a, s);
}

}  // extern "C"
