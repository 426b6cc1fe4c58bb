// Steps of trees on the CPU (qmm_pages.hip): what the kernels are given for each row, tile by tile as they read it, against
// the parents; and what a refused step leaves behind. Compiled against hip/hip_runtime.h beside this file.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <string>

#include <sys/mman.h>

#include "qmm_pages.hip"

static std::string error;
static PageAttnArgs last;

namespace sllm {
sllm_status set_error(sllm_status st, const std::string &msg) {
    error = msg;
    return st;
}
sllm_status hip_error(hipError_t, const char *what) {
    error = what;
    return SLLM_ERR_DEVICE;
}
sllm_status library_init() { return SLLM_OK; }
bool stream_capturing(hipStream_t) { return stub::capture; }
sllm_status stream_workspace(hipStream_t, size_t, void **, size_t *) { return SLLM_ERR_ARG; }
sllm_status launch_page_attention(const PageAttnArgs &a, hipStream_t) {
    last = a;
    return SLLM_OK;
}
}  // namespace sllm

#define CHECK(x)                                                                               \
    do {                                                                                       \
        if (!(x)) {                                                                            \
            std::fprintf(stderr, "%s:%d: %s (%s)\n", __FILE__, __LINE__, #x, error.c_str()); \
            std::exit(1);                                                                      \
        }                                                                                      \
    } while (0)

static unsigned seed = 7;
static int below(int n) { return (int)((seed = seed * 1664525u + 1013904223u) >> 8) % n; }

static void attend(sllm_page_batch *b, int heads, int kv, int dk) {
    alignas(16) static float x[4];
    sllm_attn_params p{};
    p.n_heads = heads;
    p.n_kv_heads = kv;
    p.d_k = dk;
    CHECK(sllm_page_attention_dev(b, 0, &p, x, x, x, x, nullptr) == SLLM_OK);
}

static std::vector<int> draw_tree(int n, int kind) {
    std::vector<int> p((size_t)n);
    for (int r = 0; r < n; r++)
        p[(size_t)r] = kind == 0 ? r - 1 : kind == 1 ? (r - 1) / 2 - (r == 0) : kind == 2 ? below(r + 1) - 1 : r < 3 ? -1 : r - 3;
    return p;
}

static void steps() {
    for (int kind = 0; kind < 80; kind++) {
        const int kv = 1 + below(4), rep = 1 + below(8), dk = 8 * (1 + below(32)), page = 16 << below(5), type = below(2);
        sllm_page_cache *c;
        sllm_page_batch *b;
        CHECK(sllm_page_cache_create(1, kv, dk, page, 5000, type, &c) == SLLM_OK);
        CHECK(sllm_page_batch_create(c, kv * rep, 20, 2600, &b) == SLLM_OK);
        int base;
        CHECK(sllm_page_seq_add(c, &base) == SLLM_OK && sllm_page_seq_extend(c, base, below(3) ? below(2500) : 0, nullptr) == SLLM_OK);
        std::vector<int> seqs(1 + (size_t)below(12)), rows, parents;
        int len;
        CHECK(sllm_page_seq_length(c, base, &len) == SLLM_OK);
        CHECK(sllm_page_seq_fork(c, base, len, (int)seqs.size(), seqs.data()) == SLLM_OK);
        std::vector<std::vector<int>> trees;
        for (size_t i = 0; i < seqs.size(); i++) {
            CHECK(sllm_page_seq_extend(c, seqs[i], below(3) ? below(50) : below(400), nullptr) == SLLM_OK);
            rows.push_back(below(5) ? below(40) : below(i ? 130 : 1025));
            trees.push_back(draw_tree(rows.back(), below(4)));
            parents.insert(parents.end(), trees.back().begin(), trees.back().end());
        }
        CHECK(sllm_page_batch_begin_tree(b, seqs.data(), rows.data(), (int)seqs.size(), parents.data(), nullptr) == SLLM_OK);
        int total = 0;
        for (int n : rows) total += n;
        if (total) attend(b, kv * rep, kv, dk);
        const int *step = total ? last.step : b->b.dev;
        CHECK(step[kStepRows] == total && step[kStepSeqs] == (int)seqs.size());
        const StepRow *sr = (const StepRow *)(step + step[kStepRowsAt]);
        const StepItem *items = (const StepItem *)(step + kStepHeader);
        const int *first = step + step[kStepSeqsAt], *of = step + step[kStepOfAt];
        std::vector<std::set<int>> sees((size_t)total), seen((size_t)total);
        for (size_t i = 0, r0 = 0; i < seqs.size(); r0 += (size_t)rows[i], i++) {
            CHECK(first[i] == (int)r0 && first[i + 1] == (int)r0 + rows[i]);
            CHECK(sllm_page_seq_length(c, seqs[i], &len) == SLLM_OK);
            const int b0 = len - rows[i];
            for (int r = 0; r < rows[i]; r++) {
                auto &s = sees[r0 + (size_t)r];
                const int up = trees[i][(size_t)r];
                if (up < 0) {
                    for (int x = 0; x < b0; x++) s.insert(x);
                } else {
                    s = sees[r0 + (size_t)up];
                }
                const StepRow &w = sr[r0 + (size_t)r];
                CHECK(of[r0 + (size_t)r] == (int)i && w.parent == (up < 0 ? -1 : (int)r0 + up));
                // its position is the number of rows that it sees before itself; its place the row's own
                CHECK(w.pos == (int)s.size() && w.end == b0 + r + 1 && w.slot == (b0 + r) % page);
                s.insert(b0 + r);
            }
        }
        for (int i = 0; i < step[kStepItems]; i++) {
            const StepItem &x = items[i];
            const bool tree = x.flags & kItemTree;
            CHECK(!(tree && x.flags & kItemCausal));
            for (int t = 0; t < x.ntok; t++) {
                const int r = x.flags & kItemRun ? x.tok + t : step[x.tok + t];
                const StepRow &w = sr[r];
                if (tree) CHECK(w.tree >= 0 && x.lim0 == w.end - 1 - (r - first[of[r]]));
                const int lim = tree ? w.tree : x.flags & kItemCausal ? std::min(x.p1, w.end) : x.p1;
                const int halves = tree ? tree_halves(x.lim0, first[of[r] + 1] - first[of[r]]) : 0;
                for (int tp : {16, 32})
                    for (int p = x.p0; p < x.p1; p += tp)
                        for (int h = 0; h < tp / 16; h++)
                            for (int k = 0; k < 16; k++) {
                                bool in = true;
                                if (p + tp > x.lim0) {
                                    const int half = (p >> 4) - (x.lim0 >> 4) + h;
                                    if (!tree) in = p + 16 * h + k < lim;
                                    else if (half >= 0) {
                                        CHECK(half < halves);
                                        in = ((const uint16_t *)step)[lim + half] >> k & 1;
                                    }
                                }
                                if (in && tp == 16) CHECK(seen[(size_t)r].insert(p + k).second);
                                if (in && tp == 32) CHECK(seen[(size_t)r].count(p + 16 * h + k));
                            }
            }
        }
        for (int r = 0; r < total; r++) {
            CHECK(seen[(size_t)r] == sees[(size_t)r]);
            // the merge takes as many pieces as may hold positions that the row sees
            int pieces = 0, have = 0;
            for (const StepPart &p : sr[r].parts) pieces += p.pieces;
            for (int i = 0; i < step[kStepItems]; i++) {
                const StepItem &x = items[i];
                for (int t = 0; t < x.ntok; t++)
                    have += (x.flags & kItemRun ? x.tok + t : step[x.tok + t]) == r && x.p0 < sr[r].end;
            }
            CHECK(pieces == have);
        }
        sllm_page_batch_destroy(b);
        sllm_page_cache_destroy(c);
    }
}

// Wrong parents, a tree that is too large, a step without room: refused, and the sequences are as they were.
static void refused() {
    sllm_page_cache *c;
    sllm_page_batch *b;
    CHECK(sllm_page_cache_create(1, 1, 64, 16, 100, 0, &c) == SLLM_OK);
    CHECK(sllm_page_batch_create(c, 2, 4, 1600, &b) == SLLM_OK);
    int s[2];
    CHECK(sllm_page_seq_add(c, &s[0]) == SLLM_OK && sllm_page_seq_add(c, &s[1]) == SLLM_OK);
    CHECK(sllm_page_seq_extend(c, s[0], 20, nullptr) == SLLM_OK);
    auto begin = [&](std::vector<int> rows, const std::vector<int> &parents) {
        return sllm_page_batch_begin_tree(b, s, rows.data(), (int)rows.size(), parents.data(), nullptr);
    };
    auto same = [&] {
        int n, m, v;
        CHECK(sllm_page_seq_length(c, s[0], &n) == SLLM_OK && sllm_page_seq_length(c, s[1], &m) == SLLM_OK);
        CHECK(sllm_page_cache_vacant(c, &v) == SLLM_OK);
        return n == 20 && m == 0 && v == 98;
    };
    CHECK(begin({3}, {-1, 0, 2}) == SLLM_ERR_ARG && same());  // its own parent
    CHECK(begin({3}, {-1, 2, 0}) == SLLM_ERR_ARG && same());  // a later one
    CHECK(begin({3}, {-2, 0, 0}) == SLLM_ERR_ARG && same());
    CHECK(begin({1, 2}, {-1, 0, 0}) == SLLM_ERR_ARG && same());  // (numbered within the sequence: its first cannot follow)
    // parents with nothing readable behind them: as many as the rows say in all, but not in each sequence
    char *guard = (char *)mmap(nullptr, 8192, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    CHECK(guard != MAP_FAILED && mprotect(guard + 4096, 4096, PROT_NONE) == 0);
    int *last_two = (int *)(guard + 4096) - 2;
    last_two[0] = -1;
    last_two[1] = 0;
    const int signs[2] = {5, -3}, many[2] = {2, 1599};
    CHECK(sllm_page_batch_begin_tree(b, s, signs, 2, last_two, nullptr) == SLLM_ERR_ARG && same());
    CHECK(sllm_page_batch_begin_tree(b, s, many, 2, last_two, nullptr) == SLLM_ERR_SHAPE && same());
    munmap(guard, 8192);
    const int two = 2, none = 0;
    CHECK(sllm_page_batch_begin_tree(b, s, &two, 1, nullptr, nullptr) == SLLM_ERR_ARG && same());
    CHECK(sllm_page_batch_begin_tree(b, s, &none, 1, nullptr, nullptr) == SLLM_OK && same());
    std::vector<int> wide(1025, 0), chain(1500);
    wide[0] = -1;
    CHECK(begin({1025}, wide) == SLLM_ERR_SHAPE && same());
    for (int r = 0; r < 1500; r++) chain[(size_t)r] = r - 1;
    CHECK(begin({1500}, chain) == SLLM_OK);  // (no tree: as many rows as a batch takes)
    CHECK(sllm_page_seq_truncate(c, s[0], 20) == SLLM_OK && same());
    wide.resize(1024);
    CHECK(begin({1024}, wide) == SLLM_OK);
    CHECK(sllm_page_seq_truncate(c, s[0], 20) == SLLM_OK && same());
    // an upload that fails takes the rows back
    stub::launches_left = stub::memcpys_left = 0;
    CHECK(begin({5}, {-1, 0, 0, 1, 1}) == SLLM_ERR_DEVICE && same());
    stub::launches_left = stub::memcpys_left = -1;
    CHECK(begin({5, 0}, {-1, 0, 0, 1, 1}) == SLLM_OK);
    sllm_page_batch_destroy(b);
    sllm_page_cache_destroy(c);
}

int main(int, char **argv) {
    const std::string what = argv[1];
    if (what == "steps") steps();
    else if (what == "refused") refused();
    else return 2;
    return 0;
}
