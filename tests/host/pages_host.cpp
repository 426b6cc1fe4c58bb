// The page cache's host code (qmm_pages.hip) on the CPU: what its steps ask of the kernels, and what a refused or failed
// call leaves behind. Compiled against hip/hip_runtime.h beside this file; the first argument names the test.
#include <cstdio>
#include <cstdlib>
#include <string>

#include "qmm_pages.hip"

static std::string error;

// The library's allocations fail one after the other while `news_left` counts down to 0.
static long news_left = -1;
static bool news_failed;
void *operator new(size_t n) {
    if (news_left == 0) {
        news_failed = true;
        throw std::bad_alloc();
    }
    if (news_left > 0) news_left--;
    if (void *p = std::malloc(n ? n : 1)) return p;
    throw std::bad_alloc();
}
void *operator new(size_t n, const std::nothrow_t &) noexcept { return std::malloc(n ? n : 1); }
void operator delete(void *p) noexcept { std::free(p); }
void operator delete(void *p, size_t) noexcept { std::free(p); }

static PageAttnArgs last;
static int launches;

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
    launches++;
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

struct Cache {
    sllm_page_cache *c = nullptr;
    int kv, dk;
    Cache(int layers, int kv, int dk, int page, int pages, int type) : kv(kv), dk(dk) {
        CHECK(sllm_page_cache_create(layers, kv, dk, page, pages, type, &c) == SLLM_OK);
    }
    ~Cache() { sllm_page_cache_destroy(c); }
    int add(int rows = 0) {
        int s;
        CHECK(sllm_page_seq_add(c, &s) == SLLM_OK && sllm_page_seq_extend(c, s, rows, nullptr) == SLLM_OK);
        return s;
    }
    std::vector<int> fork(int s, int rows, int n) {
        std::vector<int> out((size_t)n);
        CHECK(sllm_page_seq_fork(c, s, rows, n, out.data()) == SLLM_OK);
        return out;
    }
    int length(int s) const {
        int n;
        CHECK(sllm_page_seq_length(c, s, &n) == SLLM_OK);
        return n;
    }
    int vacant() const {
        int n;
        CHECK(sllm_page_cache_vacant(c, &n) == SLLM_OK);
        return n;
    }
    std::vector<int> table(int s) const {
        int n;
        CHECK(sllm_page_seq_tables(c, &s, 1, nullptr, 0, &n) == SLLM_OK);
        std::vector<int> t((size_t)n);
        if (n) CHECK(sllm_page_seq_tables(c, &s, 1, t.data(), n, nullptr) == SLLM_OK);
        return t;
    }
    // everything that a call may change
    std::vector<int> state(const std::vector<int> &seqs) const {
        std::vector<int> all = {vacant()};
        for (int s : seqs) {
            all.push_back(length(s));
            for (int p : table(s)) all.push_back(p);
        }
        return all;
    }
};

struct Batch {
    sllm_page_batch *b = nullptr;
    const Cache &c;
    int heads;
    Batch(const Cache &c, int heads, int seqs, int rows) : c(c), heads(heads) {
        CHECK(sllm_page_batch_create(c.c, heads, seqs, rows, &b) == SLLM_OK);
    }
    ~Batch() { sllm_page_batch_destroy(b); }
    sllm_status begin(const std::vector<int> &seqs, const std::vector<int> &rows) {
        return sllm_page_batch_begin(b, seqs.data(), rows.data(), (int)seqs.size(), nullptr);
    }
    sllm_status attend(int layer = 0) {
        alignas(16) static float x[4];
        sllm_attn_params p{};
        p.n_heads = heads;
        p.n_kv_heads = c.kv;
        p.d_k = c.dk;
        return sllm_page_attention_dev(b, layer, &p, x, x, x, x, nullptr);
    }
};

// The step that the last attention call was given, as the kernels read it: every row's place, and every position that
// it sees in exactly one piece, whose state is where the merge looks for it.
static void check_step(const Cache &c, const std::vector<int> &seqs, const std::vector<int> &rows) {
    const int *step = last.step, rep = last.rep, page_rows = 1 << last.shift;
    int total = 0;
    for (int n : rows) total += n;
    CHECK(step[kStepRows] == total);
    const StepRow *sr = (const StepRow *)(step + step[kStepRowsAt]);
    const StepItem *items = (const StepItem *)(step + kStepHeader);
    struct Seen {
        int p0, p1, slot;
        bool direct;
    };
    std::vector<std::vector<Seen>> seen((size_t)total);
    std::vector<std::vector<int>> tables;
    std::vector<int> of, pos;
    for (size_t i = 0; i < seqs.size(); i++) {
        tables.push_back(c.table(seqs[i]));
        for (int r = 0; r < rows[i]; r++) {
            of.push_back((int)i);
            pos.push_back(c.length(seqs[i]) - rows[i] + r);
        }
    }
    const int *most = kShapeRows[shape_class(last.d_k, last.type == SLLM_CACHE_F16)];
    for (int i = 0; i < step[kStepItems]; i++) {
        const StepItem &x = items[i];
        CHECK(x.p0 >= 0 && x.p0 % 16 == 0 && x.p1 > x.p0 && x.ntok > 0 && x.ntok * rep <= most[x.flags & kItemShape]);
        for (int t = 0; t < x.ntok; t++) {
            const int r = x.flags & kItemRun ? x.tok + t : step[x.tok + t];
            CHECK(r >= 0 && r < total);
            const std::vector<int> &tab = tables[(size_t)of[(size_t)r]];
            const int end = x.flags & kItemCausal ? std::min(x.p1, pos[(size_t)r] + 1) : x.p1;
            CHECK(x.p1 <= c.length(seqs[(size_t)of[(size_t)r]]) && (end == x.p1 || x.lim0 <= end));
            if (end <= x.p0) continue;
            for (int p : {x.p0, (int)(x.p0 + ((int64_t)end - x.p0) / 2), end - 1}) {
                CHECK(step[x.table + p / page_rows] == tab[(size_t)(p / page_rows)]);
                const int u = p / page_rows - x.p0 / page_rows;
                if (u < 8) CHECK(x.pages[u] == tab[(size_t)(p / page_rows)]);
            }
            seen[(size_t)r].push_back({x.p0, end, x.slot + t * rep, (x.flags & kItemDirect) != 0});
        }
    }
    for (int r = 0; r < total; r++) {
        const StepRow &w = sr[r];
        CHECK(w.pos == pos[(size_t)r] && w.slot == w.pos % page_rows);
        CHECK(w.page == tables[(size_t)of[(size_t)r]][(size_t)(w.pos / page_rows)]);
        auto &s = seen[(size_t)r];
        std::sort(s.begin(), s.end(), [](const Seen &a, const Seen &b) { return a.p0 < b.p0; });
        int at = 0;
        size_t n = 0;
        for (int k = 0; k < kMaxParts; k++)
            for (int j = 0; j < w.parts[k].pieces; j++, n++) {
                CHECK(n < s.size() && s[n].p0 == at && s[n].direct == (w.direct != 0));
                at = s[n].p1;
                if (w.direct) continue;
                CHECK(s[n].slot == w.parts[k].first + j * w.parts[k].step);
                CHECK(s[n].slot >= 0 && s[n].slot + rep <= last.slots);
            }
        CHECK(n == s.size() && at == w.pos + 1 && (!w.direct || n == 1));
    }
}

static void run(const Cache &c, Batch &b, const std::vector<int> &seqs, const std::vector<int> &rows) {
    CHECK(b.begin(seqs, rows) == SLLM_OK);
    launches = 0;
    CHECK(b.attend() == SLLM_OK);
    if (launches) check_step(c, seqs, rows);
}

// Steps of many kinds: the plan covers what each row sees.
static void steps() {
    unsigned seed = 1;
    auto below = [&](int n) { return (int)((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
    for (int kind = 0; kind < 60; kind++) {
        const int kv = 1 + below(8), rep = 1 + below(8), dk = 8 * (1 + below(32)), page = 16 << below(5), type = below(2);
        Cache c(1, kv, dk, page, 6000, type);
        Batch b(c, kv * rep, 40, 700);
        std::vector<int> seqs = {c.add(below(5) ? below(3000) : 0)};
        const int n = 2 + below(30);
        while ((int)seqs.size() < n) {
            const int from = seqs[(size_t)below((int)seqs.size())], len = c.length(from);
            const int s = c.fork(from, below(3) ? len : below(len + 1), 1)[0];
            CHECK(sllm_page_seq_extend(c.c, s, below(3) ? below(40) : below(700), nullptr) == SLLM_OK);
            seqs.push_back(s);
        }
        for (int i = 0; i < 4; i++) {
            std::vector<int> rows;
            for (int k = 0; k < n; k++) rows.push_back(i == 0 ? 1 : below(4) ? below(3) : below(20));
            run(c, b, seqs, rows);
        }
        run(c, b, {seqs[0], seqs[1]}, {below(300), 300});
    }
}

// A step that is refused leaves the one before it as it was, also where it would have needed a larger buffer.
static void refused_begin() {
    for (int why = 0; why < 3; why++) {
        Cache c(1, 2, 64, 16, why ? 400 : 40, 0);
        Batch b(c, 4, 2, 4000);
        const int x = c.add(100), y = c.add(3);
        run(c, b, {x}, {2});
        const auto before = c.state({x, y});
        if (why == 1) stub::mallocs_left = 0;
        if (why == 2) stub::host_mallocs_left = 0;
        CHECK(b.begin({x, y}, {1, 3500}) == SLLM_ERR_OOM);
        stub::mallocs_left = stub::host_mallocs_left = -1;
        CHECK(c.state({x, y}) == before);
        CHECK(b.attend() == SLLM_OK);
        check_step(c, {x}, {2});
        run(c, b, {x, y}, {1, 40});
        if (why) run(c, b, {x, y}, {1, 3500});
    }
}

// Host memory that runs out anywhere in a call: it says so, and nothing has changed.
template <class Call, class State>
static void every_allocation_fails(Call call, State state) {
    const auto before = state();
    for (long n = 0;; n++) {
        CHECK(n < 1000);
        news_failed = false;
        news_left = n;
        const sllm_status st = call();
        news_left = -1;
        if (!news_failed) {
            CHECK(st == SLLM_OK);
            return;
        }
        CHECK(st == SLLM_ERR_OOM && state() == before);
    }
}

static void out_of_memory() {
    Cache c(1, 2, 64, 16, 400, 1);
    Batch b(c, 4, 8, 64);
    std::vector<int> seqs = {c.add(700)};
    for (int s : c.fork(seqs[0], 650, 5)) seqs.push_back(s);
    const std::vector<int> first = {1, 0, 2, 1, 1, 3};
    run(c, b, seqs, first);
    auto whole = [&] { return c.state(seqs); };
    auto step_too = [&] {
        CHECK(b.attend() == SLLM_OK);
        check_step(c, seqs, first);
        return c.state(seqs);
    };
    int out[3];
    every_allocation_fails([&] { return sllm_page_seq_fork(c.c, seqs[1], 333, 3, out); }, whole);
    every_allocation_fails([&] { return sllm_page_seq_copy(c.c, seqs[1], 333, 3, out, nullptr); }, whole);
    every_allocation_fails([&] { return sllm_page_seq_extend(c.c, out[0], 99, nullptr); }, whole);
    std::vector<int> grown;
    for (int s : seqs) grown.push_back(s);
    const std::vector<int> rows = {1, 3, 2, 20, 1, 3};
    every_allocation_fails([&] { return sllm_page_batch_begin(b.b, grown.data(), rows.data(), 6, nullptr); }, step_too);
    CHECK(b.attend() == SLLM_OK);
    check_step(c, seqs, rows);
    every_allocation_fails([&] { return sllm_page_seq_free(c.c, seqs.data() + 1, 2); }, whole);
    seqs = {seqs[0], seqs[3], seqs[4], seqs[5]};
    every_allocation_fails([&] { return sllm_page_cache_compact(c.c, nullptr, nullptr); }, whole);
    run(c, b, seqs, {1, 1, 1, 1});
}

// Copies that can't be launched: the call says so, and its sequences, their pages and the step before it are as they were.
static void failed_copies() {
    Cache c(1, 2, 64, 16, 900, 1);
    Batch b(c, 4, 8, 64);
    std::vector<int> seqs = {c.add(700)};
    for (int s : c.fork(seqs[0], 650, 5)) seqs.push_back(s);
    for (int s : c.fork(seqs[1], 645, 1)) seqs.push_back(s);
    const std::vector<int> first = {1, 0, 2, 0, 0, 0, 0};
    run(c, b, seqs, first);
    const auto before = c.state(seqs);
    auto refused = [&](sllm_status st) {
        stub::launches_left = -1;
        CHECK(st == SLLM_ERR_DEVICE && c.state(seqs) == before);
        CHECK(b.attend() == SLLM_OK);
        check_step(c, seqs, first);
    };
    int out[9];
    stub::launches_left = 1;  // (the second of two)
    refused(sllm_page_seq_copy(c.c, seqs[1], 650, 9, out, nullptr));
    stub::launches_left = 0;
    refused(sllm_page_seq_extend(c.c, seqs[3], 50, nullptr));
    stub::launches_left = 0;
    refused(b.begin(seqs, {1, 1, 1, 20, 1, 1, 30}));
    stub::launches_left = 0;
    refused(sllm_page_seq_extend(c.c, seqs[6], 50, nullptr));
    stub::launches_left = 0;
    CHECK(sllm_page_seq_free(c.c, seqs.data() + 3, 1) == SLLM_OK);
    seqs.erase(seqs.begin() + 3);
    const auto gap = c.state(seqs);
    CHECK(sllm_page_cache_compact(c.c, nullptr, nullptr) == SLLM_OK);  // (nothing to move)
    stub::launches_left = -1;
    CHECK(c.state(seqs) == gap);
    run(c, b, seqs, {1, 1, 1, 1, 1, 30});
    // neither can the step's description: no step, and no rows either
    for (const auto &rows : {std::vector<int>{1, 1, 1, 1, 1, 1}, std::vector<int>{9, 9, 9, 9, 9, 9}}) {
        seqs.push_back(c.fork(seqs[0], 701, 1)[0]);  // (and a tail page to copy)
        const auto before = c.state(seqs);
        std::vector<int> all = rows;
        all.resize(seqs.size());
        stub::launches_left = 1;
        stub::memcpys_left = 0;
        CHECK(b.begin(seqs, all) == SLLM_ERR_DEVICE && c.state(seqs) == before && b.attend() == SLLM_ERR_ARG);
        stub::launches_left = stub::memcpys_left = -1;
        run(c, b, seqs, all);
    }
    CHECK(seqs[6] == 3 && seqs[7] == 7 && c.add() == 8);  // numbers of sequences that were not made are free
}

// Sequences up to the longest, whose pieces end next to what 32 bits hold.
static void long_sequences() {
    const int longest = INT32_MAX - 512;
    for (int rows : {longest - 40, longest - 4000000, longest / 2 + 77})
        for (int type = 0; type < 2; type++) {
            Cache c(1, 1, 8, 256, 1 << 23, type);
            Batch b(c, 1, 2, 64);
            const int s = c.add(rows);
            run(c, b, {s}, {1});
            run(c, b, {s}, {30});
            run(c, b, c.fork(s, rows, 2), {1, 2});
            CHECK(sllm_page_seq_extend(c.c, s, longest - rows, nullptr) == SLLM_ERR_SHAPE);
        }
}

// Batches of more rows and heads than a launch can have threads for are refused; the largest are made.
static void many_rows() {
    for (int dk : {8, 16, 24}) {
        Cache c(1, 1, dk, 16, 4, 1);
        sllm_page_batch *b = nullptr;
        for (int heads : {1, 8}) {
            CHECK(sllm_page_batch_create(c.c, heads, 1, (1 << 24) / heads, &b) == SLLM_ERR_SHAPE && !b);
            const int most = std::min((1 << 24) / heads - 1, (1 << 28) / heads / dk);
            CHECK(sllm_page_batch_create(c.c, heads, 1, most, &b) == SLLM_OK);
            sllm_page_batch_destroy(b);
        }
    }
    // more pieces than workgroups: a row each of many sequences, for many kv heads
    Cache c(1, 3000, 8, 16, 4000, 1);
    Batch b(c, 3000, 3000, 3000);
    std::vector<int> seqs, rows(3000, 1);
    for (int i = 0; i < 3000; i++) seqs.push_back(c.add(0));
    run(c, b, seqs, rows);
    CHECK((uint64_t)last.grid_items * 256 >> 32 == 0 && last.items == 3000 * 3000);
}

int main(int argc, char **argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "steps") steps();
    else if (what == "refused_begin") refused_begin();
    else if (what == "out_of_memory") out_of_memory();
    else if (what == "failed_copies") failed_copies();
    else if (what == "long_sequences") long_sequences();
    else if (what == "many_rows") many_rows();
    else return 2;
    std::puts("ok");
    return 0;
}
