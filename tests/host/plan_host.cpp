// What a step's begin plans (qmm_pages.hip), on the CPU: compiled against hip/hip_runtime.h beside this file. A step on a line
// of stdin: heads, kv heads, d_k, type, page rows, rows of a shared prefix, sequences, whether they have parents; for each
// sequence rows of its own and rows of the step, and the parents of these. Printed for each: the most pieces of a row, then its
// blocks of rows: shape, whether they are a tree, whether causal, rows (of q heads), tiles of 32 positions, how many.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <string>
#include <tuple>

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

int main() {
    int heads, kv, dk, type, page, prefix, n, trees;
    while (std::scanf("%d %d %d %d %d %d %d %d", &heads, &kv, &dk, &type, &page, &prefix, &n, &trees) == 8) {
        std::vector<int> own((size_t)n), rows((size_t)n), seqs((size_t)n), parents;
        int total = 0, pages = prefix / page + 2;
        for (int i = 0; i < n; i++) {
            CHECK(std::scanf("%d %d", &own[(size_t)i], &rows[(size_t)i]) == 2);
            total += rows[(size_t)i];
            pages += (own[(size_t)i] + rows[(size_t)i]) / page + 3;
            for (int r = 0; trees && r < rows[(size_t)i]; r++) {
                int p;
                CHECK(std::scanf("%d", &p) == 1);
                parents.push_back(p);
            }
        }
        sllm_page_cache *c;
        sllm_page_batch *b;
        CHECK(sllm_page_cache_create(1, kv, dk, page, pages, type, &c) == SLLM_OK);
        CHECK(sllm_page_batch_create(c, heads, n, total, &b) == SLLM_OK);
        int base;
        CHECK(sllm_page_seq_add(c, &base) == SLLM_OK && sllm_page_seq_extend(c, base, prefix, nullptr) == SLLM_OK);
        CHECK(sllm_page_seq_fork(c, base, prefix, n, seqs.data()) == SLLM_OK);
        for (int i = 0; i < n; i++) CHECK(sllm_page_seq_extend(c, seqs[(size_t)i], own[(size_t)i], nullptr) == SLLM_OK);
        CHECK((trees ? sllm_page_batch_begin_tree(b, seqs.data(), rows.data(), n, parents.data(), nullptr)
                     : sllm_page_batch_begin(b, seqs.data(), rows.data(), n, nullptr)) == SLLM_OK);
        alignas(16) static float x[4];
        sllm_attn_params p{};
        p.n_heads = heads;
        p.n_kv_heads = kv;
        p.d_k = dk;
        CHECK(sllm_page_attention_dev(b, 0, &p, x, x, x, x, nullptr) == SLLM_OK);
        const StepItem *items = (const StepItem *)(last.step + kStepHeader);
        std::map<std::tuple<int, int, int, int, int>, int> blocks;
        for (int i = 0; i < last.step[kStepItems]; i++) {
            const StepItem &it = items[i];
            blocks[{it.flags & kItemShape, (it.flags & kItemTree) != 0, (it.flags & kItemCausal) != 0, it.ntok * heads / kv,
                    (it.p1 - it.p0 + 31) / 32}]++;
        }
        std::printf("%d", last.combine);
        for (const auto &[k, many] : blocks)
            std::printf(" %d %d %d %d %d %d", std::get<0>(k), std::get<1>(k), std::get<2>(k), std::get<3>(k), std::get<4>(k), many);
        std::printf("\n");
        sllm_page_batch_destroy(b);
        sllm_page_cache_destroy(c);
    }
    return 0;
}
