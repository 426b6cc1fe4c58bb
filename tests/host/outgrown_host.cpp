// A captured batch's buffer (qmm_pages.hip), on the CPU: a step that outgrows it is refused for what it is made of. Compiled
// against hip/hip_runtime.h beside this file.
#include <cstdio>
#include <cstdlib>
#include <string>

#include "qmm_pages.hip"

static std::string error;

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
sllm_status launch_page_attention(const PageAttnArgs &, hipStream_t) { return SLLM_OK; }
}  // namespace sllm

#define CHECK(x)                                                                               \
    do {                                                                                       \
        if (!(x)) {                                                                            \
            std::fprintf(stderr, "%s:%d: %s (%s)\n", __FILE__, __LINE__, #x, error.c_str()); \
            std::exit(1);                                                                      \
        }                                                                                      \
    } while (0)

int main() {
    sllm_page_cache *c;
    sllm_page_batch *b;
    CHECK(sllm_page_cache_create(1, 1, 64, 16, 400, 0, &c) == SLLM_OK);
    CHECK(sllm_page_batch_create(c, 2, 4, 4096, &b) == SLLM_OK);
    int s[4];
    for (int &x : s) CHECK(sllm_page_seq_add(c, &x) == SLLM_OK);
    int one = 1, root = -1, len;
    CHECK(sllm_page_batch_begin_tree(b, s, &one, 1, &root, nullptr) == SLLM_OK);
    alignas(16) static float x[4];
    sllm_attn_params p{};
    p.n_heads = 2;
    p.n_kv_heads = 1;
    p.d_k = 64;
    stub::capture = true;
    CHECK(sllm_page_attention_dev(b, 0, &p, x, x, x, x, nullptr) == SLLM_OK);
    stub::capture = false;
    // (a tree of 1000 rows has 130 KB of bits beside its rows and pages)
    std::vector<int> wide;
    for (int i = 0; i < 1000; i++) wide.push_back(i ? 0 : -1);
    int rows = 1000;
    const sllm_status grown = sllm_page_batch_begin_tree(b, s + 1, &rows, 1, wide.data(), nullptr);
    CHECK(grown == SLLM_ERR_SHAPE);
    CHECK(error.find("trees") != std::string::npos && error.find("captured") != std::string::npos);
    CHECK(sllm_page_seq_length(c, s[1], &len) == SLLM_OK && len == 0);
    // the step before stays
    CHECK(sllm_page_attention_dev(b, 0, &p, x, x, x, x, nullptr) == SLLM_OK);
    sllm_page_batch_destroy(b);
    sllm_page_cache_destroy(c);
    return 0;
}
