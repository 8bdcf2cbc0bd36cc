// Pre-launch argument validation of the entry points for windowed attention, caches cut by weight
// and drafted tokens, built as tests/abi_validation.cpp is: host code under AddressSanitizer and
// UBSan, a HIP runtime with no device (tests/hip_stub.cpp), fake pointers that nothing may
// dereference. Every integer argument in turn takes extreme values; a call that passes
// validation fails its launch.
#include <climits>
#include <cmath>
#include <cstdio>
#include <functional>
#include <string>
#include <vector>

#include "crucible_attn.h"

namespace {

int g_failed = 0, g_checks = 0, g_swept = 0;

void expect(const char* what, int got, int want) {
    ++g_checks;
    if (got != want) {
        char msg[256];
        crucible_attn_last_error(msg, sizeof msg);
        std::printf("FAIL %s: status %d, want %d (%s)\n", what, got, want, msg);
        ++g_failed;
    }
}

void* const F = reinterpret_cast<void*>(0x1000);  // 16-byte aligned, never dereferenced
void* const ODD = reinterpret_cast<void*>(0x1008);
const int32_t* const FI = reinterpret_cast<const int32_t*>(0x1000);
int32_t* const FO = reinterpret_cast<int32_t*>(0x1000);
float* const FW = reinterpret_cast<float*>(0x1000);
const size_t BIG = (size_t)1 << 40;

const int64_t kExtremes[] = {-1, 0, 1, 7, 65535, 65536, INT32_MAX, (int64_t)INT32_MAX + 1, (int64_t)1 << 40,
                             INT64_MAX, INT64_MIN, INT64_MAX / 64};

struct Entry {
    const char* name;
    std::vector<int64_t> base;
    std::function<int(const std::vector<int64_t>&, void* pool, void* ws, size_t bytes)> call;
    std::function<size_t(const std::vector<int64_t>&)> bytes;
};

std::vector<Entry> entries() {
    using V = const std::vector<int64_t>&;
    std::vector<Entry> e;
    e.push_back({"decode_window", {16, 12, 3, 64, 256, 12, 0, 192, 4096, 1024, 4},
                 [](V a, void* pool, void* ws, size_t n) {
        return crucible_attention_decode_window_paged(F, CRUCIBLE_F32, pool, F, F, CRUCIBLE_F16, FI, FI, a[0], a[1],
                                                      a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], ws, n,
                                                      nullptr);
    }, [](V a) {
        return crucible_attention_decode_window_workspace_bytes(a[0], a[1], a[2], a[3], a[8], a[9], a[10]);
    }});
    e.push_back({"prefill_window", {4, 300, 256, 12, 3, 64, 12, 0, 192, 1024, 4},
                 [](V a, void* pool, void* ws, size_t n) {
        return crucible_attention_prefill_window_tiled(F, CRUCIBLE_F16, pool, F, F, CRUCIBLE_F32, FI, FI, a[0], a[1],
                                                       a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], ws, n,
                                                       nullptr);
    }, [](V a) {
        return crucible_attention_prefill_window_workspace_bytes(a[0], a[1], a[2], a[3], a[4], a[5], a[9], a[10]);
    }});
    e.push_back({"decode_weigh", {16, 12, 3, 64, 256, 12, 0, 192, 4096},
                 [](V a, void* pool, void* ws, size_t n) {
        return crucible_attention_decode_weigh_paged(F, CRUCIBLE_F32, pool, F, FW, FO, F, CRUCIBLE_F32, FI, FI, FI,
                                                     a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], ws, n,
                                                     nullptr);
    }, [](V a) { return crucible_attention_decode_weigh_workspace_bytes(a[0], a[1], a[2], a[3], a[8]); }});
    e.push_back({"cache_weigh", {4, 300, 256, 12, 3, 64, 12, 0, 192, 64},
                 [](V a, void* pool, void* ws, size_t n) {
        return crucible_cache_weigh_tiled(F, CRUCIBLE_F32, pool, FW, FO, FI, FI, FI, a[0], a[1], a[2], a[3], a[4],
                                          a[5], a[6], a[7], a[8], a[9], ws, n, nullptr);
    }, [](V a) { return crucible_cache_weigh_workspace_bytes(a[0], a[1], a[2], a[3], a[4], a[5], a[9]); }});
    e.push_back({"cache_evict", {16, 3, 64, 256, 12, 192, 4096, 1024, 4, 256},
                 [](V a, void* pool, void* ws, size_t n) {
        return crucible_cache_evict_paged(pool, F, FW, FO, FI, FI, FO, a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7],
                                          a[8], a[9], ws, n, nullptr);
    }, [](V a) { return crucible_cache_evict_workspace_bytes(a[0], a[1], a[4], a[6], a[7]); }});
    e.push_back({"verify_drafts", {16, 4, 50257}, [](V a, void*, void* ws, size_t n) {
        return crucible_verify_drafts(F, F, CRUCIBLE_F32, FI, FI, FW, FW, FO, FO, a[0], a[1], a[2], 1.0, ws, n,
                                      nullptr);
    }, [](V a) { return crucible_verify_drafts_workspace_bytes(a[0], a[1], a[2]); }});
    return e;
}

void sweep() {
    for (const Entry& e : entries()) {
        const std::string name = e.name;
        expect((name + ": ordinary arguments reach the launch").c_str(), e.call(e.base, F, F, BIG),
               CRUCIBLE_ERR_LAUNCH);
        const size_t need = e.bytes(e.base);
        if (need) {
            expect((name + ": no workspace").c_str(), e.call(e.base, F, nullptr, 0), CRUCIBLE_ERR_WORKSPACE);
            expect((name + ": workspace short by a byte").c_str(), e.call(e.base, F, F, need - 1),
                   CRUCIBLE_ERR_WORKSPACE);
            expect((name + ": workspace as large as asked").c_str(), e.call(e.base, F, F, need),
                   CRUCIBLE_ERR_LAUNCH);
            expect((name + ": workspace off 16 bytes").c_str(), e.call(e.base, F, ODD, BIG), CRUCIBLE_ERR_INVALID);
        }
        if (name != "verify_drafts") {
            expect((name + ": pool off 16 bytes").c_str(), e.call(e.base, ODD, F, BIG), CRUCIBLE_ERR_INVALID);
            expect((name + ": null pool").c_str(), e.call(e.base, nullptr, F, BIG), CRUCIBLE_ERR_INVALID);
        }
        for (size_t i = 0; i < e.base.size(); ++i)
            for (int64_t v : kExtremes) {
                std::vector<int64_t> a = e.base;
                a[i] = v;
                (void)e.bytes(a);
                (void)e.call(a, F, F, BIG);
                for (size_t j = 0; j < e.base.size(); ++j)  // and in pairs
                    for (int64_t w : {(int64_t)-1, (int64_t)INT32_MAX, INT64_MAX}) {
                        if (j == i) continue;
                        std::vector<int64_t> b = a;
                        b[j] = w;
                        (void)e.bytes(b);
                        (void)e.call(b, F, F, BIG);
                        ++g_swept;
                    }
                if (v < 0) {
                    const int rc = e.call(a, F, F, BIG);
                    expect((name + ": a negative argument").c_str(),
                           rc == CRUCIBLE_ERR_INVALID || rc == CRUCIBLE_ERR_UNSUPPORTED ? 0 : rc + 1000, 0);
                }
            }
    }
}

void explicit_cases() {
    const auto window = [](int q, int o, int64_t hd, int64_t kv, int64_t heads, int64_t layer, int64_t w, int64_t s) {
        return crucible_attention_decode_window_paged(F, q, F, F, F, o, FI, FI, 2, heads, 3, hd, 64, 12, layer, kv,
                                                      1024, w, s, F, BIG, nullptr);
    };
    expect("bad q dtype", window(7, 0, 64, 192, 12, 0, 9, 0), CRUCIBLE_ERR_INVALID);
    expect("bad out dtype", window(0, 2, 64, 192, 12, 0, 9, 0), CRUCIBLE_ERR_INVALID);
    expect("head_dim 100", window(0, 0, 100, 300, 12, 0, 9, 0), CRUCIBLE_ERR_UNSUPPORTED);
    expect("head_dim 264", window(0, 0, 264, 792, 12, 0, 9, 0), CRUCIBLE_ERR_UNSUPPORTED);
    expect("kv_dim", window(0, 0, 64, 200, 12, 0, 9, 0), CRUCIBLE_ERR_INVALID);
    expect("heads", window(0, 0, 64, 192, 13, 0, 9, 0), CRUCIBLE_ERR_INVALID);
    expect("layer", window(0, 0, 64, 192, 12, 12, 9, 0), CRUCIBLE_ERR_INVALID);
    expect("window", window(0, 0, 64, 192, 12, 0, -1, 0), CRUCIBLE_ERR_INVALID);
    expect("sinks", window(0, 0, 64, 192, 12, 0, 9, -1), CRUCIBLE_ERR_INVALID);
    expect("max_seq past the table",
           crucible_attention_decode_window_paged(F, 0, F, F, F, 0, FI, FI, 2, 12, 3, 64, 64, 12, 0, 192, 1025, 9, 0, F,
                                                  BIG, nullptr),
           CRUCIBLE_ERR_INVALID);
    const auto pages = [](int64_t n) {
        return crucible_attention_prefill_window_tiled(F, 0, F, F, F, 0, FI, FI, 1, 5, n, 12, 3, 64, 12, 0, 192, 9, 0, F,
                                                       BIG, nullptr);
    };
    expect("the largest table", pages((int64_t)1 << 26), CRUCIBLE_ERR_LAUNCH);
    expect("a page more", pages(((int64_t)1 << 26) + 1), CRUCIBLE_ERR_INVALID);
    const auto weigh_pages = [](int64_t n) {
        return crucible_cache_weigh_tiled(F, 0, F, FW, FO, FI, FI, FI, 1, 5, n, 12, 3, 64, 12, 0, 192, 8, F, BIG, nullptr);
    };
    expect("the largest table, weighed", weigh_pages((int64_t)1 << 26), CRUCIBLE_ERR_LAUNCH);
    expect("a page more, weighed", weigh_pages(((int64_t)1 << 26) + 1), CRUCIBLE_ERR_INVALID);
    expect("empty batch", crucible_attention_decode_window_paged(nullptr, 0, nullptr, nullptr, nullptr, 0, nullptr,
                                                                 nullptr, 0, 12, 3, 64, 64, 12, 0, 192, 1024, 9, 0,
                                                                 nullptr, 0, nullptr),
           CRUCIBLE_OK);
    const auto evict = [](int64_t keep, int64_t sink, int64_t recent) {
        return crucible_cache_evict_paged(F, F, FW, FO, FI, FI, FO, 2, 3, 64, 64, 12, 192, 1024, keep, sink, recent, F,
                                          BIG, nullptr);
    };
    expect("keep 0", evict(0, 0, 0), CRUCIBLE_ERR_INVALID);
    expect("first tokens past keep", evict(10, 11, 0), CRUCIBLE_ERR_INVALID);
    expect("first and newest past keep", evict(10, 5, 6), CRUCIBLE_ERR_INVALID);
    const auto verify = [](const void* target, const void* draft, const int32_t* drafts, int64_t k, double t) {
        return crucible_verify_drafts(target, draft, CRUCIBLE_F32, drafts, FI, FW, FW, FO, FO, 2, k, 100, t, F, BIG,
                                      nullptr);
    };
    expect("temperature 0", verify(F, F, FI, 4, 0.0), CRUCIBLE_ERR_INVALID);
    expect("temperature below 0", verify(F, F, FI, 4, -1.0), CRUCIBLE_ERR_INVALID);
    expect("temperature NaN", verify(F, F, FI, 4, NAN), CRUCIBLE_ERR_INVALID);
    expect("temperature infinite", verify(F, F, FI, 4, INFINITY), CRUCIBLE_ERR_INVALID);
    expect("65 drafts", verify(F, F, FI, 65, 1.0), CRUCIBLE_ERR_INVALID);
    expect("no target", verify(nullptr, F, FI, 4, 1.0), CRUCIBLE_ERR_INVALID);
    expect("no drafts", verify(F, F, nullptr, 4, 1.0), CRUCIBLE_ERR_INVALID);
    expect("a certain draft", verify(F, nullptr, FI, 4, 1.0), CRUCIBLE_ERR_LAUNCH);
    expect("no drafts to verify", verify(F, nullptr, nullptr, 0, 1.0), CRUCIBLE_ERR_LAUNCH);
}

void paging() {
    crucible_page_pool* p = crucible_page_pool_new(8, 12, 192);
    crucible_seq_pages* s = crucible_seq_pages_new();
    expect("grow", crucible_seq_pages_grow(s, p, 100), CRUCIBLE_OK);
    for (int64_t v : {(int64_t)-1, (int64_t)101, INT64_MAX, INT64_MIN})
        expect("shrink to more, or less than nothing", crucible_seq_pages_shrink(s, p, v), CRUCIBLE_ERR_INVALID);
    expect("length kept", (int)crucible_seq_pages_len(s), 100);
    expect("shrink", crucible_seq_pages_shrink(s, p, 33), CRUCIBLE_OK);
    expect("pages held", (int)crucible_seq_pages_n_pages(s), 3);
    expect("pages free", (int)crucible_page_pool_free_pages(p), 5);
    expect("shrink to nothing", crucible_seq_pages_shrink(s, p, 0), CRUCIBLE_OK);
    expect("all free", (int)crucible_page_pool_free_pages(p), 8);
    crucible_seq_pages_free(s);
    crucible_page_pool_free(p);
}

}  // namespace

int main() {
    std::setvbuf(stdout, nullptr, _IOLBF, 0);
    explicit_cases();
    paging();
    sweep();
    std::printf("%d checks, %d failed; %d extreme-value calls swept\n", g_checks, g_failed, g_swept);
    return g_failed ? 1 : 0;
}
