// kvb_api_pages.cu - kvb_page_* (include/kvb.h): validation and launches of the 8-bit paged cache's writes,
// reads and page operations (kvb_pages.cuh).
#include <cuda_runtime.h>

#include <algorithm>

#include "kvb_host.h"
#include "kvb_pages.cuh"
#include "kvb_pages_host.h"

namespace {

constexpr int kMaxSequences = 6000;        // offsets of one call's sequences in the planning block's shared memory

// "" or what is wrong with a packed rows call
kvb_status check_rows(const char* who, const kvb_pages* p, const int32_t* slots, const int32_t* start, const int32_t* cu,
                      int n, const void* k, const void* v, int dtype, int64_t rows) {
    if (kvb_status st = kvbh::check_pages(who, p)) return st;
    if (n > 0 && rows > 0 && (!slots || !start || !cu || !k || !v)) return fail(KVB_EINVAL, "%s: null argument", who);
    if (n < 0 || rows < 0 || rows > INT32_MAX) return fail(KVB_EINVAL, "%s: n >= 0 and 0 <= rows < 2^31", who);
    if (dtype != KVB_F32 && dtype != KVB_F16 && dtype != KVB_BF16)
        return fail(KVB_EINVAL, "%s: dtype float32, float16 or bfloat16", who);
    return KVB_OK;
}

// Rounds of 8 values a thread that hold a whole page of rows.
template <typename T>
kvb_status launch_write(const kvb::PageRowsParams& a, dim3 grid, cudaStream_t s) {
    const int rounds = a.P.page * a.P.d / (8 * kvb::PW_THREADS);
    const auto kern = rounds <= 1   ? kvb::page_write_kernel<T, 1>
                      : rounds == 2 ? kvb::page_write_kernel<T, 2>
                      : rounds == 4 ? kvb::page_write_kernel<T, 4>
                      : rounds == 8 ? kvb::page_write_kernel<T, 8>
                                    : kvb::page_write_kernel<T, 16>;
    return launch_chained("page_write", kern, grid, kvb::PW_THREADS, 0, s, a);
}

// Threads of a planning block: 32 per 1024 pages (their barriers cost more than the pages of a small pool), 128 to 1024.
unsigned page_block(const kvb_pages* p) { return unsigned(std::min<int64_t>(kvb::PG_THREADS, std::max<int64_t>(128, (p->n_pages + 1023) / 1024 * 32))); }

// Pools of one table: the layers of a model.
kvb_status check_layers(const char* who, const kvb_pages* p, int n_pools) {
    if (!p || n_pools <= 0) return fail(KVB_EINVAL, "%s: null argument", who);
    for (int i = 0; i < n_pools; ++i) {
        if (kvb_status st = kvbh::check_pages(who, p + i)) return st;
        if (p[i].table != p->table || p[i].lens != p->lens || p[i].refs != p->refs || p[i].n_pages != p->n_pages ||
            p[i].page != p->page || p[i].n_slots != p->n_slots || p[i].max_blocks != p->max_blocks)
            return fail(KVB_EINVAL, "%s: pools of one call share table, lens, refs and sizes", who);
    }
    return KVB_OK;
}

size_t fork_rows_offset(int n) { return (size_t(64 + 2 * size_t(n)) * 4 + 255) / 256 * 256; }

kvb::ForkWork fork_work(void* ws, int n) {
    int32_t* b = static_cast<int32_t*>(ws);
    return {b, b + 64, b + 64 + n, reinterpret_cast<int32_t*>(static_cast<char*>(ws) + fork_rows_offset(n))};
}

}  // namespace

namespace kvbh {

kvb_status check_pages(const char* who, const kvb_pages* p) {
    if (!p || !p->kc || !p->vc || !p->ks || !p->vs || !p->table || !p->lens || !p->refs)
        return fail(KVB_EINVAL, "%s: null argument", who);
    if (p->n_pages <= 0 || p->n_pages > INT32_MAX || p->Hkv <= 0 || p->Hkv > 4096 || p->n_slots <= 0 || p->max_blocks <= 0)
        return fail(KVB_EINVAL, "%s: sizes of the pool (0 < Hkv <= 4096, 0 < n_pages < 2^31)", who);
    if (p->page != 16 && p->page != 32 && p->page != 64 && p->page != 128)
        return fail(KVB_EUNSUPPORTED, "%s: pages of 16, 32, 64 or 128 tokens", who);
    if (p->d != 64 && p->d != 128) return fail(KVB_EUNSUPPORTED, "%s: d 64 or 128", who);
    if (int64_t(p->max_blocks) * p->page > INT32_MAX) return fail(KVB_EINVAL, "%s: max_blocks * page < 2^31", who);
    if (!aligned(p->kc, 16) || !aligned(p->vc, 16)) return fail(KVB_EINVAL, "%s: codes need 16-byte alignment", who);
    return KVB_OK;
}

kvb::PagesView view_of(const kvb_pages* p) {
    return {p->kc, p->vc, p->ks, p->vs, p->table, p->lens, p->refs, p->n_pages, p->Hkv, p->d, p->page, p->n_slots, p->max_blocks};
}

}  // namespace kvbh

extern "C" {

kvb_status kvb_page_write(const kvb_pages* p, const int32_t* slots, const int32_t* start, const int32_t* cu, int n,
                          const void* k, const void* v, int dtype, int64_t rows, int64_t k_row, int64_t k_head,
                          int64_t v_row, int64_t v_head, void* stream) {
    if (kvb_status st = check_rows("page_write", p, slots, start, cu, n, k, v, dtype, rows)) return st;
    if (n == 0 || rows == 0) return KVB_OK;
    kvb::PageRowsParams a{kvbh::view_of(p), slots, start, cu, n, rows, {k, v}, {k_row, v_row}, {k_head, v_head}, {}};
    const dim3 grid(unsigned(rows / p->page + 2 * int64_t(n)), unsigned(p->Hkv), 2);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool vectors = dtype != KVB_F32 && aligned(k, 16) && aligned(v, 16) && (k_row | k_head | v_row | v_head) % 8 == 0;
    if (vectors) return dtype == KVB_F16 ? launch_write<__half>(a, grid, s) : launch_write<__nv_bfloat16>(a, grid, s);
    const auto kern = dtype == KVB_F32   ? kvb::page_write_any_kernel<float>
                      : dtype == KVB_F16 ? kvb::page_write_any_kernel<__half>
                                         : kvb::page_write_any_kernel<__nv_bfloat16>;
    return launch_chained("page_write", kern, grid, 256, 0, s, a);
}

kvb_status kvb_page_read(const kvb_pages* p, const int32_t* slots, const int32_t* start, const int32_t* cu, int n, void* k,
                         void* v, int dtype, int64_t rows, void* stream) {
    if (kvb_status st = check_rows("page_read", p, slots, start, cu, n, k, v, dtype, rows)) return st;
    if (n == 0 || rows == 0) return KVB_OK;
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(KVB_EINVAL, "page_read: k and v need 16-byte alignment");
    kvb::PageRowsParams a{kvbh::view_of(p), slots, start, cu, n, rows, {}, {}, {}, {k, v}, aligned(k, 32) && aligned(v, 32)};
    const dim3 grid(unsigned(rows / p->page + 2 * int64_t(n)),
                    unsigned((2 * int64_t(p->Hkv) * p->page * p->d + kvb::PR_SHARE - 1) / kvb::PR_SHARE));
    const auto kern = dtype == KVB_F32   ? kvb::page_read_kernel<float>
                      : dtype == KVB_F16 ? kvb::page_read_kernel<__half>
                                         : kvb::page_read_kernel<__nv_bfloat16>;
    return launch_chained("page_read", kern, grid, kvb::PW_THREADS, 0, static_cast<cudaStream_t>(stream), a);
}

kvb_status kvb_page_extend(const kvb_pages* p, const int32_t* slots, const int32_t* add, int n, int32_t* start, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_extend", p)) return st;
    if (n > 0 && (!slots || !add || !start)) return fail(KVB_EINVAL, "page_extend: null argument");
    if (n < 0 || n > kMaxSequences) return fail(KVB_EINVAL, "page_extend: 0 <= n <= %d sequences a call", kMaxSequences);
    if (n == 0) return KVB_OK;
    return launch_chained("page_extend", kvb::page_extend_kernel, 1, page_block(p), size_t(n) * 4, static_cast<cudaStream_t>(stream),
                          kvbh::view_of(p), slots, add, n, start);
}

kvb_status kvb_page_free(const kvb_pages* p, const int32_t* slots, int n, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_free", p)) return st;
    if (n > 0 && !slots) return fail(KVB_EINVAL, "page_free: null argument");
    if (n < 0) return fail(KVB_EINVAL, "page_free: n >= 0");
    if (n == 0) return KVB_OK;
    return launch_chained("page_free", kvb::page_free_kernel, unsigned(n), 128, 0, static_cast<cudaStream_t>(stream), kvbh::view_of(p),
                          slots);
}

kvb_status kvb_page_copy(const kvb_pages* p, int n_pools, const int32_t* src, const int32_t* dst, int n, void* stream) {
    if (kvb_status st = check_layers("page_copy", p, n_pools)) return st;
    if (n > 0 && (!src || !dst)) return fail(KVB_EINVAL, "page_copy: null argument");
    if (n < 0) return fail(KVB_EINVAL, "page_copy: n >= 0");
    if (n == 0) return KVB_OK;
    for (int i = 0; i < n_pools; ++i)
        if (kvb_status st = launch_chained("page_copy", kvb::page_copy_kernel, dim3(unsigned(n), 4), kvb::PG_COPY_THREADS, 0,
                                           static_cast<cudaStream_t>(stream), kvbh::view_of(p + i), src, dst))
            return st;
    return KVB_OK;
}

size_t kvb_page_fork_workspace(const kvb_pages* p, int n) {
    if (kvbh::check_pages("page_fork", p) || n < 0 || n > kMaxSequences) return 0;
    return fork_rows_offset(n) + size_t(n) * p->max_blocks * 4;
}

kvb_status kvb_page_fork(const kvb_pages* p, int n_pools, const int32_t* src, const int32_t* dst, int n, void* workspace,
                         size_t workspace_bytes, void* stream) {
    if (kvb_status st = check_layers("page_fork", p, n_pools)) return st;
    if (n > 0 && (!src || !dst || !workspace)) return fail(KVB_EINVAL, "page_fork: null argument");
    if (n < 0 || n > kMaxSequences) return fail(KVB_EINVAL, "page_fork: 0 <= n <= %d sequences a call", kMaxSequences);
    if (n == 0) return KVB_OK;
    const size_t need = kvb_page_fork_workspace(p, n);
    if (workspace_bytes < need) return fail(KVB_EINVAL, "page_fork: workspace of %zu bytes, need %zu", workspace_bytes, need);
    if (!aligned(workspace, 256)) return fail(KVB_EINVAL, "page_fork: workspace needs 256-byte alignment");
    const kvb::PagesView v = kvbh::view_of(p);
    const kvb::ForkWork w = fork_work(workspace, n);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kvb_status st = launch_chained("page_fork plan", kvb::fork_plan_kernel, 1, page_block(p), size_t(n + 1) * 4, s, v, src, dst, n, w))
        return st;
    for (int i = 0; i < n_pools; ++i)
        if (kvb_status st = launch_chained("page_fork copy", kvb::fork_copy_kernel, dim3(unsigned(n), 1 + 8), kvb::PG_COPY_THREADS, 0, s,
                                           kvbh::view_of(p + i), src, w))
            return st;
    return launch_chained("page_fork commit", kvb::fork_commit_kernel, unsigned(n), 128, 0, s, v, src, dst, w);
}

size_t kvb_page_compact_workspace(const kvb_pages* p) {
    if (kvbh::check_pages("page_compact", p)) return 0;
    return (64 + 3 * size_t(p->n_pages)) * 4;
}

kvb_status kvb_page_compact(const kvb_pages* p, int n_pools, int32_t* n_live, void* workspace, size_t workspace_bytes,
                            void* stream) {
    if (kvb_status st = check_layers("page_compact", p, n_pools)) return st;
    if (!n_live || !workspace) return fail(KVB_EINVAL, "page_compact: null argument");
    const size_t need = kvb_page_compact_workspace(p);
    if (workspace_bytes < need) return fail(KVB_EINVAL, "page_compact: workspace of %zu bytes, need %zu", workspace_bytes, need);
    if (!aligned(workspace, 256)) return fail(KVB_EINVAL, "page_compact: workspace needs 256-byte alignment");
    const kvb::PagesView v = kvbh::view_of(p);
    int32_t* b = static_cast<int32_t*>(workspace);
    const kvb::CompactWork w{b, b + 64, b + 64 + p->n_pages, b + 64 + 2 * p->n_pages};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kvb_status st = launch_chained("page_compact plan", kvb::compact_plan_kernel, 1, page_block(p), 0, s, v, w)) return st;
    for (int i = 0; i < n_pools; ++i)
        if (kvb_status st = launch_chained("page_compact move", kvb::compact_move_kernel, 148 * 16, kvb::PG_COPY_THREADS, 0, s,
                                           kvbh::view_of(p + i), w, n_live, i + 1 == n_pools))
            return st;
    return KVB_OK;
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_pages)
