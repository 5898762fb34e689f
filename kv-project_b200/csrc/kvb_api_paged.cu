// kvb_api_paged.cu - kvb_page_attend (include/kvb.h): validation and launch of the attention over the 8-bit paged cache
// (kvb_paged_decode.cuh).
#include "kvb_paged_host.cuh"

extern "C" {

size_t kvb_page_attend_workspace(const kvb_pages* p, int n, int Hq, int Tq) {
    if (kvbh::check_pages("page_attend", p) || n < 0 || Hq <= 0 || Tq <= 0) return 0;
    return kvbh::paged_part_bytes(p->d);
}

kvb_status kvb_page_attend(const kvb_pages* p, const void* q, int dtype, int Hq, int Tq, const int32_t* slots, int n,
                           float scaling, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_attend", p)) return st;
    kvb::PagedDecodeParams a{};
    if (kvb_status st = kvbh::paged_params("page_attend", p, q, dtype, Hq, Tq, slots, n, scaling, out, lse, workspace, a)) return st;
    if (n == 0) return KVB_OK;
    if (workspace_bytes < kvb_page_attend_workspace(p, n, Hq, Tq) || !aligned(workspace, 256))
        return fail(KVB_EINVAL, "page_attend: workspace of %zu bytes, 256-byte aligned", kvb_page_attend_workspace(p, n, Hq, Tq));
    if (kvb_status st = kvbh::paged_maps("page_attend", p, a)) return st;
    kvbh::paged_workspace(workspace, a);
    return kvbh::paged_launch_any<kvb::PD_ALL>("page_attend", a, dtype, int64_t(a.rep) * Tq, static_cast<cudaStream_t>(stream));
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_paged)
