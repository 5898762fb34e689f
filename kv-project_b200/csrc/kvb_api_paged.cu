// kvb_api_paged.cu - kvb_page_attend (include/kvb.h): validation and launch of the attention over the 8-bit
// paged cache.
#include <cuda_runtime.h>

#include "kvb_host.h"
#include "kvb_pages_host.h"
#include "kvb_rowattn.cuh"

namespace {

template <typename T>
void launch(const kvb::PagedAttendParams& a, cudaStream_t s) {
    const dim3 grid(unsigned((int64_t(a.n) * a.Tq + kvb::RA_WARPS - 1) / kvb::RA_WARPS), unsigned(a.Hq));
    if (a.P.d == 64) kvb::paged_rows_kernel<T, 64><<<grid, kvb::RA_WARPS * 32, 0, s>>>(a);
    else kvb::paged_rows_kernel<T, 128><<<grid, kvb::RA_WARPS * 32, 0, s>>>(a);
}

}  // namespace

extern "C" {

size_t kvb_page_attend_workspace(const kvb_pages* p, int n, int Hq, int Tq) {
    if (kvbh::check_pages("page_attend", p) || n < 0 || Hq <= 0 || Tq <= 0) return 0;
    return 256;
}

kvb_status kvb_page_attend(const kvb_pages* p, const void* q, int dtype, int Hq, int Tq, const int32_t* slots, int n,
                           float scaling, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_attend", p)) return st;
    if (n > 0 && (!q || !slots || !out || !workspace)) return fail(KVB_EINVAL, "page_attend: null argument");
    if (Hq <= 0 || Hq % p->Hkv != 0 || Hq > 65535) return fail(KVB_EINVAL, "page_attend: Hq a multiple of Hkv, at most 65535");
    if (n < 0 || Tq <= 0) return fail(KVB_EINVAL, "page_attend: n >= 0, Tq >= 1");
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "page_attend: q of float16 or bfloat16");
    if (workspace_bytes < kvb_page_attend_workspace(p, n, Hq, Tq) || !aligned(workspace, 256))
        return fail(KVB_EINVAL, "page_attend: workspace of %zu bytes, 256-byte aligned", kvb_page_attend_workspace(p, n, Hq, Tq));
    if (n == 0) return KVB_OK;
    const kvb::PagedAttendParams a{kvbh::view_of(p), q, slots, n, Hq, Tq, scaling * 1.44269504088896340736f, out, lse};
    if (dtype == KVB_F16) launch<__half>(a, static_cast<cudaStream_t>(stream));
    else launch<__nv_bfloat16>(a, static_cast<cudaStream_t>(stream));
    return launch_check("page_attend");
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_paged)
