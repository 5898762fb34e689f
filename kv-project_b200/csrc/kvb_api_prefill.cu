// kvb_api_prefill.cu - kvb_prefill_attention (include/kvb.h): validation and launch of the causal attention of
// packed prompts.
#include <cuda_runtime.h>

#include "kvb_host.h"
#include "kvb_common.cuh"
#include "kvb_rowattn.cuh"

namespace {

template <typename T>
void launch(const kvb::PrefillParams& a, int d, cudaStream_t s) {
    const dim3 grid(unsigned((a.nq + kvb::RA_WARPS - 1) / kvb::RA_WARPS), unsigned(a.Hq));
    if (d == 64) kvb::prefill_rows_kernel<T, 64><<<grid, kvb::RA_WARPS * 32, 0, s>>>(a);
    else kvb::prefill_rows_kernel<T, 128><<<grid, kvb::RA_WARPS * 32, 0, s>>>(a);
}

}  // namespace

extern "C" {

kvb_status kvb_prefill_attention(const void* q, const void* k, const void* v, int dtype, int64_t nq, int64_t nk, int Hq,
                                 int Hkv, int d, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                                 int64_t v_row, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, int n,
                                 float scaling, void* out, float* lse, void* stream) {
    if (n < 0 || nq < 0 || nk < 0 || nq > INT32_MAX || nk > INT32_MAX)
        return fail(KVB_EINVAL, "prefill_attention: n >= 0 and row counts in [0, 2^31)");
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || Hq > 65535)
        return fail(KVB_EINVAL, "prefill_attention: Hq a multiple of Hkv, at most 65535");
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "prefill_attention: float16 or bfloat16");
    if (d != 64 && d != 128) return fail(KVB_EUNSUPPORTED, "prefill_attention: d 64 or 128");
    if (n == 0 || nq == 0) return KVB_OK;
    if (!q || (!k && nk) || (!v && nk) || !cu_q || !cu_k || !out) return fail(KVB_EINVAL, "prefill_attention: null argument");
    for (int64_t st : {q_row, q_head, k_row, k_head, v_row, v_head})
        if (st < 0 || st % 8 != 0) return fail(KVB_EINVAL, "prefill_attention: row and head strides multiples of 8 elements");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
        return fail(KVB_EINVAL, "prefill_attention: q, k, v and out need 16-byte alignment");
    const kvb::PrefillParams a{q, k, v, q_row, q_head, k_row, k_head, v_row, v_head, cu_q, cu_k, nq, nk, n, Hq, Hkv,
                               scaling * 1.44269504088896340736f, out, lse};
    if (dtype == KVB_F16) launch<__half>(a, d, static_cast<cudaStream_t>(stream));
    else launch<__nv_bfloat16>(a, d, static_cast<cudaStream_t>(stream));
    return launch_check("prefill_attention");
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_prefill)
