// kvb_api_prefill.cu - kvb_prefill_attention (include/kvb.h): validation and launch of the causal attention of packed
// prompts (kvb_prefill.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "kvb_host.h"
#include "kvb_common.cuh"
#include "kvb_prefill.cuh"

namespace {

constexpr int kMaxCtas = 512;                                  // that run at a time
constexpr size_t kCountBytes = 2 * kMaxCtas * 4 * 4;          // per piece and warp

int prefill_ctas() { return std::min(resolve_ctas(0) * kvb::PF_CTAS_PER_SM, kMaxCtas); }

template <typename T, int D>
kvb_status launch(const kvb::PrefillParams& a, cudaStream_t s) {
    constexpr int SM = kvb::PfShape<D>::SMEM;
    const auto kern = kvb::prefill_kernel<T, D>;
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = kvbh::allow_smem("prefill_attention", reinterpret_cast<const void*>(kern), SM, done)) return st;
    // at most so many items and pieces; a CTA that finds none leaves at once
    const int64_t items = a.Hkv * (a.nq / a.tt + a.n) + (a.part ? 2 * a.ctas : 0);
    if (items > INT32_MAX) return fail(KVB_EINVAL, "prefill_attention: (query rows + sequences) x KV heads too many");
    kern<<<unsigned(items), kvb::PF_THREADS, SM, s>>>(a);
    return launch_check("prefill_attention");
}

}  // namespace

extern "C" {

size_t kvb_prefill_workspace(int d) {
    return d == 64 || d == 128 ? kCountBytes + size_t(prefill_ctas()) * 2 * (d + 2) * kvb::PF_ROWS * 4 : 0;
}

kvb_status kvb_prefill_attention(const void* q, const void* k, const void* v, int dtype, int64_t nq, int64_t nk, int Hq,
                                 int Hkv, int d, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head,
                                 int64_t v_row, int64_t v_head, const int32_t* cu_q, const int32_t* cu_k, int n,
                                 float scaling, void* out, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || nq < 0 || nk < 0 || nq > INT32_MAX || nk > INT32_MAX)
        return fail(KVB_EINVAL, "prefill_attention: n >= 0 and row counts in [0, 2^31)");
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || Hq > 65535)
        return fail(KVB_EINVAL, "prefill_attention: Hq a multiple of Hkv, at most 65535");
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "prefill_attention: float16 or bfloat16");
    if (d != 64 && d != 128) return fail(KVB_EUNSUPPORTED, "prefill_attention: d 64 or 128");
    if (Hq / Hkv > 128) return fail(KVB_EUNSUPPORTED, "prefill_attention: at most 128 query heads per KV head");
    if (n == 0 || nq == 0) return KVB_OK;
    if (!q || (!k && nk) || (!v && nk) || !cu_q || !cu_k || !out) return fail(KVB_EINVAL, "prefill_attention: null argument");
    for (int64_t st : {q_row, q_head, k_row, k_head, v_row, v_head})
        if (st < 0 || st % 8 != 0) return fail(KVB_EINVAL, "prefill_attention: row and head strides multiples of 8 elements");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 32) || !aligned(lse, 4))
        return fail(KVB_EINVAL, "prefill_attention: q, k and v need 16-byte alignment, out 32-byte, lse 4-byte");
    if (!std::isfinite(scaling)) return fail(KVB_EINVAL, "prefill_attention: scaling must be finite");
    if (workspace && (workspace_bytes < kvb_prefill_workspace(d) || !aligned(workspace, 256)))
        return fail(KVB_EINVAL, "prefill_attention: workspace of %zu bytes, 256-byte aligned (or none)", kvb_prefill_workspace(d));
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (kvb_status st = kvbh::cuda_check(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture), "prefill_attention")) return st;
    if (capture != cudaStreamCaptureStatusNone)      // a replay would repeat this call's number, which tells leftovers from arrivals
        return fail(KVB_EUNSUPPORTED, "prefill_attention: not in a stream capture");
    kvb::PrefillParams a{};
    a.count = static_cast<uint32_t*>(workspace);
    a.part = workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + kCountBytes) : nullptr;
    a.rep = Hq / Hkv;
    a.tt = kvb::PF_ROWS / a.rep;
    a.by_rep = 65536 / a.rep + 1;
    a.ctas = prefill_ctas();
    static std::atomic<uint32_t> calls{0};
    a.call = calls.fetch_add(1) % 0xfffff + 1;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_row = q_row;
    a.q_head = q_head;
    a.k_row = k_row;
    a.k_head = k_head;
    a.v_row = v_row;
    a.v_head = v_head;
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.nq = nq;
    a.nk = nk;
    a.n = n;
    a.Hq = Hq;
    a.Hkv = Hkv;
    // a scaling of zero becomes one too small to matter, so that -inf stays -inf
    a.lam = std::max(std::fabs(scaling) * 1.44269504088896340736f, 1e-37f);
    a.negate = scaling < 0;
    a.out = out;
    a.lse = lse;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == KVB_BF16) return d == 128 ? launch<__nv_bfloat16, 128>(a, s) : launch<__nv_bfloat16, 64>(a, s);
    return d == 128 ? launch<__half, 128>(a, s) : launch<__half, 64>(a, s);
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_prefill)
