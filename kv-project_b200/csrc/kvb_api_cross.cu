// kvb_api_cross.cu - kvb_cross_attention (include/kvb.h): validation, tensor maps and launch of the attention of packed
// queries to keys of another length (kvb_cross.cuh).
#include "kvb_paged_host.cuh"
#include "kvb_cross_tc.cuh"

namespace {

// Query rows (tokens x heads of a KV head) of a sequence, on average, up to which cross_few_kernel is taken: its tile.  24
// sequences of 1500 keys, 8 KV heads of 128 channels: 16 rows 40 us, cross_many_kernel 45; 24 rows 59 and 45.  48 of 4000 keys: 135
// and 159, 255 and 160.  6 of 1500: 20.5 and 21.4, 22.6 and 21.4.
constexpr int kFewRows = 16;

constexpr size_t kCrossCounts = size_t(kvb::PD_MAX_CTAS) * kvb::CR_WARPS * 4;
constexpr size_t kCrossCuts = kvb::PD_MAX_CTAS * sizeof(kvb::CmCut<kvb::CrossItem>);
static_assert(kCrossCuts % 256 == 0, "the partials begin on a 256-byte boundary");

// Rows (nk, heads, d) with their strides as (d, heads, rows), box 64 channels x 1 x `rows`, 128-byte swizzle.  A head stride of
// zero (one head for all) is a map of one head.
kvb_status cross_map(CUtensorMap* m, const void* x, const void* other, int dtype, int d, int64_t nk, int Hkv, int64_t row, int64_t head, int rows) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return fail(KVB_ECUDA, "cross_attention: cuTensorMapEncodeTiled unavailable");
    const int heads = Hkv > 1 && head > 0 ? Hkv : 1;
    const cuuint64_t dims[3] = {cuuint64_t(d), cuuint64_t(heads), cuuint64_t(std::max<int64_t>(nk, 1))};
    const cuuint64_t strides[2] = {cuuint64_t(heads > 1 ? head : d) * 2, cuuint64_t(nk > 1 ? row : d) * 2};
    const cuuint32_t box[3] = {64, 1, cuuint32_t(rows)}, estr[3] = {1, 1, 1};
    const CUresult r = fn(m, dtype == KVB_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                          const_cast<void*>(nk ? x : other), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? KVB_OK : fail(KVB_EUNSUPPORTED, "cross_attention: no tensor map for keys or values of these strides");
}

int cross_ctas() { return std::min(resolve_ctas(0), kvb::PD_MAX_CTAS); }

template <typename T, int D, bool MANY>
kvb_status launch(kvb::CrossParams a, cudaStream_t s) {
    constexpr int SM = MANY ? kvb::CrossTcShape<D>::SMEM : kvb::CrShape<D>::SMEM, THREADS = 32 * (MANY ? kvb::CM_WARPS : kvb::CR_WARPS);
    const auto kern = MANY ? kvb::cross_many_kernel<T, D> : kvb::cross_few_kernel<T, D>;
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = kvbh::allow_smem("cross_attention", reinterpret_cast<const void*>(kern), SM, done)) return st;
    const unsigned grid = unsigned(cross_ctas());
    const int n = a.n;
    for (int i = 0; i < n; i += kvb::CR_MAX_SEQS) {
        a.n = std::min(n - i, kvb::CR_MAX_SEQS);
        if (kvb_status st = launch_chained("cross_attention", kern, grid, THREADS, SM, s, a)) return st;
        if (MANY)
            if (kvb_status st = launch_chained("cross_attention join", kvb::cross_join_kernel<T, D>, 4 * grid, 32 * kvb::CJ_WARPS, 0, s, a)) return st;
        a.cu_q += kvb::CR_MAX_SEQS;
        a.cu_k += kvb::CR_MAX_SEQS;
    }
    return KVB_OK;
}

template <bool MANY>
kvb_status launch_any(const kvb::CrossParams& a, int dtype, int d, cudaStream_t s) {
    if (dtype == KVB_BF16) return d == 128 ? launch<__nv_bfloat16, 128, MANY>(a, s) : launch<__nv_bfloat16, 64, MANY>(a, s);
    return d == 128 ? launch<__half, 128, MANY>(a, s) : launch<__half, 64, MANY>(a, s);
}

}  // namespace

extern "C" {

size_t kvb_cross_workspace(int d) {
    // two partials a CTA: of 2 x 128 rows (cross_many_kernel), of 16 (cross_few_kernel)
    return d == 64 || d == 128 ? kCrossCounts + kCrossCuts + size_t(2) * cross_ctas() * 2 * kvb::CM_ROWS * (d + 3) * 4 : 0;
}

kvb_status kvb_cross_attention(const void* q, const void* k, const void* v, int dtype, int64_t nq, int64_t nk, int Hq, int Hkv,
                               int d, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                               const int32_t* cu_q, const int32_t* cu_k, int n, float scaling, void* out, float* lse,
                               void* workspace, size_t workspace_bytes, void* stream) {
    if (n < 0 || nq < 0 || nk < 0 || nq > INT32_MAX - 65536 || nk > INT32_MAX - 65536)
        return fail(KVB_EINVAL, "cross_attention: n >= 0 and row counts in [0, 2^31 - 2^16]");
    if (Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || Hq > 65535)
        return fail(KVB_EINVAL, "cross_attention: Hq a multiple of Hkv, at most 65535");
    if (dtype != KVB_F16 && dtype != KVB_BF16) return fail(KVB_EUNSUPPORTED, "cross_attention: float16 or bfloat16");
    if (d != 64 && d != 128) return fail(KVB_EUNSUPPORTED, "cross_attention: d 64 or 128");
    if (!std::isfinite(scaling)) return fail(KVB_EINVAL, "cross_attention: scaling must be finite");
    if (n == 0 || nq == 0) return KVB_OK;
    if (!q || (!k && nk) || (!v && nk) || !cu_q || !cu_k || !out || !workspace) return fail(KVB_EINVAL, "cross_attention: null argument");
    // strides of an extent of one address nothing
    if (nq == 1) q_row = 0;
    if (Hq == 1) q_head = 0;
    if (nk <= 1) k_row = v_row = 0;
    if (Hkv == 1) k_head = v_head = 0;
    for (int64_t st : {q_row, q_head, k_row, k_head, v_row, v_head})
        if (st < 0 || st % 8 != 0 || st >= int64_t(1) << 38) return fail(KVB_EINVAL, "cross_attention: row and head strides multiples of 8 elements");
    if (nk > 1 && (k_row == 0 || v_row == 0)) return fail(KVB_EUNSUPPORTED, "cross_attention: key and value rows of their own (row strides above 0)");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 32) || !aligned(lse, 4))
        return fail(KVB_EINVAL, "cross_attention: q, k and v need 16-byte alignment, out 32-byte, lse 4-byte");
    kvb::CrossParams a{};
    a.rep = Hq / Hkv;
    a.ctas = cross_ctas();
    const bool many = nq * a.rep > int64_t(kFewRows) * n;
    const int keys = many ? kvb::CM_KEYS : 2048 / d, rows = many ? 2 * kvb::CM_ROWS : kvb::CR_ROWS;
    // One sequence alone has work of 32 bits.  How the rows of several are dealt to them only the kernels see: they leave out a
    // sequence, or the up to CR_MAX_SEQS of a launch, whose work is more.
    const int64_t units = nk / keys + 2 + kvb::PD_FIXED, groups = (nq * a.rep + rows - 1) / rows;
    if (nq * a.rep > INT32_MAX - 65536 || (n == 1 && units > INT32_MAX / Hkv / groups))
        return fail(KVB_EUNSUPPORTED, "cross_attention: query rows times keys too many for one call");
    if (workspace_bytes < kvb_cross_workspace(d) || !aligned(workspace, 256))
        return fail(KVB_EINVAL, "cross_attention: workspace of %zu bytes, 256-byte aligned", kvb_cross_workspace(d));
    if (kvb_status st = cross_map(&a.tm_k, k, q, dtype, d, nk, Hkv, k_row, k_head, keys)) return st;
    if (kvb_status st = cross_map(&a.tm_v, v, q, dtype, d, nk, Hkv, v_row, v_head, keys)) return st;
    a.q = q;
    a.q_row = q_row;
    a.q_head = q_head;
    a.cu_q = cu_q;
    a.cu_k = cu_k;
    a.nq = nq;
    a.nk = nk;
    a.n = n;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.k_heads = k_head > 0;
    a.v_heads = v_head > 0;
    a.by_rep = kvbh::reciprocal(a.rep);
    a.lam = scaling * 1.44269504088896340736f;
    a.negate = scaling < 0;
    // a scaling of zero becomes one too small to matter, so that -inf stays -inf
    if (many) a.lam = std::max(std::fabs(a.lam), 1e-37f);
    a.out = out;
    a.lse = lse;
    a.count = static_cast<uint32_t*>(workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCrossCounts + kCrossCuts);
    a.cuts = static_cast<char*>(workspace) + kCrossCounts;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return many ? launch_any<true>(a, dtype, d, s) : launch_any<false>(a, dtype, d, s);
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_cross)
