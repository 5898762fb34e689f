// kvb_api_shared.cu - kvb_page_share and kvb_page_attend_shared (include/kvb.h): validation and launches of the search for
// shared pages (kvb_share.cuh) and of the attention that computes them once for all their sequences (kvb_paged_decode.cuh).
#include "kvb_paged_host.cuh"
#include "kvb_share.cuh"
#include "kvb_shared_tc.cuh"

namespace {

// Segments cover a sequence at most this often: each has two or more parts below it.
int levels_of(int n) { return std::min(kvb::PS_LEVELS, std::max(n - 1, 0)); }

// Items of the sequences' own tokens up to which the eight warps of a CTA work on one together (PD_OWN); above, each on its own
// (PD_LONE).  attend_shared behind 640 shared tokens with 60, 1200 and 4000 of their own: 32 items 26, 30 and 34 us together,
// 26, 34 and 50 alone; 128 items 28, 38 and 57, 28, 39 and 58; 192 items 34, 44 and 69, 29, 41 and 68; 512 items 43, 75 and 126,
// 32, 63 and 121.
constexpr int64_t kTogether = 160;

int shared_ctas() { return std::min(resolve_ctas(0), kvb::PD_MAX_CTAS); }

constexpr int64_t kCuts = (kvb::PD_MAX_CTAS * sizeof(kvb::CmCut<kvb::SharedItem>) + 255) / 256 * 256;

// The workspace: counters; what is cut; partials of cut items, first of the segments, then of the sequences' own tokens (the former are
// joined by then); the rows' parts by level.
int64_t level_offset(int d) {
    const int64_t segments = int64_t(2) * shared_ctas() * 2 * kvb::CM_ROWS * (d + 3), own = int64_t(2) * shared_ctas() * 8 * 16 * (d + 4);
    return kvbh::kCountBytes + kCuts + (std::max(segments, own) * 4 + 255) / 256 * 256;
}

template <typename T, int D>
kvb_status launch_segments(const kvb::SharedTcParams& a, cudaStream_t s) {
    constexpr int SM = kvb::StShape<D>::SMEM;
    const auto kern = kvb::shared_pages_kernel<T, D>;
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = kvbh::allow_smem("page_attend_shared", reinterpret_cast<const void*>(kern), SM, done)) return st;
    if (kvb_status st = launch_chained("page_attend_shared", kern, unsigned(a.ctas), 32 * kvb::ST_WARPS, SM, s, a)) return st;
    return launch_chained("page_attend_shared join", kvb::shared_join_kernel<D>, unsigned(4 * a.ctas), 32 * kvb::CJ_WARPS, 0, s, a);
}

kvb_status launch_share(const kvb_pages* p, const int32_t* slots, int n, int32_t* plan, int32_t* kept, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_share", p)) return st;
    if (!plan || (n > 0 && !slots)) return fail(KVB_EINVAL, "page_share: null argument");
    if (n < 0 || n > kvb::PS_MAX_SEQS) return fail(KVB_EINVAL, "page_share: 0 <= n <= %d sequences a call", kvb::PS_MAX_SEQS);
    static std::atomic<uint64_t> done{0};
    if (kvb_status st = kvbh::allow_smem("page_share", reinterpret_cast<const void*>(kvb::page_share_kernel), int(sizeof(kvb::ShareSmem)), done))
        return st;
    return launch_chained("page_share", kvb::page_share_kernel, 1, kvb::PS_THREADS, sizeof(kvb::ShareSmem), static_cast<cudaStream_t>(stream),
                          kvbh::view_of(p), slots, n, plan, kept);
}

}  // namespace

extern "C" {

kvb_status kvb_page_share(const kvb_pages* p, const int32_t* slots, int n, int32_t* plan, void* stream) {
    return launch_share(p, slots, n, plan, nullptr, stream);
}

kvb_status kvb_page_share_kept(const kvb_pages* p, const int32_t* slots, int n, int32_t* plan, int32_t* kept, void* stream) {
    if (n > 0 && !kept) return fail(KVB_EINVAL, "page_share: null argument");
    return launch_share(p, slots, n, plan, kept, stream);
}

size_t kvb_page_attend_shared_workspace(const kvb_pages* p, int n, int Hq, int Tq) {
    if (kvbh::check_pages("page_attend_shared", p) || n < 0 || n > kvb::PS_MAX_SEQS || Hq <= 0 || Tq <= 0) return 0;
    return size_t(level_offset(p->d)) + size_t(levels_of(n)) * n * Hq * Tq * (p->d + 2) * 4;
}

kvb_status kvb_page_attend_shared(const kvb_pages* p, const void* q, int dtype, int Hq, int Tq, const int32_t* slots, int n,
                                  const int32_t* plan, float scaling, void* out, float* lse, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    if (kvb_status st = kvbh::check_pages("page_attend_shared", p)) return st;
    if (n > 0 && !plan) return fail(KVB_EINVAL, "page_attend_shared: null argument");
    if (n > kvb::PS_MAX_SEQS) return fail(KVB_EINVAL, "page_attend_shared: n <= %d sequences a call", kvb::PS_MAX_SEQS);
    kvb::PagedDecodeParams a{};
    if (kvb_status st = kvbh::paged_params("page_attend_shared", p, q, dtype, Hq, Tq, slots, n, scaling, out, lse, workspace, a)) return st;
    if (n == 0) return KVB_OK;
    // The segments' places fit 32 bits (launches of own tokens are divided until theirs do).  One of m >= 2 members has at most
    // m (rep Tq / 256 + 1 / 2) groups of rows, so that each member counts with its segments' places, at most those of a table row cut
    // in PS_LEVELS, times rep Tq / 256 + 1 / 2.
    const int64_t rows_of_kv = int64_t(n) * a.rep * Tq, groups = (rows_of_kv + int64_t(n) * kvb::CM_ROWS + 2 * kvb::CM_ROWS - 1) / (2 * kvb::CM_ROWS);
    const int64_t places = int64_t(p->max_blocks) * p->page / kvb::CM_KEYS + kvb::PS_LEVELS * (1 + kvb::CM_FIXED);
    if (rows_of_kv > INT32_MAX - 65536 || places > INT32_MAX / p->Hkv / groups)
        return fail(KVB_EUNSUPPORTED, "page_attend_shared: tokens of a table row times query rows too many for one call");
    if (workspace_bytes < kvb_page_attend_shared_workspace(p, n, Hq, Tq) || !aligned(workspace, 256))
        return fail(KVB_EINVAL, "page_attend_shared: workspace of %zu bytes, 256-byte aligned", kvb_page_attend_shared_workspace(p, n, Hq, Tq));
    if (kvb_status st = kvbh::paged_maps("page_attend_shared", p, a)) return st;
    kvbh::paged_workspace(workspace, a);
    a.whole_words = aligned(out, 16);
    a.early = n > 1;
    a.shared = kvb::SharedView{plan, slots, n, p->page, p->max_blocks * p->page, levels_of(n)};
    a.rows = int64_t(n) * Tq * Hq;
    a.level_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + level_offset(p->d));
    a.level_ml = a.level_o + levels_of(n) * a.rows * p->d;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (n > 1) {
        kvb::SharedTcParams b{};
        if (kvb_status st = kvbh::make_map("page_attend_shared", &b.tm_k, p, p->kc, kvb::CM_KEYS, false)) return st;
        if (kvb_status st = kvbh::make_map("page_attend_shared", &b.tm_v, p, p->vc, kvb::CM_KEYS, false)) return st;
        b.P = a.P;
        b.shared = a.shared;
        b.q = q;
        b.Hq = Hq;
        b.Tq = Tq;
        b.rep = a.rep;
        b.by_rep = a.by_rep;
        b.by_rows = kvbh::reciprocal(a.rep * Tq);
        b.page_log2 = a.page_log2;
        // a scaling of zero becomes one too small to matter, so that -inf stays -inf
        b.lam = std::max(std::fabs(a.lam), 1e-37f);
        b.negate = scaling < 0;
        b.rows = a.rows;
        b.level_o = a.level_o;
        b.level_ml = a.level_ml;
        b.cuts = static_cast<char*>(workspace) + kvbh::kCountBytes;
        b.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kvbh::kCountBytes + kCuts);
        b.ctas = shared_ctas();
        kvb_status st = dtype == KVB_F16 ? p->d == 128 ? launch_segments<__half, 128>(b, s) : launch_segments<__half, 64>(b, s)
                        : p->d == 128    ? launch_segments<__nv_bfloat16, 128>(b, s)
                                         : launch_segments<__nv_bfloat16, 64>(b, s);
        if (st) return st;
    }
    // items of the sequences' own tokens: up to kTogether the eight warps of a CTA work on one together, above each on its own
    const int64_t rows = int64_t(a.rep) * Tq, items = (rows <= 8 ? 1 : (rows + 15) / 16) * n * p->Hkv;
    return items <= kTogether ? kvbh::paged_launch_any<kvb::PD_OWN>("page_attend_shared", a, dtype, rows, s)
                              : kvbh::paged_launch_any<kvb::PD_LONE>("page_attend_shared", a, dtype, rows, s);
}

}  // extern "C"

KVB_STATUS_WORDS(status_words_shared)
