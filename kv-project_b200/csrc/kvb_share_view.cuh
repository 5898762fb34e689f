// kvb_share_view.cuh - which pages the sequences of a call share, as kernels read it (kvb_page_share of include/kvb.h).
#pragma once

#include "kvb_pages_view.cuh"

namespace kvb {

constexpr int PS_LEVELS = 4;                  // segments that may cover a sequence
constexpr int PS_MAX_SEQS = 1024;             // sequences of a plan (ten bits each in its sort key)

struct SharedSegment {
    int first, members, start, end, level;    // members order[first ..], tokens [start, end)
};

// plan: order (n), own (n), depth (n), segments (n, 5), count.  It is data of the caller's: whatever it holds, no address
// is formed from it that is not checked here.
struct SharedView {
    const int32_t* plan;
    const int32_t* slots;                     // of the n sequences
    int n, page, max_tokens, levels;          // levels: of the partials' buffer, at most PS_LEVELS

    __device__ __forceinline__ int segment_count() const { return min(max(plan[8 * int64_t(n)], 0), n); }
    __device__ __forceinline__ SharedSegment segment(int i) const {
        const int32_t* s = plan + 3 * int64_t(n) + 5 * int64_t(i);
        const SharedSegment g{s[0], s[1], s[2], s[3], s[4]};
        if (g.first >= 0 && g.members > 0 && g.members <= n && g.first <= n - g.members && g.start >= 0 && g.start < g.end &&
            g.end <= max_tokens && (g.start & (page - 1)) == 0 && unsigned(g.level) < unsigned(levels))
            return g;
        raise_status(KVB_DEV_BOUNDS);
        return SharedSegment{0, 1, 0, 0, 0};
    }
    __device__ __forceinline__ int member(const SharedSegment& g, int k) const {
        const int i = plan[g.first + k];
        if (unsigned(i) < unsigned(n)) return i;
        raise_status(KVB_DEV_BOUNDS);
        return 0;
    }
    // the slot whose pages are read for the segment (all members hold the same), or -1
    __device__ __forceinline__ int slot_of(const SharedSegment& g, int n_slots) const {
        const int slot = slots[member(g, 0)];
        return unsigned(slot) < unsigned(n_slots) ? slot : -1;
    }
    __device__ __forceinline__ int own_of(int i, int len) const { return min(max(plan[n + i], 0), len) & ~(page - 1); }
    __device__ __forceinline__ int depth_of(int i) const { return min(max(plan[2 * int64_t(n) + i], 0), levels); }
    __device__ __forceinline__ int length_of(int i, const PagesView& P) const {
        const int slot = slots[i];
        return unsigned(slot) < unsigned(P.n_slots) ? min(max(P.lens[slot], 0), max_tokens) : 0;
    }
};

}  // namespace kvb
