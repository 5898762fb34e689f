// kvb_share.cuh - which leading pages the sequences of a call share.
//
// In up to PS_LEVELS rounds: the sequences of one class (at first all) that hold the same page in the block behind their
// common ones form a class of the next round, and a class of two or more gets a segment, from the blocks before to the last
// block that all of its members hold in full.  A class's number is its first member, so the result does not depend on timing.
//
// One block: the classes of a round come from a hash table in shared memory (class and page, the least index and the count by
// atomics), the common blocks of a member and its class's first by eight lanes that compare their rows of the table, the order at
// the end from one sort of (class numbers of all rounds, index), 10 bits each.
//
// The floor is the rows of the table read once, n blocks 4 bytes; the time is a chain of latencies (a round: insert, look
// up, compare, minimum), because everything after a round depends on it.  480 sequences with 61 segments on four levels take 27.6
// us, 8 sequences 6; with a whole warp for each comparison the former took 41.
#pragma once

#include <climits>

#include "kvb_share_view.cuh"

namespace kvb {

constexpr int PS_THREADS = 1024;
constexpr int PS_HASH = 2 * PS_MAX_SEQS;      // entries: at most half of them are taken
constexpr int PS_UNROLL = 8;                  // entries of either row that a lane has in flight

struct ShareSmem {
    unsigned long long key[PS_HASH];          // class << 32 | page
    int least[PS_HASH], count[PS_HASH];
    unsigned long long sort[PS_MAX_SEQS];
    int slot[PS_MAX_SEQS], full[PS_MAX_SEQS], end[PS_MAX_SEQS], leader[PS_MAX_SEQS], size[PS_MAX_SEQS], common[PS_MAX_SEQS], place[PS_MAX_SEQS];
    int seg_size[PS_LEVELS][PS_MAX_SEQS], seg_start[PS_LEVELS][PS_MAX_SEQS], seg_end[PS_LEVELS][PS_MAX_SEQS];
    uint32_t heads[PS_LEVELS][32];            // a bit per place that is a segment's first
    int before[PS_LEVELS][32], total[PS_LEVELS];
};

__global__ void __launch_bounds__(PS_THREADS, 1) page_share_kernel(const __grid_constant__ PagesView P, const int32_t* slots, int n,
                                                                   int32_t* plan, int32_t* kept) {
    extern __shared__ __align__(16) uint8_t ps_raw[];
    ShareSmem& S = *reinterpret_cast<ShareSmem*>(ps_raw);
    constexpr unsigned long long EMPTY = ~0ull;
    const int i = threadIdx.x, warp = i >> 5, lane = i & 31;
    chain_kernels();
    int slot = -1, full = 0, end = 0, cls = 0, depth = 0;
    bool alive = i < n;
    unsigned long long path = 0;
    if (i < n) {
        slot = slots[i];
        if (kept) kept[i] = slot;
        if (unsigned(slot) < unsigned(P.n_slots)) full = min(max(P.lens[slot], 0) >> page_shift(P.page), P.max_blocks);
        else raise_status(KVB_DEV_BOUNDS);
    }
    S.slot[i] = slot;
    S.full[i] = full;
    S.end[i] = 0;
#pragma unroll
    for (int l = 0; l < PS_LEVELS; ++l) S.seg_size[l][i] = 0;
    if (i < PS_LEVELS * 32) S.heads[i >> 5][lane] = 0;

    bool more = true;
    for (int level = 0; level < PS_LEVELS; ++level) {
        int leader = i, size = 1;
        if (more) {
            for (int e = i; e < PS_HASH; e += PS_THREADS) {
                S.key[e] = EMPTY;
                S.least[e] = PS_MAX_SEQS;
                S.count[e] = 0;
            }
            __syncthreads();
            int at = -1;
            if (alive && end < full) {
                const int id = P.table[int64_t(slot) * P.max_blocks + end];
                if (id >= 0 && id < P.n_pages) {
                    const unsigned long long key = (unsigned long long)(cls) << 32 | uint32_t(id);
                    at = int((uint32_t(id) * 2654435761u ^ uint32_t(cls) * 40503u) >> 16) & (PS_HASH - 1);
                    for (int probes = 0; probes < PS_HASH; ++probes) {           // an empty place is found before
                        const unsigned long long was = atomicCAS(&S.key[at], EMPTY, key);
                        if (was == EMPTY || was == key) break;
                        at = (at + 1) & (PS_HASH - 1);
                    }
                    atomicMin(&S.least[at], i);
                    atomicAdd(&S.count[at], 1);
                }
            }
            __syncthreads();
            if (at >= 0) leader = S.least[at], size = S.count[at];
            S.leader[i] = leader;
            S.size[i] = size;
            S.common[i] = full;
            more = __syncthreads_or(size > 1);
        }
        if (more) {
            // blocks that a member and its class's first have in common: eight lanes a member, four members a warp, so that the loads
            // of all 480 members of a call are on their way in four rounds (a warp a member: 41 us a call, 15 rounds of latency)
            for (int m0 = warp * 4; m0 < n; m0 += PS_THREADS / 8) {
                const int mb = min(m0 + (lane >> 3), n - 1), first = S.leader[mb], stop = min(S.full[mb], S.full[first]);
                const bool compares = m0 + (lane >> 3) < n && S.size[mb] > 1 && first != mb;
                const int32_t* a = P.table + int64_t(compares ? S.slot[mb] : 0) * P.max_blocks;
                const int32_t* b = P.table + int64_t(compares ? S.slot[first] : 0) * P.max_blocks;
                int same = stop, b0 = S.end[mb] + 1;
                bool active = compares && b0 < stop;
                while (__any_sync(0xffffffffu, active)) {
                    int ids[PS_UNROLL], others[PS_UNROLL];
#pragma unroll
                    for (int u = 0; u < PS_UNROLL; ++u) {
                        const int x = b0 + 8 * u + (lane & 7);
                        const bool in = active && x < stop;
                        ids[u] = in ? a[x] : 0;
                        others[u] = in ? b[x] : 0;
                    }
                    int differ = INT_MAX;
#pragma unroll
                    for (int u = PS_UNROLL - 1; u >= 0; --u)
                        if (ids[u] != others[u] || ids[u] < 0 || ids[u] >= P.n_pages) differ = b0 + 8 * u + (lane & 7);
                    differ = min(differ, __shfl_xor_sync(0xffffffffu, differ, 1));
                    differ = min(differ, __shfl_xor_sync(0xffffffffu, differ, 2));
                    differ = min(differ, __shfl_xor_sync(0xffffffffu, differ, 4));
                    if (active) {
                        same = min(same, differ);
                        b0 += 8 * PS_UNROLL;
                        active = differ == INT_MAX && b0 < stop;
                    }
                }
                if (compares && (lane & 7) == 0) atomicMin(&S.common[first], same);
            }
            __syncthreads();
            alive = size > 1;
            if (alive) {
                const int to = S.common[leader];
                if (leader == i) S.seg_size[level][i] = size, S.seg_start[level][i] = end, S.seg_end[level][i] = to;
                end = to;
                ++depth;
                S.end[i] = end;
            }
            cls = leader;
            __syncthreads();
        }
        path = path << 10 | uint32_t(leader);
    }

    // ---- order: bitonic sort, one entry a thread
    unsigned long long x = i < n ? path << 10 | uint32_t(i) : EMPTY;
    int entries = 32;
    while (entries < n) entries *= 2;
    for (int k = 2; k <= entries; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            unsigned long long y;
            if (j >= 32) {
                S.sort[i] = x;
                __syncthreads();
                y = S.sort[i ^ j];
                __syncthreads();
            } else {
                y = __shfl_xor_sync(0xffffffffu, x, j);
            }
            const bool up = (i & k) == 0, low = (i & j) == 0;
            if ((y < x) == (up == low)) x = y;
        }
    if (i < n) {
        const int who = int(x & 1023u);
        plan[i] = who;
        S.place[who] = i;
        plan[n + i] = end << page_shift(P.page);
        plan[2 * n + i] = depth;
    }
    __syncthreads();
    // ---- segments by level and place
#pragma unroll
    for (int l = 0; l < PS_LEVELS; ++l)
        if (S.seg_size[l][i] > 0) atomicOr(&S.heads[l][S.place[i] >> 5], 1u << (S.place[i] & 31));
    __syncthreads();
    if (warp < PS_LEVELS) {
        const int own = __popc(S.heads[warp][lane]);
        int y = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int z = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) y += z;
        }
        S.before[warp][lane] = y - own;
        if (lane == 31) S.total[warp] = y;
    }
    __syncthreads();
    int base = 0;
    int32_t* segments = plan + 3 * n;
#pragma unroll
    for (int l = 0; l < PS_LEVELS; ++l) {
        if (S.seg_size[l][i] > 0) {
            const int p = S.place[i];
            int32_t* to = segments + 5 * (base + S.before[l][p >> 5] + __popc(S.heads[l][p >> 5] & ((1u << (p & 31)) - 1)));
            to[0] = p;
            to[1] = S.seg_size[l][i];
            to[2] = S.seg_start[l][i] << page_shift(P.page);
            to[3] = S.seg_end[l][i] << page_shift(P.page);
            to[4] = l;
        }
        base += S.total[l];
    }
    for (int e = 5 * base + i; e < 5 * n; e += PS_THREADS) segments[e] = 0;
    if (i == 0) plan[8 * n] = base;
}

}  // namespace kvb
