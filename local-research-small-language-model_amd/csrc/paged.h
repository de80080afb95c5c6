// What the kernels over a cache in pages share (paged.hip, paged_q4.hip,
// paged_rotate.hip): the page table, the place of a new row, and how the attention of a
// batch is cut into shares.
#pragma once

#include "common.h"
#include "packed.h"

namespace sparda {

constexpr float kPgLog2e = 1.4426950408889634f;

// the pages and the table, as both kernels read them (strides in elements)
struct Pages {
    int64_t p_st, s_st, h_st;      // page, row, head
    const int32_t* table;
    int64_t t_st;                  // between the sequences' rows of the table
    int width;                     // entries of a row
    int n_pages;
};

// Where a packed new row goes.
struct PagedRow {
    bool takes;      // the row is one of a sequence's
    int seq;
    int64_t pos;     // its position
    int page;        // -1: outside the table or the cache
    int64_t row;     // in the page
};

// Row t of N new ones: its sequence (its own, or by the offsets), position and page. The first
// row's wavefront looks at every pair of offsets. Wave-uniform; raises the status bits.
__device__ __forceinline__ PagedRow paged_row(const Pages& pg, int ps, const int32_t* __restrict__ positions,
                                              const int32_t* __restrict__ cu, int n, int64_t N, int64_t t,
                                              uint32_t* __restrict__ status) {
    const int lane = threadIdx.x % kWave;
    PagedRow r{false, 0, 0, -1, 0};
    int64_t at = 0;                               // the row's place among its sequence's new rows
    if (cu == nullptr) {
        r.seq = static_cast<int>(t);
    } else {
        if (t == 0) {
            bool wrong = false;
            for (int i = lane; i < n; i += kWave) wrong = wrong || cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > N;
            if (__ballot(wrong) != 0 && lane == 0) atomicOr(status, static_cast<uint32_t>(SPARDA_STATUS_SEQUENCE_RANGE));
        }
        // the last sequence that starts at or before t, when t is one of its rows
        int c0, c1;
        r.seq = packed_find(cu, n, [&](int c, int) { return c <= t; }, c0, c1);
        if (r.seq < 0 || t >= c1) return r;       // before the first sequence, behind the last
        if (c0 < 0 || c1 > N) return r;           // (offsets out of range: the sequence is left out)
        at = t - c0;
    }
    const int p0 = __builtin_amdgcn_readfirstlane(positions[r.seq]);
    if (p0 < 0) return r;                         // a sequence that takes no part
    r.takes = true;
    r.pos = p0 + at;
    const int64_t slot = r.pos / ps;
    if (slot < pg.width) r.page = __builtin_amdgcn_readfirstlane(pg.table[r.seq * pg.t_st + slot]);
    if (r.page < 0 || r.page >= pg.n_pages) {
        r.page = -1;
        if (lane == 0) atomicOr(status, static_cast<uint32_t>(SPARDA_STATUS_PAGE_RANGE));
    }
    r.row = r.pos - slot * ps;
    return r;
}

// Shares of a launch. A sequence's keys are walked in steps of 16 kTiles keys.
// All steps of the batch are cut into shares of the same number of steps, so
// that long and short sequences load the workgroups alike: the share length is
// the total over `target`, at least `least`, and sequence b takes
// n_b = max(1, ceil(steps_b / share)) consecutive items of about equal length, at
// most target + B of them in all. Every workgroup derives this from the lengths
// for itself.
struct Share {
    int seq;         // -1: no sequence has this item
    int part, parts; // the item's place among its sequence's
    int first;       // the sequence's first item
    int share;       // steps of each of them
    int len;         // the sequence's length, cut to the table's capacity
    bool bad;        // the length is out of range
};

// steps of 2^log_step keys (len at most 2^31 - 64)
__device__ __forceinline__ int paged_steps(int len, int cap, int log_step) {
    const uint32_t c = len < 0 ? 0 : len > cap ? cap : len;
    return static_cast<int>((c + (1u << log_step) - 1) >> log_step);
}

// Inclusive sums over the lanes: within rows of 16 by shifts, then the rows' totals.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_dpp(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan_i32(int v) {
    asm volatile("s_nop 1" : "+v"(v));  // the wait states of the first DPP, on every way here
    v = add_dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v = add_dpp<0x112, 0xf>(v);
    v = add_dpp<0x114, 0xf>(v);
    v = add_dpp<0x118, 0xf>(v);
    v = add_dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v = add_dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int wave_last(int v) { return __builtin_amdgcn_readlane(v, kWave - 1); }

// The item's sequence (by_item), or sequence `want`'s items. Wave-uniform. The total
// of the steps stays below 2^30 (checked by the host against the capacity), so that
// the sums with the target or a share stay in 32 bits.
__device__ __forceinline__ Share paged_item(const int32_t* __restrict__ len, int B, int cap, int log_step, int target,
                                            int least, bool by_item, int want) {
    const int lane = threadIdx.x % kWave;
    auto at_least = [&](int total) { return max(least, (total + target - 1) / target); };
    auto found = [&](int seq, int l, int parts, int first) {
        return Share{seq, by_item ? want - first : 0, parts, first, (paged_steps(l, cap, log_step) + parts - 1) / parts,
                     l < 0 ? 0 : l > cap ? cap : l, l < 0 || l > cap};
    };
    if (B == 1) {
        const int l = __builtin_amdgcn_readfirstlane(len[0]), steps = paged_steps(l, cap, log_step), share = at_least(steps);
        const int parts = max(1, (steps + share - 1) / share);
        return by_item && want >= parts ? Share{-1} : found(0, l, parts, 0);
    }
    int total = 0;
    for (int b0 = 0; b0 < B; b0 += kWave) total += wave_last(wave_scan_i32(b0 + lane < B ? paged_steps(len[b0 + lane], cap, log_step) : 0));
    const int share = at_least(total);
    int before = 0;
    for (int b0 = 0; b0 < B; b0 += kWave) {
        const int b = b0 + lane, l = b < B ? len[b] : 0;
        const int n = b < B ? max(1, (paged_steps(l, cap, log_step) + share - 1) / share) : 0;
        const int end = before + wave_scan_i32(n);      // items of sequences 0 .. b
        const uint64_t m = __ballot(b < B && (by_item ? end > want : b == want));
        if (m != 0) {
            const int at = __builtin_ctzll(m), parts = __builtin_amdgcn_readlane(n, at);
            return found(b0 + at, __builtin_amdgcn_readlane(l, at), parts, __builtin_amdgcn_readlane(end, at) - parts);
        }
        before = wave_last(end);
    }
    return Share{-1};
}

constexpr int kPgJoin = 512;        // threads of a join

// (What only several tokens or 4-bit pages need stands at the end, on a cache line of its own: every further line
// of arguments that a kernel reads at its start costs it 0.3 us.)
struct PagedDecode {
    const void* q;
    int64_t q_sb, q_sh;           // sequence, head
    const void *k, *v;
    Pages pg;
    int ps16;                     // 16-key tiles of a page
    const int32_t* len;
    int B, cap;
    int Hq, Hkv, R, head_tiles;   // head tiles of 16 query heads per KV head
    int target, least;
    int whole;                    // every sequence is one item
    int lds_heads;                // heads of the largest tile
    float scale_log2;             // the scores' scale in log2 units
    int T;                        // tokens of a sequence; Hq = T heads, token-major
    void* out;
    int64_t out_sb;
    float *part_o, *part_ml;      // [items, Hq, D], [items, Hq, 2]
    uint32_t* status;
    int64_t q_st;                 // between tokens
    int heads;
    int negate;                   // (4-bit pages: scale_log2 is its magnitude, q takes the sign)
};

// joins the items of every sequence that has several (paged.hip), of steps of 2^log_step keys (5, or 4 with
// fp32); few: they are few in the mean
void launch_paged_join(const PagedDecode& a, int64_t D, int dtype, int log_step, bool few, hipStream_t stream);

}  // namespace sparda
