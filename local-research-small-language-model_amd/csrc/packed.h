// Packed sequences: rows of n sequences back to back, sequence i in rows
// [cu[i], cu[i+1]) of N, cu a device array of n + 1 offsets that the host
// does not read. Work over all sequences is cut into windows of BM columns
// (R columns a row) without a host pass or a prefix over the lengths:
//     first(i) = floor(cu[i] R / BM) + i
// leaves sequence i the slots first(i) .. first(i+1) - 1, and those are
// floor((cu[i] R + len R) / BM) + 1 - floor(cu[i] R / BM) >= ceil(len R / BM),
// enough for its windows; the last slot is below floor(N R / BM) + n. A slot
// past its sequence's windows has nothing to do (at most one a sequence).
#pragma once

#include "common.h"

namespace sparda {

// Slots of n sequences of N rows, R columns a row, in windows of BM columns.
__host__ __device__ inline int64_t packed_slots(int64_t N, int64_t n, int64_t R, int64_t BM) { return N * R / BM + n; }

struct PackedWindow {
    int seq;            // sequence, -1: none
    int row0, len;      // its first row and rows
    int64_t win;        // the window's index in the sequence
};

// floor(cu R / BM) + i, offsets taken into [0, N]: whatever the array holds, a
// slot's window stays inside N rows
__device__ __forceinline__ int64_t packed_first(int c, int i, int64_t N, int R, int BM) {
    const int64_t k = c < 0 ? 0 : c > N ? N : c;
    return k * R / BM + i;
}

// The last of n sequences whose offset passes `before`, of those that can be the
// answer where offsets rise: 64 evenly spaced ones first, then 64 at a time behind the
// last of those that pass (two rounds up to 4096 sequences). -1: none. c0, c1: the
// sequence's offsets. Wave-uniform results.
template <class Before>
__device__ __forceinline__ int packed_find(const int32_t* __restrict__ cu, int n, Before before, int& c0, int& c1) {
    const int lane = threadIdx.x % kWave;
    int from = 0, to = n;
    if (n > kWave) {
        const int step = (n + kWave - 1) / kWave, i = lane * step < n ? lane * step : n - 1;
        const uint64_t m = __ballot(lane * step < n && before(cu[i], i));
        from = m == 0 ? 0 : (63 - __builtin_clzll(m)) * step;
        to = from + step < n ? from + step : n;
    }
    int seq = -1;
    c0 = c1 = 0;
    for (int i0 = from; i0 < to; i0 += kWave) {
        const int i = i0 + lane < to ? i0 + lane : to - 1;
        const int a0 = cu[i], a1 = cu[i + 1];   // (both at once: no second load behind the search)
        const uint64_t m = __ballot(i0 + lane < to && before(a0, i));
        if (m == 0) break;                      // (no later sequence either)
        const int at = 63 - __builtin_clzll(m);
        seq = i0 + at;
        c0 = __builtin_amdgcn_readlane(a0, at);
        c1 = __builtin_amdgcn_readlane(a1, at);
        if (m != ~0ull) break;
    }
    return seq;
}

// The window of a slot, found by every wave for itself: the last sequence whose
// first slot is not past `slot`. Offsets that fall or leave [0, N] set bad (every pair
// is looked at by slot 0, a slot's own pair by the slot, which then has nothing to
// do). Wave-uniform results.
__device__ __forceinline__ PackedWindow packed_window(const int32_t* __restrict__ cu, int n, int64_t N, int R, int BM,
                                                      int64_t slot, bool& bad) {
    const int lane = threadIdx.x % kWave;
    int c0, c1;
    const int seq = packed_find(cu, n, [&](int c, int i) { return packed_first(c, i, N, R, BM) <= slot; }, c0, c1);
    bad = c0 < 0 || c1 < c0 || c1 > N;
    PackedWindow w{-1, 0, 0, 0};
    const bool own = bad;
    if (slot == 0)
        for (int i = lane; i < n; i += kWave) bad = bad || cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > N;
    bad = __ballot(bad) != 0;
    if (own || seq < 0) return w;
    const int64_t win = slot - packed_first(c0, seq, N, R, BM);
    if (win < 0 || win * BM >= static_cast<int64_t>(c1 - c0) * R) return w;
    w.seq = seq;
    w.row0 = c0;
    w.len = c1 - c0;
    w.win = win;
    return w;
}

}  // namespace sparda
