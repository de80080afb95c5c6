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

// The window of a slot, found by every wave for itself: 64 sequences' first
// slots at a time, the last sequence whose first slot is not past `slot`. Offsets
// that fall or leave [0, N] set bad (every pair is looked at by slot 0, a slot's
// own pair by the slot, which then has nothing to do). Wave-uniform results.
__device__ __forceinline__ PackedWindow packed_window(const int32_t* __restrict__ cu, int n, int64_t N, int R, int BM,
                                                      int64_t slot, bool& bad) {
    const int lane = threadIdx.x % kWave;
    int seq = 0, c0 = 0, c1 = 0;
    for (int i0 = 0; i0 < n; i0 += kWave) {
        const int i = i0 + lane < n ? i0 + lane : n - 1;
        const int a0 = cu[i], a1 = cu[i + 1];   // (both at once: no second load behind the search)
        const uint64_t m = __ballot(i0 + lane < n && packed_first(a0, i, N, R, BM) <= slot);
        if (m == 0 && i0 > 0) break;            // (offsets that rise: no later sequence either)
        const int at = m == 0 ? 0 : 63 - __builtin_clzll(m);
        seq = i0 + at;
        c0 = __builtin_amdgcn_readlane(a0, at);
        c1 = __builtin_amdgcn_readlane(a1, at);
        if (m != ~0ull) break;
    }
    bad = c0 < 0 || c1 < c0 || c1 > N;
    PackedWindow w{-1, 0, 0, 0};
    const bool own = bad;
    if (slot == 0)
        for (int i = lane; i < n; i += kWave) bad = bad || cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > N;
    bad = __ballot(bad) != 0;
    if (own) return w;
    const int64_t win = slot - packed_first(c0, seq, N, R, BM);
    if (win < 0 || win * BM >= static_cast<int64_t>(c1 - c0) * R) return w;
    w.seq = seq;
    w.row0 = c0;
    w.len = c1 - c0;
    w.win = win;
    return w;
}

}  // namespace sparda
