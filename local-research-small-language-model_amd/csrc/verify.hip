// Verification of drafted tokens (sparda_verify_drafts): which of a sequence's
// drafts its target distributions accept, and the token drawn behind them.
//
//   p_i = softmax(logits[b, i] / temperature[b]), q_i the draft's distribution of draft i (all of it on
//   the draft where none is given). Draft d_i is accepted while u_i q_i(d_i) < p_i(d_i). Behind n
//   accepted ones the token is the first at which the cumulated sum of r passes u_K times
//   its total: r = max(p_n - q_n, 0) after a rejection (p_n where that leaves nothing), r = p_n
//   where no draft is left. Temperature 0: the drafts are compared with the largest logits' lowest indexes.
//
// What is accepted and which token a long sum passes must not hang on how fp32 rounds, nor on the batch that a
// sequence is in, so both are decided in fp64. Two launches. One reads all logits once and leaves the maximum and
// the sum of every chunk of every row, for calls of up to 2^21 logits in fp64, in fp32 beyond, where fp64 would take
// longer than the memory (64 x 8 x 50257: a call of 47 us against 31). In the other, workgroups of a (chunk, sequence)
// find the accepted drafts, and each sums its chunk of the row that the token comes from again, in fp64; the last one that
// comes draws. Where fp32 left an acceptance open (one in 10^5), it does all of this once more in fp64. A token from p
// over sums in fp64 is drawn by the first workgroup alone.
//
// The sums of max(p - q, 0) need p's total Z, which no workgroup has. They are taken apart: over the tokens
// where w / Z' > q, w = p Z and Z' the total in fp32, sum (w / Z - q) = A / Z - Q with
// A = sum w, Q = sum q, and the last workgroup has Z. Tokens between the two borders are off by at most kVdOff q;
// where the token that is drawn begins or ends so near to the target that this could matter, the last workgroup
// does it over too.
#include "common.h"
#include "kernels.h"

namespace sparda {

namespace {

constexpr int kVdThreads = 256, kVdWaves = kVdThreads / kWave;
constexpr int kVdRows = 65;           // rows of a sequence (drafts + 1), at most
constexpr int kVdRounds = 16;         // rounds of a chunk (one 16-byte piece a thread), at most; a row has at most 64 chunks
constexpr double kVdLog2e = 1.4426950408889634074;
// How far a row's sum in fp32 may be off, relatively: up to 64 weights a thread (63 2^-24) and six sums of lanes, a
// weight by its exponential (2^-23) and by three roundings of its exponent t, 3 2^-24 ln 2 |t|, of which the mean over the
// weights is below 16 (of 2^20 weights at most), 2 10^-6: together 6.4 10^-6.
constexpr double kVdOff = 0x1p-17;

struct alignas(16) ChunkStat {
    float m;         // largest logit of the chunk
    int32_t arg;     // its lowest index (greedy sequences)
    double sum;      // of 2^((x - m) log2 e / temperature)
};
struct ChunkSum {
    double w, above, q;  // of the weights, those above q, q there
    double near;         // of q where w / Z' is so near to q that w / Z may lie on its other side
};
struct SequenceState {
    uint32_t done, pad;  // workgroups of the second launch that are through
};

struct Verify {
    const void* logits;
    int64_t l_sb, l_st;
    const int32_t* drafts;
    int64_t d_sb;
    const float* uniform;
    int64_t u_sb;
    const float* probs;
    int64_t p_sb, p_st;
    const int32_t* counts;       // drafts of a sequence; nullptr: K of each
    const float* temperature;    // of a sequence; nullptr: all_temperature
    float all_temperature;
    int K;
    int64_t V;
    int rounds1, rounds2;        // rounds of a chunk in either launch
    int chunks1, chunks2;
    ChunkStat* stats;            // [B, K + 1, chunks1]
    ChunkSum* sums;              // [B, chunks2]
    SequenceState* state;        // [B]
    int32_t *tokens, *accepted;  // [B, K + 1], [B]
};

__device__ __forceinline__ int vd_count(const Verify& a, int b) {
    if (a.counts == nullptr) return a.K;
    const int n = a.counts[b];
    return n < 0 ? 0 : n > a.K ? a.K : n;
}
__device__ __forceinline__ float vd_temperature(const Verify& a, int b) {
    const float T = a.temperature != nullptr ? a.temperature[b] : a.all_temperature;
    return T > 3.4e38f ? 3.4e38f : T;             // (inf: -inf logits keep their weight of 0)
}

// 2^t for -1020 <= t <= 0: t = n + f, |f| <= 1/2, and the Taylor series of 2^f up to f^10, whose
// rest is below 3 10^-13. n is rounded by the addition of 1.5 2^52, whose low word then holds it, and goes
// into the exponent as an integer (the conversions and the scaling of fp64 run at a
// quarter of the rate: 50257 x 512 logits 31.5 us with them, 28 without).
__device__ __forceinline__ double vd_exp2(double t) {
    constexpr double kShift = 6755399441055744.0;
    const double y = t + kShift, f = t - (y - kShift);
    double p = 7.0549116208011209e-09;            // (ln 2)^k / k!, k = 10 .. 0
    p = __builtin_fma(p, f, 1.0178086009239696e-07);
    p = __builtin_fma(p, f, 1.3215486790144305e-06);
    p = __builtin_fma(p, f, 1.5252733804059838e-05);
    p = __builtin_fma(p, f, 1.5403530393381606e-04);
    p = __builtin_fma(p, f, 1.3333558146428441e-03);
    p = __builtin_fma(p, f, 9.6181291076284769e-03);
    p = __builtin_fma(p, f, 5.5504108664821576e-02);
    p = __builtin_fma(p, f, 2.4022650695910069e-01);
    p = __builtin_fma(p, f, 6.9314718055994529e-01);
    p = __builtin_fma(p, f, 1.0);
    const uint64_t u = __builtin_bit_cast(uint64_t, p);
    const uint32_t n = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, y));
    return __builtin_bit_cast(double, (static_cast<uint64_t>(static_cast<uint32_t>(u >> 32) + (n << 20)) << 32) | static_cast<uint32_t>(u));
}
// for every t <= 0: 0 below -1020, which leaves -inf no weight
__device__ __forceinline__ double vd_weight(double t) {
    const double w = vd_exp2(fmax(t, -1020.0));
    return t > -1020.0 ? w : 0.0;
}

template <int DT>
struct VdType {
    static constexpr int kEs = DT == SPARDA_F32 ? 4 : 2, kVe = 16 / kEs;   // bytes of an element, elements of a piece
    static constexpr int kRound = kVdThreads * kVe;                        // elements of a round
};

// A piece of 16 bytes of a row, elements [at, at + kVe); those outside [0, V) are -inf. A piece
// that leaves the row is read element by element.
template <int DT>
__device__ __forceinline__ uint4 vd_load(const char* row, int64_t at, int64_t V) {
    constexpr int kVe = VdType<DT>::kVe, kEs = VdType<DT>::kEs;
    if (at >= 0 && at + kVe <= V) return *reinterpret_cast<const uint4*>(row + at * kEs);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == SPARDA_F32) {
            w[i] = at + i >= 0 && at + i < V ? reinterpret_cast<const uint32_t*>(row)[at + i] : 0xff800000u;
        } else {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
            const int64_t e = at + 2 * i;
            w[i] = (e >= 0 && e < V ? p[e] : 0xff80u) | static_cast<uint32_t>(e + 1 >= 0 && e + 1 < V ? p[e + 1] : 0xff80u) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int DT>
__device__ __forceinline__ float vd_element(const uint4& x, int e) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    if constexpr (DT == SPARDA_F32) return __uint_as_float(w[e]);
    else return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
}

// elements before a row's start in its first aligned piece
template <int DT>
__device__ __forceinline__ int vd_shift(const char* row) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16) / VdType<DT>::kEs;
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// inclusive sums over the lanes: within rows of 16 by shifts, then the rows' totals
__device__ __forceinline__ double wave_scan_f64(double v) {
    v += dpp_f64<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp_f64<0x112, 0xf>(v);
    v += dpp_f64<0x114, 0xf>(v);
    v += dpp_f64<0x118, 0xf>(v);
    v += dpp_f64<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp_f64<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}
// over the 16 lanes of a row, the result in every one
__device__ __forceinline__ float row16_max(float v) {
    v = fmaxf(v, dpp_f32<kDppXor1>(v));
    v = fmaxf(v, dpp_f32<kDppXor2>(v));
    v = fmaxf(v, dpp_f32<kDppHalfMirror>(v));
    return fmaxf(v, dpp_f32<kDppMirror>(v));
}
__device__ __forceinline__ double row16_sum_f64(double v) {
    v += dpp_f64<kDppXor1, 0xf>(v);
    v += dpp_f64<kDppXor2, 0xf>(v);
    v += dpp_f64<kDppHalfMirror, 0xf>(v);
    return v + dpp_f64<kDppMirror, 0xf>(v);
}
__device__ __forceinline__ int row16_min(int v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 16));
    return v;
}
__device__ __forceinline__ double wave_sum_f64(double v) { return lane_f64(wave_scan_f64(v), kWave - 1); }

}  // namespace

// Maximum and sum of a chunk of a row, in one read: the chunk's pieces stay in registers. Every
// wavefront measures its exponentials against its own maximum, so that the wavefronts meet once. Bound by memory in
// large calls: 64 x 8 rows of 50257 in bf16 (51.5 MB) take 13.3 us = 3.9 TB/s, 32 x 6 of 32000 in fp32
// (24.6 MB) 7.2-8.9; 5 rows of 32000 take 4.0, a launch, a load and a reduction.
template <int DT, int ROUNDS, bool EXACT>
__global__ void __launch_bounds__(kVdThreads) verify_stats_kernel(Verify a) {
    constexpr int kVe = VdType<DT>::kVe, kEs = VdType<DT>::kEs;
    __shared__ float rm[kVdWaves];
    __shared__ double rs[kVdWaves];
    __shared__ int ra[kVdWaves];
    const int tid = threadIdx.x, wave = tid / kWave, chunk = blockIdx.x;
    const int b = blockIdx.y / (a.K + 1), i = blockIdx.y % (a.K + 1);
    if (chunk == 0 && i == 0 && tid == 0) a.state[b].done = 0;
    const char* row = static_cast<const char*>(a.logits) + (b * a.l_sb + i * a.l_st) * kEs;
    const int64_t first = static_cast<int64_t>(chunk) * ROUNDS * VdType<DT>::kRound - vd_shift<DT>(row);
    if (i > vd_count(a, b)) return;                           // no draft's row
    uint4 x[ROUNDS];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) x[k] = vd_load<DT>(row, first + (tid + k * kVdThreads) * kVe, a.V);
    const float T = vd_temperature(a, b);
    const bool greedy = !(T > 0.0f);
    const double c = greedy ? kVdLog2e : kVdLog2e / static_cast<double>(T);
    float m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
        for (int e = 0; e < kVe; ++e) m = fmaxf(m, vd_element<DT>(x[k], e));
    m = wave_max(m);
    double s = 0.0;
    int arg = 0x7fffffff;
    // a NaN comes back in every sum in fp32, the masked and the greedy ones' too
    if constexpr (!EXACT) {
        const float c32 = static_cast<float>(fmin(c, 3e38)), ref = m == -__builtin_inff() ? 0.0f : m;
        float s32 = 0.0f;
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
            for (int e = 0; e < kVe; ++e) s32 += __builtin_amdgcn_exp2f((vd_element<DT>(x[k], e) - ref) * c32);
        s = wave_sum(s32);
    } else {
        float nan = 0.0f;                                     // NaN or 0, one operation a logit
#pragma unroll
        for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
            for (int e = 0; e < kVe; ++e) nan = __builtin_fmaf(vd_element<DT>(x[k], e) == -__builtin_inff() ? 0.0f : vd_element<DT>(x[k], e), 0.0f, nan);
        if (!greedy && m > -__builtin_inff()) {               // (wave-uniform)
#pragma unroll
            for (int k = 0; k < ROUNDS; ++k)
#pragma unroll
                for (int e = 0; e < kVe; ++e)
                    s += vd_exp2(fmax((static_cast<double>(vd_element<DT>(x[k], e)) - static_cast<double>(m)) * c, -1020.0));
        }
        s = wave_sum_f64(s);
        if (__ballot(nan != nan) != 0) s = __builtin_nan("");
    }
    if (greedy) {
#pragma unroll
        for (int k = ROUNDS - 1; k >= 0; --k)
#pragma unroll
            for (int e = kVe - 1; e >= 0; --e)
                if (vd_element<DT>(x[k], e) == m) arg = static_cast<int>(first + (tid + k * kVdThreads) * kVe + e);
        arg = wave_min_i32(arg);
    }
    if (tid % kWave == 0) rm[wave] = m, rs[wave] = s, ra[wave] = arg;
    __syncthreads();
    if (tid == 0) {
        ChunkStat st{rm[0], 0x7fffffff, 0.0};
#pragma unroll
        for (int w = 1; w < kVdWaves; ++w) st.m = fmaxf(st.m, rm[w]);
#pragma unroll
        for (int w = 0; w < kVdWaves; ++w) {
            // (a wavefront without a finite logit adds nothing, NaN among them stays)
            st.sum += rm[w] == -__builtin_inff() ? rs[w] : rs[w] * vd_weight((static_cast<double>(rm[w]) - st.m) * c);
            if (rm[w] == st.m) st.arg = min(st.arg, ra[w]);
        }
        a.stats[static_cast<int64_t>(blockIdx.y) * a.chunks1 + chunk] = st;
    }
}

namespace {

// What a token is drawn from, and what is taken off its weights.
struct VdRow {
    const char* row;
    const float* q;          // nullptr, or the weights are max(p - q, 0)
    int64_t without;         // no weight for this token (-1: none)
    double c, m;             // a weight is 2^((x - m) c): 1 for every x of m, whatever they are
    double inv_total;        // one over p's weights (with q)
};

// weights of a piece, not yet against q, and q
template <int DT>
__device__ __forceinline__ void vd_piece(const VdRow& r, int64_t at, int64_t V, double (&w)[VdType<DT>::kVe], float (&q)[VdType<DT>::kVe]) {
    constexpr int kVe = VdType<DT>::kVe;
    const uint4 x = vd_load<DT>(r.row, at, V);
    if (r.q != nullptr) {
        if (at >= 0 && at + kVe <= V) {
#pragma unroll
            for (int e = 0; e < kVe; ++e) q[e] = r.q[at + e];
        } else {
#pragma unroll
            for (int e = 0; e < kVe; ++e) q[e] = at + e >= 0 && at + e < V ? r.q[at + e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < kVe; ++e) {
        w[e] = vd_weight((static_cast<double>(vd_element<DT>(x, e)) - r.m) * r.c);
        if (at + e == r.without) w[e] = 0.0;
    }
}
template <int DT>
__device__ __forceinline__ void vd_weights(const VdRow& r, int64_t at, int64_t V, double (&w)[VdType<DT>::kVe]) {
    constexpr int kVe = VdType<DT>::kVe;
    float q[kVe];
    vd_piece<DT>(r, at, V, w, q);
    if (r.q == nullptr) return;
#pragma unroll
    for (int e = 0; e < kVe; ++e) {
        const double d = __builtin_fma(w[e], r.inv_total, -static_cast<double>(q[e]));
        w[e] = d > 0.0 ? d : 0.0;
    }
}

// the sums of a chunk's weights, by all threads; the result in every one (NEAR: `near` among them)
template <int DT, bool NEAR>
__device__ __forceinline__ ChunkSum vd_chunk_sum(const VdRow& r, int64_t first, int rounds, int64_t V, double* red) {
    constexpr int kVe = VdType<DT>::kVe;
    ChunkSum s{0.0, 0.0, 0.0, 0.0};
    float near = 0.0f;                            // (its size matters, not its last bits)
    for (int k = 0; k < rounds; ++k) {
        double w[kVe];
        float q[kVe];
        vd_piece<DT>(r, first + (threadIdx.x + k * kVdThreads) * kVe, V, w, q);
#pragma unroll
        for (int e = 0; e < kVe; ++e) {
            s.w += w[e];
            if (r.q != nullptr) {
                const double d = __builtin_fma(w[e], r.inv_total, -static_cast<double>(q[e]));
                if (d > 0.0) s.above += w[e], s.q += q[e];
                if constexpr (NEAR) near += __builtin_fabsf(static_cast<float>(d)) < static_cast<float>(kVdOff) * q[e] ? q[e] : 0.0f;
            }
        }
    }
    s.w = wave_sum_f64(s.w);
    if (r.q != nullptr) {
        s.above = wave_sum_f64(s.above), s.q = wave_sum_f64(s.q);
        if constexpr (NEAR) s.near = wave_sum(near);
    }
    const int wave = threadIdx.x / kWave;
    __syncthreads();                              // (the array's last use)
    if (threadIdx.x % kWave == 0) red[4 * wave] = s.w, red[4 * wave + 1] = s.above, red[4 * wave + 2] = s.q, red[4 * wave + 3] = s.near;
    __syncthreads();
    s = ChunkSum{red[0], red[1], red[2], red[3]};
#pragma unroll
    for (int w = 1; w < kVdWaves; ++w) s.w += red[4 * w], s.above += red[4 * w + 1], s.q += red[4 * w + 2], s.near += red[4 * w + 3];
    return s;
}

// The token of the chunks' sums (lane c of every wavefront holds chunk c's): the chunk where they pass
// u times their total, the round and the wavefront in it, then the token. All threads of the workgroup; red: one
// number a round and wavefront; gap: how far the target is from both ends of the token's part of the sum, 0 where
// no sum passes it.
template <int DT>
__device__ __forceinline__ int vd_draw(const VdRow& r, double of_lane, int rounds, int64_t V, float u, double* red, int* found, double* gap) {
    constexpr int kVe = VdType<DT>::kVe;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const double upto_chunk = wave_scan_f64(of_lane);
    const double target = static_cast<double>(u) * lane_f64(upto_chunk, kWave - 1);
    const uint64_t pass = __ballot(upto_chunk > target), some = __ballot(of_lane > 0.0);
    // (none passes where u is 1, or the last by a rounding: the last token that weighs anything)
    const int chunk = pass != 0 ? __builtin_ctzll(pass) : 63 - __builtin_clzll(some | 1);
    const double base = lane_f64(upto_chunk, chunk) - lane_f64(of_lane, chunk);
    const int64_t first = static_cast<int64_t>(chunk) * rounds * VdType<DT>::kRound - vd_shift<DT>(r.row);
    double w[kVe];
    __syncthreads();                              // (the arrays' last use)
    for (int k = 0; k < rounds; ++k) {
        vd_weights<DT>(r, first + (tid + k * kVdThreads) * kVe, V, w);
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < kVe; ++e) s += w[e];
        s = wave_sum_f64(s);
        if (lane == 0) red[k * kVdWaves + wave] = s;
    }
    if (tid == 0) *found = -1, *gap = 0.0;
    __syncthreads();
    // lane: a (round, wavefront), in the order of the row
    const double part = lane < rounds * kVdWaves ? red[lane] : 0.0, upto = wave_scan_f64(part);
    const uint64_t here = __ballot(base + upto > target), any = __ballot(part > 0.0);
    const int at_part = pass != 0 && here != 0 ? __builtin_ctzll(here) : 63 - __builtin_clzll(any | 1);
    if (wave == at_part % kVdWaves) {             // the wavefront whose pieces they are
        const int64_t at = first + (tid + at_part / kVdWaves * kVdThreads) * kVe;
        if (at_part / kVdWaves != rounds - 1) vd_weights<DT>(r, at, V, w);   // (the last round's are there)
        double mine = 0.0;
#pragma unroll
        for (int e = 0; e < kVe; ++e) mine += w[e];
        const double scan = wave_scan_f64(mine), before = base + (lane_f64(upto, at_part) - lane_f64(part, at_part));
        const uint64_t over = __ballot(mine > 0.0 && before + scan > target), have = __ballot(mine > 0.0);
        // (rounding may leave these sums below the parts': the last that weighs anything)
        const bool passes = pass != 0 && here != 0 && over != 0;
        if (lane == (passes ? __builtin_ctzll(over) : 63 - __builtin_clzll(have | 1))) {
            double acc = before + (scan - mine);
            int hit = -1, last = -1;
#pragma unroll
            for (int e = 0; e < kVe; ++e) {
                acc += w[e];
                if (w[e] > 0.0) {
                    last = e;
                    if (hit < 0 && acc > target) hit = e, *gap = fmin(acc - target, target - (acc - w[e]));
                }
            }
            *found = last < 0 ? -1 : static_cast<int>(at + (passes && hit >= 0 ? hit : last));
        }
    }
    __syncthreads();
    return *found;
}

// What workgroups of a launch hand to the last of them goes through stores and loads at the device's
// scope, which pass the caches that they do not share; a store is waited for before its workgroup
// is counted. (A release or acquire at that scope would write back and drop whole caches instead, once a
// workgroup: 35 us a launch of 1024.)
__device__ __forceinline__ double vd_read(const double* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void vd_write(double* p, double v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ ChunkSum vd_read_sum(const ChunkSum* p) {   // (all on their way at once)
    ChunkSum s;
    s.w = vd_read(&p->w), s.above = vd_read(&p->above), s.q = vd_read(&p->q), s.near = vd_read(&p->near);
    return s;
}
// writes the workgroup's sums and counts it; true in the last of `all`
__device__ __forceinline__ bool vd_last(ChunkSum* to, const ChunkSum& s, uint32_t* done, uint32_t all, int* flag) {
    if (threadIdx.x == 0) {
        vd_write(&to->w, s.w);
        vd_write(&to->above, s.above);
        vd_write(&to->q, s.q);
        vd_write(&to->near, s.near);
        __builtin_amdgcn_s_waitcnt(0x0f70);       // vmcnt(0): the stores have arrived
        asm volatile("" ::: "memory");
        *flag = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == all;
    }
    __syncthreads();
    return *flag != 0;
}

}  // namespace

// One workgroup per (chunk, sequence), or per sequence where all sums are there and no distributions are given.
// Bound by its chain: the statistics, the row (a load that waits for what was accepted), a reduction,
// the sums' way through memory, the last workgroup's loads of them and of its chunk again. 64 rows of 50257 with
// q (19 MB) 17.0 us, of which the last workgroups' draw is 2.2 and the exponentials in fp64 1.7 (measured
// without each); 32 of 32000 in fp32 12.7; one sequence 6.0. Drafts' logits and q fetched by the first launch instead of
// here: no difference in a call (28.5 / 28.3, 20.1 / 20.1 us).
// Where fp32 leaves a decision open (a call of 64 x 7 in a hundred), the last workgroup goes through the sequence again:
// some 30 us a row. It is inlined, with the registers of six wavefronts a SIMD, which run the 1600 workgroups of 64 x 50257
// at once: a call of 31.6 us; without the bound 33.3, out of line 34.2, without that way 31.0.
template <int DT, bool EXACT>
__global__ void __launch_bounds__(kVdThreads, 6) verify_draw_kernel(Verify a) {
    constexpr int kEs = VdType<DT>::kEs;
    __shared__ double red[kVdRounds * kVdWaves], rz[kVdRows];   // (red: a number a round and wavefront, four a wavefront)
    __shared__ double gap;
    __shared__ float rmax[kVdRows];
    __shared__ int rarg[kVdRows], ok[kVdRows], found, flag;
    const int tid = threadIdx.x, lane = tid % kWave, chunk = blockIdx.x, b = blockIdx.y;
    const int count = vd_count(a, b);
    const float T = vd_temperature(a, b);
    const bool greedy = !(T > 0.0f);
    const double c = greedy ? kVdLog2e : kVdLog2e / static_cast<double>(T);
    const ChunkStat* stats = a.stats + static_cast<int64_t>(b) * (a.K + 1) * a.chunks1;
    // a chunk's sum, measured against the row's maximum
    auto in_row = [&](const ChunkStat& s, float m) {
        return s.m == -__builtin_inff() ? s.sum : s.sum * vd_weight((static_cast<double>(s.m) - m) * c);
    };
    for (int i = tid / 16; i <= a.K; i += kVdThreads / 16) {  // 16 lanes a row
        const int l16 = tid % 16;
        ChunkStat own[4];                                     // chunks l16, l16 + 16 ..
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            own[j] = ChunkStat{-__builtin_inff(), 0x7fffffff, 0.0};
            if (l16 + 16 * j < a.chunks1) own[j] = stats[i * a.chunks1 + l16 + 16 * j];
        }
        // (the draft's own numbers under the chunks'; of a row behind the last draft nothing is used)
        int d = -1;
        float x = -__builtin_inff(), u = 0.0f, q = 1.0f;
        if (i < a.K) {
            d = a.drafts[b * a.d_sb + i];
            u = a.uniform[b * a.u_sb + i];
            if (d >= 0 && d < a.V) {
                x = load_elem<DT>(a.logits, b * a.l_sb + i * a.l_st + d);
                if (a.probs) q = a.probs[b * a.p_sb + i * a.p_st + d];
            }
        }
        const float m = row16_max(fmaxf(fmaxf(own[0].m, own[1].m), fmaxf(own[2].m, own[3].m)));
        const bool finite = m > -__builtin_inff() && m < __builtin_inff();
        double z = 0.0;
        int arg = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (16 * j < a.chunks1) z += finite ? in_row(own[j], m) : 0.0;
            arg = own[j].m == m ? min(arg, own[j].arg) : arg;
        }
        z = row16_sum_f64(z);
        if (greedy) arg = row16_min(arg);
        if (l16 == 0) {
            const bool valid = finite && z < __builtin_inf();
            const bool inside = d >= 0 && d < a.V;
            const double p = valid && inside ? vd_weight((static_cast<double>(x) - m) * c) : 0.0;
            rmax[i] = m, rz[i] = z, rarg[i] = valid ? (greedy ? arg : 0) : -1;
            const double uq = static_cast<double>(u) * q;
            const bool yes = greedy ? d == arg : uq < p / z;
            // bit 1: open, z in fp32 may be wrong by as much (or c is one that fp32 does not hold)
            const bool unsure = !EXACT && !greedy && p > 0.0 && (__builtin_fabs(uq * z - p) <= kVdOff * p || c > 3e38);
            ok[i] = valid && inside ? (yes ? 1 : 0) | (unsure ? 2 : 0) : 0;
        }
    }
    __syncthreads();
    int n = 0, open = !EXACT && c > 3e38 ? 2 : 0;
    for (; n < count; ++n) {
        const int yes = ok[n];
        open |= yes;
        if ((yes & 1) == 0) break;
    }
    auto write = [&](int token) {
        for (int i = tid; i <= a.K; i += kVdThreads)
            a.tokens[static_cast<int64_t>(b) * (a.K + 1) + i] = i < n ? a.drafts[b * a.d_sb + i] : i == n ? token : -1;
        if (tid == 0) a.accepted[b] = n;
    };
    if ((rarg[n] < 0 && (open & 2) == 0) || greedy) {
        if (chunk == 0) write(rarg[n]);
        return;
    }
    const float u01 = a.uniform[b * a.u_sb + a.K], u = u01 < 0.0f ? 0.0f : u01;
    auto of_row = [&](double total) {                         // row n, as the token is drawn from it where q is not taken off
        VdRow r{};
        r.row = static_cast<const char*>(a.logits) + (b * a.l_sb + n * a.l_st) * kEs;
        r.c = c, r.m = rmax[n], r.inv_total = 1.0 / total, r.without = -1;
        const int64_t d = n < count && a.probs == nullptr ? a.drafts[b * a.d_sb + n] : -1;   // the rejected draft weighs nothing
        if (d >= 0 && d < a.V) r.without = d;
        return r;
    };
    VdRow r = of_row(rz[n]);
    const bool against = n < count && a.probs != nullptr;
    const int64_t shift = vd_shift<DT>(r.row);
    double of_lane;                                           // a chunk's weight
    int rounds = a.rounds2, token = -1;
    VdRow less = r;
    if (against) less.q = a.probs + b * a.p_sb + n * a.p_st;
    if (!EXACT || against) {
        ChunkSum* sums = a.sums + static_cast<int64_t>(b) * a.chunks2;
        const ChunkSum s = vd_chunk_sum<DT, !EXACT>(less, static_cast<int64_t>(chunk) * rounds * VdType<DT>::kRound - shift, rounds, a.V, red);
        if (!vd_last(&sums[chunk], s, &a.state[b].done, static_cast<uint32_t>(a.chunks2), &flag)) return;
        const ChunkSum of = lane < a.chunks2 ? vd_read_sum(&sums[lane]) : ChunkSum{0.0, 0.0, 0.0, 0.0};
        of_lane = of.w;
        bool again = (open & 2) != 0;
        if (against) {
            less.inv_total = 1.0 / wave_sum_f64(of_lane);
            const double left = __builtin_fma(of.above, less.inv_total, -of.q);
            const double of_less = left > 0.0 ? left : 0.0;
            // (the sums up to the token and the target each move by `off` at most)
            const double off = EXACT ? 0.0 : kVdOff * wave_sum_f64(of.near);
            if (__ballot(of_less > 0.0) != 0) token = vd_draw<DT>(less, of_less, rounds, a.V, u, red, &found, &gap);
            again = again || (off > 0.0 && (token < 0 || gap <= 3.0 * off));
        }
        if (!EXACT && __builtin_expect(again, 0)) {           // (workgroup-uniform) the sequence again, all sums in fp64
            double of_p = 0.0;
            bool last = false;                                // row n's total is known: now what the token is drawn from
            for (n = 0;;) {
                const int yes = n < count ? ok[n] : 0;
                if (!last) {
                    if (yes == 1) {
                        ++n;
                        continue;
                    }
                    if (rarg[n] < 0) {
                        write(-1);
                        return;
                    }
                    r = of_row(1.0);
                }
                const int64_t without = r.without;
                r.without = last ? without : -1;
                double z = 0.0;
                of_lane = 0.0;
                for (int i = 0; i < a.chunks2; ++i) {
                    const ChunkSum s = vd_chunk_sum<DT, false>(r, static_cast<int64_t>(i) * rounds * VdType<DT>::kRound - vd_shift<DT>(r.row), rounds, a.V, red);
                    z += s.w;
                    const double left = r.q != nullptr ? __builtin_fma(s.above, r.inv_total, -s.q) : s.w;
                    if (lane == i) of_lane = left > 0.0 ? left : 0.0;
                }
                r.without = without;
                if (last) break;
                if (yes != 0) {                               // open: its draft is in the vocabulary
                    const int32_t d = a.drafts[b * a.d_sb + n];
                    const double w = vd_weight((static_cast<double>(load_elem<DT>(a.logits, b * a.l_sb + n * a.l_st + d)) - r.m) * c);
                    const float q = a.probs ? a.probs[b * a.p_sb + n * a.p_st + d] : 1.0f;
                    if (static_cast<double>(a.uniform[b * a.u_sb + n]) * q < w / z) {
                        ++n;
                        continue;
                    }
                }
                if (n < count && a.probs != nullptr) r.q = a.probs + b * a.p_sb + n * a.p_st;
                else if (without < 0) break;
                of_p = of_lane, r.inv_total = 1.0 / z, last = true;
            }
            if (r.q != nullptr && __ballot(of_lane > 0.0) == 0) r.q = nullptr, of_lane = of_p;   // nothing is left
            token = -1;
        }
    } else {
        if (chunk != 0) return;
        rounds = a.rounds1;
        of_lane = lane < a.chunks1 ? in_row(stats[n * a.chunks1 + lane], rmax[n]) : 0.0;
        if (r.without >= 0) {
            const int at = static_cast<int>((r.without + shift) / (static_cast<int64_t>(rounds) * VdType<DT>::kRound));
            const ChunkSum s = vd_chunk_sum<DT, false>(r, static_cast<int64_t>(at) * rounds * VdType<DT>::kRound - shift, rounds, a.V, red);
            of_lane = lane == at ? s.w : of_lane;
        }
    }
    // from p (without the draft, which holds all of it where nothing is left)
    if (token < 0) token = __ballot(of_lane > 0.0) != 0 ? vd_draw<DT>(r, of_lane, rounds, a.V, u, red, &found, &gap) : static_cast<int>(r.without);
    write(token);
}

namespace {

// Sizes, with what was measured on either side (us a call):
// - fp64 statistics up to 2^21 logits, where the launch and the loads hide them (5 x 32000: 10.1 either way) and
//   a token from p needs no second pass; beyond, 64 x 8 x 50257 47 with them, 31 without.
// - The first launch's chunks grow from one round (256 pieces of 16 bytes) to eight while there are more than
//   4096 of them: two / four / eight rounds at 64 x 8 x 50257 32.3 / 31.4 / 34.5 (then; four is the rule's).
// - The second launch's grow while there are more than 2048: limits of 256 / 512 / 1024 / 2048 / 4096 at 64 x
//   50257 38.0 / 32.8 / 29.8 / 28.4 / 28.4, at 32 x 32000 in fp32 21.0 / 19.2 / 20.0 / 20.4 / 20.0.
// - A row has at most 64 chunks, a lane each.
struct VerifyPlan {
    bool exact;
    int rounds1, rounds2, chunks1, chunks2;
    size_t stats, sums, state, bytes;   // offsets, and all
};
VerifyPlan verify_plan(int64_t B, int64_t K, int64_t V, int dtype) {
    VerifyPlan p{};
    const int64_t ve = dtype == SPARDA_F32 ? 4 : 8, round = kVdThreads * ve, all = V + ve - 1;   // (a row may start inside a piece)
    p.exact = B * (K + 1) * V <= (1 << 21);
    p.rounds1 = 1;
    while (p.rounds1 < kVdRounds && ((p.rounds1 < 8 && B * (K + 1) * cdiv(all, round * p.rounds1) > 4096) || cdiv(all, round * p.rounds1) > kWave)) p.rounds1 *= 2;
    p.chunks1 = static_cast<int>(cdiv(all, round * p.rounds1));
    p.rounds2 = static_cast<int>(cdiv(all, round * kWave));
    while (p.rounds2 < kVdRounds && B * cdiv(all, round * p.rounds2) > 2048) ++p.rounds2;
    p.chunks2 = static_cast<int>(cdiv(all, round * p.rounds2));
    p.stats = 0;
    p.sums = p.stats + static_cast<size_t>(B * (K + 1) * p.chunks1) * sizeof(ChunkStat);
    p.state = p.sums + static_cast<size_t>(B * p.chunks2) * sizeof(ChunkSum);
    p.bytes = p.state + static_cast<size_t>(B) * sizeof(SequenceState);
    return p;
}

}  // namespace

size_t verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V, int dtype) { return verify_plan(B, K, V, dtype).bytes; }

int launch_verify_drafts(const void* logits, int dtype, int64_t l_sb, int64_t l_st, const int32_t* drafts, int64_t d_sb,
                         const float* uniform, int64_t u_sb, const float* probs, int64_t p_sb, int64_t p_st,
                         const int32_t* counts, const float* temperature, float all_temperature, int64_t B, int64_t K,
                         int64_t V, int32_t* tokens, int32_t* accepted, void* workspace, hipStream_t stream) {
    const VerifyPlan p = verify_plan(B, K, V, dtype);
    char* ws = static_cast<char*>(workspace);
    const Verify a{logits, l_sb, l_st, drafts, d_sb, uniform, u_sb, probs, p_sb, p_st, counts, temperature, all_temperature,
                   static_cast<int>(K), V, p.rounds1, p.rounds2, p.chunks1, p.chunks2,
                   reinterpret_cast<ChunkStat*>(ws + p.stats), reinterpret_cast<ChunkSum*>(ws + p.sums),
                   reinterpret_cast<SequenceState*>(ws + p.state), tokens, accepted};
    if (!grid_fits(static_cast<int64_t>(p.chunks1) * B * (K + 1), kVdThreads) || !grid_fits(static_cast<int64_t>(p.chunks2) * B, kVdThreads))
        return set_error(SPARDA_ERR_SHAPE, "verify_drafts: grid too large");
    const dim3 grid1(static_cast<unsigned>(p.chunks1), static_cast<unsigned>(B * (K + 1))), threads(kVdThreads);
    const dim3 grid2(static_cast<unsigned>(probs || !p.exact ? p.chunks2 : 1), static_cast<unsigned>(B));
#define SPARDA_VD_R(DT_, R_)                                                                             \
    do {                                                                                                 \
        if (p.exact) hipLaunchKernelGGL((verify_stats_kernel<DT_, R_, true>), grid1, threads, 0, stream, a); \
        else hipLaunchKernelGGL((verify_stats_kernel<DT_, R_, false>), grid1, threads, 0, stream, a);    \
    } while (0)
#define SPARDA_VD(DT_)                                                                       \
    do {                                                                                     \
        switch (p.rounds1) {                                                                 \
            case 1: SPARDA_VD_R(DT_, 1); break;                                              \
            case 2: SPARDA_VD_R(DT_, 2); break;                                              \
            case 4: SPARDA_VD_R(DT_, 4); break;                                              \
            case 8: SPARDA_VD_R(DT_, 8); break;                                              \
            default: SPARDA_VD_R(DT_, 16); break;                                            \
        }                                                                                    \
        if (p.exact) hipLaunchKernelGGL((verify_draw_kernel<DT_, true>), grid2, threads, 0, stream, a); \
        else hipLaunchKernelGGL((verify_draw_kernel<DT_, false>), grid2, threads, 0, stream, a);        \
    } while (0)
    if (dtype == SPARDA_F32) SPARDA_VD(SPARDA_F32);
    else SPARDA_VD(SPARDA_BF16);
#undef SPARDA_VD
#undef SPARDA_VD_R
    return check_hip(hipGetLastError(), "verify_drafts");
}

}  // namespace sparda
