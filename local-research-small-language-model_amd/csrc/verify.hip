// Verification of drafted tokens (sparda_verify_drafts): which of a sequence's
// drafts its target distributions accept, and the token drawn behind them.
//
//   p_i = softmax(logits[b, i] / temperature[b]), q_i the draft's distribution of draft i
//   (all of it on the draft where none is given). Draft d_i is accepted while u_i q_i(d_i) < p_i(d_i). Behind n
//   accepted ones the token is the first at which the cumulated sum of r passes u_K times
//   its total: r = max(p_n - q_n, 0) after a rejection (p_n where that leaves nothing),
//   r = p_n where no draft is left. Temperature 0: the drafts are compared with
//   the largest logits' lowest indexes.
//
// The first launch reads all logits once, in fp32: maximum and sum of every chunk of
// every row. The test of a draft needs no more. The token is where a long sum
// passes a number, and which token that is must not hang on how fp32 rounds, so the one row
// it is drawn from is summed again in fp64: a second launch over (chunk, sequence),
// and after rejections against given distributions a third, which needs the row's total.
// The workgroup that comes last among a sequence's draws the token from the chunks' sums.
#include "common.h"
#include "kernels.h"

namespace sparda {

namespace {

constexpr int kVdThreads = 256;
constexpr int kVdChunks = 256;        // chunks of a row in the first launch, at most
constexpr int kVdRows = 65;           // rows of a sequence (drafts + 1), at most
constexpr float kVdLog2e = 1.4426950408889634f;

struct alignas(16) ChunkStat {
    float m;         // largest logit of the chunk
    int32_t arg;     // its lowest index (greedy sequences)
    double sum;      // of exp((x - m) / temperature)
};
struct alignas(16) ChunkSum {
    double p, r;     // sums of p's weights and of r's
};
struct SequenceState {
    uint32_t done[2];    // workgroups of the second and third launch that are through
    int32_t n, mode;     // drafts accepted, how the token is drawn
    double m;            // the row's largest logit
};
enum { kVdNone = 0, kVdPlain = 1, kVdWithout = 2, kVdResidual = 3 };  // modes: nothing to draw, p, p without the draft, max(p - q, 0)

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
    int64_t len1, len2;          // elements of a chunk in the first launch, in the others
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
    return a.temperature != nullptr ? a.temperature[b] : a.all_temperature;
}

template <int DT>
struct VdType {
    static constexpr int kEs = DT == SPARDA_F32 ? 4 : 2, kVe = 16 / kEs;   // bytes of an element, elements of a piece
};

// Elements [at, at + kVe) of a row of V in aligned pieces of 16 bytes; those outside [0, V) are
// -inf. A piece that leaves the row is read element by element.
template <int DT>
__device__ __forceinline__ void vd_load(const char* row, int64_t at, int64_t V, float (&x)[VdType<DT>::kVe]) {
    constexpr int kVe = VdType<DT>::kVe, kEs = VdType<DT>::kEs;
    if (at >= 0 && at + kVe <= V) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + at * kEs);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (DT == SPARDA_F32) {
                x[e] = __uint_as_float(u[e]);
            } else {
                x[2 * e] = __uint_as_float(u[e] << 16);
                x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < kVe; ++e) x[e] = at + e >= 0 && at + e < V ? load_elem<DT>(row, at + e) : -__builtin_inff();
    }
}

// elements before a row's start in its first aligned piece
template <int DT>
__device__ __forceinline__ int vd_shift(const char* row) {
    return static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16) / VdType<DT>::kEs;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
    return v;
}
// inclusive sums over the lanes
__device__ __forceinline__ double wave_scan_f64(double v) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const double w = __shfl_up(v, o, kWave);
        if (lane >= o) v += w;
    }
    return v;
}

}  // namespace

// Maximum and sum of a chunk of a row, in one read: the chunk's pieces stay in registers.
template <int DT, int PIECES>
__global__ void __launch_bounds__(kVdThreads) verify_stats_kernel(Verify a) {
    constexpr int kVe = VdType<DT>::kVe, kEs = VdType<DT>::kEs;
    __shared__ float rm[kVdThreads / kWave];
    __shared__ double rs[kVdThreads / kWave];
    __shared__ int ra[kVdThreads / kWave];
    const int tid = threadIdx.x, wave = tid / kWave, chunk = blockIdx.x;
    const int b = blockIdx.y / (a.K + 1), i = blockIdx.y % (a.K + 1);
    if (chunk == 0 && i == 0 && tid == 0) a.state[b].done[0] = a.state[b].done[1] = 0;
    if (i > vd_count(a, b)) return;                           // no draft's row
    const float T = vd_temperature(a, b);
    const bool greedy = !(T > 0.0f);
    const float c = greedy ? kVdLog2e : fminf(kVdLog2e / T, 3e38f);
    const char* row = static_cast<const char*>(a.logits) + (b * a.l_sb + i * a.l_st) * kEs;
    const int64_t first = chunk * a.len1 - vd_shift<DT>(row);
    float x[PIECES][kVe];
#pragma unroll
    for (int k = 0; k < PIECES; ++k) vd_load<DT>(row, first + (tid + k * kVdThreads) * kVe, a.V, x[k]);
    float m = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int e = 0; e < kVe; ++e) m = fmaxf(m, x[k][e]);
    m = wave_max(m);
    if (tid % kWave == 0) rm[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kVdThreads / kWave; ++w) m = fmaxf(m, rm[w]);
    const float ref = m == -__builtin_inff() ? 0.0f : m;
    float s = 0.0f;
    int arg = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < PIECES; ++k)
#pragma unroll
        for (int e = 0; e < kVe; ++e) s += __builtin_amdgcn_exp2f((x[k][e] - ref) * c);
    if (greedy) {
#pragma unroll
        for (int k = PIECES - 1; k >= 0; --k)
#pragma unroll
            for (int e = kVe - 1; e >= 0; --e)
                if (x[k][e] == m) arg = static_cast<int>(first + (tid + k * kVdThreads) * kVe + e);
        arg = wave_min_i32(arg);
    }
    s = wave_sum(s);
    if (tid % kWave == 0) rs[wave] = s, ra[wave] = arg;
    __syncthreads();
    if (tid == 0) {
        ChunkStat st{m, ra[0], rs[0]};
#pragma unroll
        for (int w = 1; w < kVdThreads / kWave; ++w) st.sum += rs[w], st.arg = min(st.arg, ra[w]);
        a.stats[static_cast<int64_t>(blockIdx.y) * a.chunks1 + chunk] = st;
    }
}

namespace {

// What a token is drawn from: row, and what is taken off its weights.
struct VdRow {
    const char* row;
    const float* q;       // mode kVdResidual
    int without;          // mode kVdWithout
    int mode;
    double m, inv_t, inv_total;   // inv_total: one over the sum of p's weights (kVdResidual)
};

// r of eight or four elements; w: p's weights, not divided by their total
template <int DT>
__device__ __forceinline__ void vd_weights(const VdRow& r, int64_t at, int64_t V, bool residual, double (&w)[VdType<DT>::kVe]) {
    constexpr int kVe = VdType<DT>::kVe;
    float x[kVe];
    vd_load<DT>(r.row, at, V, x);
#pragma unroll
    for (int e = 0; e < kVe; ++e) {
        w[e] = exp((static_cast<double>(x[e]) - r.m) * r.inv_t);
        if (r.mode == kVdWithout && at + e == r.without) w[e] = 0.0;
        if (residual) {
            const double q = at + e >= 0 && at + e < V ? static_cast<double>(r.q[at + e]) : 0.0;
            const double d = w[e] * r.inv_total - q;
            w[e] = d > 0.0 ? d : 0.0;
        }
    }
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
    const int wave = threadIdx.x / kWave;
    v = wave_sum_f64(v);
    __syncthreads();                              // (the array's last use)
    if (threadIdx.x % kWave == 0) red[wave] = v;
    __syncthreads();
    double s = red[0];
#pragma unroll
    for (int w = 1; w < kVdThreads / kWave; ++w) s += red[w];
    return s;
}

// The token of the chunks' sums (lane c of every wavefront holds chunk c's): the chunk where they pass
// u times their total, then the token in it. All threads of the workgroup.
template <int DT>
__device__ __forceinline__ int vd_draw(const VdRow& r, double mine_of_all, int64_t len, int64_t V, bool residual, float u, double* red,
                                       int* found) {
    constexpr int kVe = VdType<DT>::kVe, kW = kVdThreads / kWave;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
    const double upto_chunk = wave_scan_f64(mine_of_all);
    const double target = static_cast<double>(u) * __shfl(upto_chunk, kWave - 1, kWave);
    const uint64_t pass = __ballot(upto_chunk > target), some = __ballot(mine_of_all > 0.0);
    // (none passes where u is 1, or the last by a rounding: the last token that weighs anything)
    const int chunk = pass != 0 ? __builtin_ctzll(pass) : 63 - __builtin_clzll(some | 1);
    double base = __shfl(upto_chunk - mine_of_all, chunk, kWave);
    const int64_t first = chunk * len - vd_shift<DT>(r.row);
    int best = -1;                                // the last token with a weight so far
    for (int64_t p0 = 0; p0 < len; p0 += kVdThreads * kVe) {
        const int64_t at = first + p0 + tid * kVe;
        double w[kVe], mine = 0.0;
        vd_weights<DT>(r, at, V, residual, w);
        int top = -1;
#pragma unroll
        for (int e = 0; e < kVe; ++e) {
            mine += w[e];
            if (w[e] > 0.0) top = static_cast<int>(at + e);
        }
        const double upto = wave_scan_f64(mine);
        __syncthreads();                          // (the arrays' last use)
        if (lane == kWave - 1) red[wave] = upto;
        if (tid == 0) found[0] = 0x7fffffff;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) top = max(top, __shfl_xor(top, o, kWave));
        if (lane == 0) found[1 + wave] = top;
        __syncthreads();
        double before = base;
        for (int v = 0; v < wave; ++v) before += red[v];
        if (pass != 0 && mine > 0.0 && before + upto > target) {
            // (rounding may leave the piece's own sums below: its last weight)
            double acc = before + upto - mine;
            int hit = -1, last = -1;
#pragma unroll
            for (int e = 0; e < kVe; ++e) {
                acc += w[e];
                if (w[e] > 0.0) {
                    last = e;
                    if (hit < 0 && acc > target) hit = e;
                }
            }
            atomicMin(&found[0], static_cast<int>(at + (hit >= 0 ? hit : last)));
        }
        __syncthreads();
        if (found[0] != 0x7fffffff) return found[0];
#pragma unroll
        for (int v = 0; v < kW; ++v) best = max(best, found[1 + v]);
#pragma unroll
        for (int v = 0; v < kW; ++v) base += red[v];
    }
    return best;
}

// What workgroups of a launch hand to the last of them goes through stores and loads at the device's
// scope, which pass the caches that they do not share; a store is waited for before its
// workgroup is counted. (A release or acquire at that scope would write back and drop whole caches instead, once a workgroup.)
__device__ __forceinline__ double vd_read(const double* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// writes the workgroup's number and counts it; true in the last of `all`
__device__ __forceinline__ bool vd_last(double* to, double v, uint32_t* done, uint32_t all, int* flag) {
    if (threadIdx.x == 0) {
        __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __builtin_amdgcn_s_waitcnt(0x0f70);       // vmcnt(0): the store has arrived
        asm volatile("" ::: "memory");
        *flag = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == all;
    }
    __syncthreads();
    return *flag != 0;
}

// the sum of a chunk's weights, by all threads
template <int DT>
__device__ __forceinline__ double vd_chunk_sum(const VdRow& r, int chunk, int64_t len, int64_t V, bool residual, double* red) {
    constexpr int kVe = VdType<DT>::kVe;
    const int64_t first = chunk * len - vd_shift<DT>(r.row);
    double s = 0.0;
    for (int64_t p0 = threadIdx.x * kVe; p0 < len; p0 += kVdThreads * kVe) {
        double w[kVe];
        vd_weights<DT>(r, first + p0, V, residual, w);
#pragma unroll
        for (int e = 0; e < kVe; ++e) s += w[e];
    }
    return block_sum_f64(s, red);
}

}  // namespace

// One workgroup per (chunk, sequence). Every one finds the accepted drafts for itself, from the
// chunks' statistics; then the chunk's sum of the row behind them, and the last one the token,
// unless it is drawn from max(p - q, 0), which takes p's total.
template <int DT>
__global__ void __launch_bounds__(kVdThreads) verify_accept_kernel(Verify a) {
    constexpr int kEs = VdType<DT>::kEs, kW = kVdThreads / kWave;
    __shared__ double red[kW];
    __shared__ float rmax[kVdRows];
    __shared__ int rarg[kVdRows], ok[kVdRows], found[1 + kW], flag;
    const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave, chunk = blockIdx.x, b = blockIdx.y;
    const int count = vd_count(a, b);
    const float T = vd_temperature(a, b);
    const bool greedy = !(T > 0.0f);
    const double inv_t = greedy ? 1.0 : 1.0 / static_cast<double>(T);
    for (int i = wave; i <= count; i += kW) {                 // a wavefront a row
        const ChunkStat* st = a.stats + (static_cast<int64_t>(b) * (a.K + 1) + i) * a.chunks1;
        // (the draft's own numbers under the chunks')
        int d = -1;
        float x = -__builtin_inff(), u = 0.0f, q = 1.0f;
        if (i < count) {
            d = a.drafts[b * a.d_sb + i];
            if (d >= 0 && d < a.V) {
                x = load_elem<DT>(a.logits, b * a.l_sb + i * a.l_st + d);
                u = a.uniform[b * a.u_sb + i];
                if (a.probs) q = a.probs[b * a.p_sb + i * a.p_st + d];
            }
        }
        ChunkStat own{-__builtin_inff(), 0x7fffffff, 0.0};
        if (lane < a.chunks1) own = st[lane];
        float m = own.m;
        for (int c = lane + kWave; c < a.chunks1; c += kWave) m = fmaxf(m, st[c].m);
        m = wave_max(m);
        double z = 0.0;
        int arg = 0x7fffffff;
        auto add = [&](const ChunkStat& s) {
            // (a chunk without a finite logit: nothing; NaN among them stays)
            z += s.m == -__builtin_inff() ? s.sum : s.sum * exp((static_cast<double>(s.m) - m) * inv_t);
            if (s.m == m) arg = min(arg, s.arg);
        };
        add(own);
        for (int c = lane + kWave; c < a.chunks1; c += kWave) add(st[c]);
        z = wave_sum_f64(z);
        if (greedy) arg = wave_min_i32(arg);
        if (lane == 0) {
            const bool valid = m > -__builtin_inff() && m < __builtin_inff() && z < __builtin_inf();
            const bool accept = greedy ? d == arg
                                       : d >= 0 && d < a.V && static_cast<double>(u) * q < exp((static_cast<double>(x) - m) * inv_t) / z;
            rmax[i] = m, rarg[i] = valid ? (greedy ? arg : 0) : -1, ok[i] = valid && i < count && accept ? 1 : 0;
        }
    }
    __syncthreads();
    int n = 0;
    while (n < count && ok[n] != 0) ++n;
    VdRow r{};
    r.row = static_cast<const char*>(a.logits) + (b * a.l_sb + n * a.l_st) * kEs;
    r.m = rmax[n], r.inv_t = inv_t;
    const int d = n < count ? a.drafts[b * a.d_sb + n] : -1;
    r.mode = rarg[n] < 0 || greedy ? kVdNone : n == count ? kVdPlain : a.probs ? kVdResidual : kVdWithout;
    r.without = d;
    auto write = [&](int token) {
        for (int i = tid; i <= a.K; i += kVdThreads)
            a.tokens[static_cast<int64_t>(b) * (a.K + 1) + i] = i < n ? a.drafts[b * a.d_sb + i] : i == n ? token : -1;
        if (tid == 0) a.accepted[b] = n;
    };
    if (chunk == 0 && tid == 0) a.state[b].n = n, a.state[b].mode = r.mode, a.state[b].m = r.m;
    if (r.mode == kVdNone) {
        if (chunk == 0) write(rarg[n]);
        return;
    }
    const double s = vd_chunk_sum<DT>(r, chunk, a.len2, a.V, false, red);
    ChunkSum* sums = a.sums + static_cast<int64_t>(b) * a.chunks2;
    if (r.mode == kVdResidual) {
        if (tid == 0) sums[chunk].p = s;                      // the third launch goes on
        return;
    }
    if (!vd_last(&sums[chunk].p, s, &a.state[b].done[0], static_cast<uint32_t>(a.chunks2), &flag)) return;
    const double mine = lane < a.chunks2 ? vd_read(&sums[lane].p) : 0.0;
    if (__ballot(mine > 0.0) == 0) {                          // p is all on the draft that was rejected: p
        write(d);
        return;
    }
    write(vd_draw<DT>(r, mine, a.len2, a.V, false, a.uniform[b * a.u_sb + a.K], red, found));
}

// The same for max(p - q, 0), p's total known.
template <int DT>
__global__ void __launch_bounds__(kVdThreads) verify_residual_kernel(Verify a) {
    constexpr int kEs = VdType<DT>::kEs, kW = kVdThreads / kWave;
    __shared__ double red[kW];
    __shared__ int found[1 + kW], flag;
    const int tid = threadIdx.x, lane = tid % kWave, chunk = blockIdx.x, b = blockIdx.y;
    if (a.state[b].mode != kVdResidual) return;
    const int n = a.state[b].n;
    VdRow r{};
    r.row = static_cast<const char*>(a.logits) + (b * a.l_sb + n * a.l_st) * kEs;
    r.q = a.probs + b * a.p_sb + n * a.p_st;
    r.mode = kVdResidual;
    r.m = a.state[b].m, r.inv_t = 1.0 / static_cast<double>(vd_temperature(a, b));
    ChunkSum* sums = a.sums + static_cast<int64_t>(b) * a.chunks2;
    const double plain = lane < a.chunks2 ? sums[lane].p : 0.0;
    r.inv_total = 1.0 / wave_sum_f64(plain);
    const double s = vd_chunk_sum<DT>(r, chunk, a.len2, a.V, true, red);
    if (!vd_last(&sums[chunk].r, s, &a.state[b].done[1], static_cast<uint32_t>(a.chunks2), &flag)) return;
    const double less = lane < a.chunks2 ? vd_read(&sums[lane].r) : 0.0;
    const bool residual = __ballot(less > 0.0) != 0;          // otherwise from p
    const int token = vd_draw<DT>(r, residual ? less : plain, a.len2, a.V, residual, a.uniform[b * a.u_sb + a.K], red, found);
    for (int i = tid; i <= a.K; i += kVdThreads)
        a.tokens[static_cast<int64_t>(b) * (a.K + 1) + i] = i < n ? a.drafts[b * a.d_sb + i] : i == n ? token : -1;
    if (tid == 0) a.accepted[b] = n;
}

namespace {

struct VerifyPlan {
    int pieces;                  // 16-byte pieces of a thread in the first launch
    int64_t len1, len2;
    int chunks1, chunks2;
    size_t stats, sums, state, bytes;   // offsets, and all
};
VerifyPlan verify_plan(int64_t B, int64_t K, int64_t V, int dtype) {
    VerifyPlan p{};
    const int64_t ve = dtype == SPARDA_F32 ? 4 : 8, round = kVdThreads * ve, all = V + ve;   // (a row may start inside a piece)
    p.pieces = 1;
    while (p.pieces < 8 && (B * (K + 1) * cdiv(all, round * p.pieces) > 2048 || cdiv(all, round * p.pieces) > kVdChunks)) p.pieces *= 2;
    p.len1 = round * p.pieces;
    p.chunks1 = static_cast<int>(cdiv(all, p.len1));
    p.len2 = round;
    while (cdiv(all, p.len2) > kWave) p.len2 += round;
    p.chunks2 = static_cast<int>(cdiv(all, p.len2));
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
                   static_cast<int>(K), V, p.len1, p.len2, p.chunks1, p.chunks2,
                   reinterpret_cast<ChunkStat*>(ws + p.stats), reinterpret_cast<ChunkSum*>(ws + p.sums),
                   reinterpret_cast<SequenceState*>(ws + p.state), tokens, accepted};
    if (!grid_fits(static_cast<int64_t>(p.chunks1) * B * (K + 1), kVdThreads) || !grid_fits(static_cast<int64_t>(p.chunks2) * B, kVdThreads))
        return set_error(SPARDA_ERR_SHAPE, "verify_drafts: grid too large");
    const dim3 grid1(static_cast<unsigned>(p.chunks1), static_cast<unsigned>(B * (K + 1)));
    const dim3 grid2(static_cast<unsigned>(p.chunks2), static_cast<unsigned>(B)), threads(kVdThreads);
#define SPARDA_VD(DT_)                                                                                       \
    do {                                                                                                     \
        if (p.pieces == 1) hipLaunchKernelGGL((verify_stats_kernel<DT_, 1>), grid1, threads, 0, stream, a);   \
        else if (p.pieces == 2) hipLaunchKernelGGL((verify_stats_kernel<DT_, 2>), grid1, threads, 0, stream, a); \
        else if (p.pieces == 4) hipLaunchKernelGGL((verify_stats_kernel<DT_, 4>), grid1, threads, 0, stream, a); \
        else hipLaunchKernelGGL((verify_stats_kernel<DT_, 8>), grid1, threads, 0, stream, a);                 \
        hipLaunchKernelGGL((verify_accept_kernel<DT_>), grid2, threads, 0, stream, a);                        \
        if (probs && K > 0) hipLaunchKernelGGL((verify_residual_kernel<DT_>), grid2, threads, 0, stream, a);  \
    } while (0)
    if (dtype == SPARDA_F32) SPARDA_VD(SPARDA_F32);
    else SPARDA_VD(SPARDA_BF16);
#undef SPARDA_VD
    return check_hip(hipGetLastError(), "verify_drafts");
}

}  // namespace sparda
