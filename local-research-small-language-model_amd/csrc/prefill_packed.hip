// Attention over packed prompts (sparda_prefill_packed): n sequences of any
// lengths back to back in q, k, v [N, H, D], each attending to itself alone,
// causally or not, query head h over KV head h / R.
#include "common.h"
#include "kernels.h"
#include "mfma.h"
#include "packed.h"

namespace sparda {

namespace {

constexpr float kPkLog2e = 1.4426950408889634f;

}  // namespace

// ---------------------------------------------------------------------------
// bf16, D = 32, 64 and 128, on the matrix cores
// ---------------------------------------------------------------------------

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr float kPkGuard = 18446744073709551616.0f;  // 2^64: a sum of weights past it means a score far above the reference
constexpr float kPkOutGuard = 1329227995784915872903807060280344576.0f;  // 2^120: below it the key groups' outputs add up without overflow
// 2^12: outputs are looked at where a lane's sum of weights passes it. Smaller sums (short prompts of ordinary
// scores) take values below 2^112 nowhere near overflow; looking at all outputs took 0.2-0.3 us of 11-17.
constexpr float kPkFar = 4096.0f;

// 16-byte piece `c` of row `r` in an LDS tile of D-element rows: pieces are
// exchanged within a row so that both reads of a tile are spread over the banks:
// 16 consecutive rows at one piece (K) take 16 different places of 256 bytes, and
// 4 consecutive rows at 4 consecutive pieces (V, transposed) do too.
template <int D>
__device__ __forceinline__ int pk_piece(int r, int c) {
    if constexpr (D == 32) return c ^ (r >> 2 & 3);
    else if constexpr (D == 64) return c ^ ((r >> 1 & 1) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1));
    else return c ^ ((r & 3) << 2 | (r >> 2 & 3));
}

template <int D, int KB, int KG>
struct PackedStage {
    uint16_t k[2][KG][KB * D];
    uint16_t v[2][KG][KB * D];
};
template <int N, int CW, int NT, int KG>
struct PackedMerge {
    float o[KG - 1][CW][N][kWave];
    float l[KG - 1][CW][NT][kWave];
};
template <int N, int CW, int NT>
struct PackedMerge<N, CW, NT, 1> {};

// A barrier behind loads to LDS: they are counted by vmcnt, and the barrier itself
// does not wait for a wavefront's own.
__device__ __forceinline__ void staged_barrier() {
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0), the other counters at their maximum
    __syncthreads();
}

struct PackedPrefill {
    const uint16_t* q;
    int64_t q_st, q_sh;
    const uint16_t *k, *v;
    int64_t kv_st, kv_sh;
    const int32_t* cu;
    int n;
    int64_t N;
    int Hkv, R, causal;
    int64_t slots;
    float scale_log2;
    uint16_t* out;
    int64_t out_st;
    uint32_t* status;
};

}  // namespace

// One workgroup per (KV head, window of BM = 32 NT CW columns of one sequence),
// a column being a (token, query head of the group) pair: column c is token c / R,
// head c % R, so that every head of the group shares the staged keys and any R
// fits. CW wavefronts of 32 NT columns each walk blocks of KB keys staged in LDS
// (the next block's loads in flight); KG groups of CW wavefronts take every KG-th
// block. Per 32 keys and 32 columns, with v_mfma_f32_32x32x16_bf16:
//     S^T[key, col] = K[key, :] . Q[col, :]
//     P = exp2(S scale log2 e - ref[col])
//     O^T[d, col] += V^T[d, key] . P^T[key, col]
// P is rounded to bf16 for the second product (half a step, 2^-8 of sum p |v| at most);
// ref[col] is the column's maximum over the sequence's first 32 keys (key 0 is
// allowed to every column), which every key group takes from group 0's first block
// before the walk, so that nothing is rescaled (each wavefront reading those keys from
// memory again: 16 x 256 tokens 13.3 against 10.2 us). A sum past 2^64, an output past 2^120
// (weights far above 1 times large values), or a first tile of -inf alone sends the
// workgroup over its keys twice more: for the exact maxima, then against them, where
// no weight passes 1. Bound by the matrix cores and the exponentials, which share the
// issue slots, at the clock that the card holds under them (about 1.9 GHz): 16384 tokens of
// 12/4 heads of 64 take 407-437 us = 940-1010 TFLOP/s of the 1210 that a large library
// product reaches, the matrix cores busy in half of the cycles; 8 sequences of 16000 in all,
// 32/8 heads of 128, 354-387 us = 880-960 TFLOP/s.
template <int D, int NT, int CW, int KG, int KB>
__global__ void __launch_bounds__(CW* KG* kWave, 2) prefill_packed_kernel(PackedPrefill a) {
    constexpr int kCols = 32 * NT, kBM = CW * kCols;
    constexpr int kPieces = D / 8, kRun = kWave / kPieces, kRuns = KB / (CW * kRun);
    static_assert(kRuns * CW * kRun == KB, "whole runs");
    constexpr int kKS = D / 16, kDT = D / 32, kHalves = KB / 32;
    __shared__ union {
        PackedStage<D, KB, KG> st;
        PackedMerge<NT * kDT * 16, CW, NT, KG> mg;
    } sm;
    __shared__ int flag;
    const int lane = threadIdx.x % kWave;
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int wave = wv % CW, kg = wv / CW;
    const int col = lane % 32, hf = lane / 32;
    const int g = blockIdx.x % a.Hkv;
    const int64_t slot = a.slots - 1 - blockIdx.x / a.Hkv;    // a sequence's last windows, the longest walks, first
    bool bad;
    const PackedWindow w = packed_window(a.cu, a.n, a.N, a.R, kBM, slot, bad);
    if (bad && threadIdx.x == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_SEQUENCE_RANGE));
    if (w.seq < 0) return;                                    // workgroup-uniform
    const int len = w.len, ncol = len * a.R;
    const int col0 = static_cast<int>(w.win) * kBM, wcol0 = col0 + wave * kCols;
    const bool live = wcol0 < ncol;
    const int w_first = wcol0 / a.R;
    const int w_last = (wcol0 + kCols <= ncol ? wcol0 + kCols - 1 : ncol - 1) / a.R;
    const int w_end = !live ? 0 : a.causal ? w_last + 1 : len;      // the wavefront's keys
    const int g_last = (col0 + kBM <= ncol ? col0 + kBM - 1 : ncol - 1) / a.R;
    const int nblk = ((a.causal ? g_last + 1 : len) + KB - 1) / KB;

    const uint16_t* kb = a.k + static_cast<int64_t>(w.row0) * a.kv_st + static_cast<int64_t>(g) * a.kv_sh;
    const uint16_t* vb = a.v + static_cast<int64_t>(w.row0) * a.kv_st + static_cast<int64_t>(g) * a.kv_sh;

    // this lane's columns (those past the sequence repeat its last one, not written)
    int tok[NT], lim[NT];
    bf16x8 qreg[NT][kKS];
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
        const int c = wcol0 + 32 * tt + col < ncol ? wcol0 + 32 * tt + col : ncol - 1;
        tok[tt] = c / a.R;
        lim[tt] = a.causal ? tok[tt] : len - 1;               // its last key
        const uint16_t* qp = a.q + (w.row0 + static_cast<int64_t>(tok[tt])) * a.q_st +
                             static_cast<int64_t>(g * a.R + c % a.R) * a.q_sh + 8 * hf;
#pragma unroll
        for (int kk = 0; kk < kKS; ++kk) qreg[tt][kk] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(qp + 16 * kk));
    }

    // Staging goes from memory to LDS without registers, 16 bytes a lane, lanes in
    // LDS order: lane i of a load holds place i % kPieces of row i / kPieces, and
    // fetches the piece that belongs there. A wavefront loads every CW-th run of
    // kRun rows. Rows behind the sequence repeat its last one.
    const int srow = wave * kRun + lane / kPieces, kv_st = static_cast<int>(a.kv_st);
    auto stage = [&](int j, int buf) __attribute__((always_inline)) {
        typedef const __attribute__((address_space(1))) void* G;
        typedef __attribute__((address_space(3))) void* L;
        const int row0 = j * KB, last = len - 1 - row0;
        const char* kr = reinterpret_cast<const char*>(kb + static_cast<int64_t>(row0) * a.kv_st);
        const char* vr = reinterpret_cast<const char*>(vb + static_cast<int64_t>(row0) * a.kv_st);
#pragma unroll
        for (int i = 0; i < kRuns; ++i) {
            const int r = i * CW * kRun, row = srow + r < last ? srow + r : last;
            // (rows a multiple of 16 apart place their pieces alike)
            const uint32_t at = 2 * static_cast<uint32_t>(row * kv_st + 8 * pk_piece<D>(srow + r, lane % kPieces));
            __builtin_amdgcn_global_load_lds((G)(kr + at), (L)&sm.st.k[buf][kg][(r + wave * kRun) * D], 16, 0, 0);
            __builtin_amdgcn_global_load_lds((G)(vr + at), (L)&sm.st.v[buf][kg][(r + wave * kRun) * D], 16, 0, 0);
        }
    };

    // the columns' maxima over the keys [0, upto), straight from memory (second pass)
    float ref[NT], l[NT];
    auto take_refs = [&](int upto) __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) ref[tt] = -__builtin_inff();
        for (int key0 = 0; key0 < upto; key0 += 32) {
            bf16x8 ka[kKS];
            const uint16_t* kr = kb + static_cast<int64_t>(key0 + col < len ? key0 + col : len - 1) * a.kv_st + 8 * hf;
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk) ka[kk] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(kr + 16 * kk));
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
                f32x16 s{};
#pragma unroll
                for (int kk = 0; kk < kKS; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kk], qreg[tt][kk], s, 0, 0, 0);
                const int mine = lim[tt] - key0 - 4 * hf;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    ref[tt] = fmaxf(ref[tt], 8 * (i / 4) + i % 4 <= mine ? s[i] * a.scale_log2 : -__builtin_inff());
            }
        }
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) ref[tt] = pair32_max(ref[tt]);
    };

    f32x16 o[NT][kDT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            l[tt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt) o[tt][dt] = f32x16{};
        }
    };

    // operand reads of 32 keys: K rows at this lane's key, V transposed (a 16-lane
    // group reads 4 rows x 16 dims, lane j of it row j / 4, dims 4 (j % 4) .. +3);
    // 16 rows further the places within a row are the same
    int k_at[kKS], v_at[kDT][2];
#pragma unroll
    for (int kk = 0; kk < kKS; ++kk) k_at[kk] = col * D + 8 * pk_piece<D>(col, 2 * kk + hf);
#pragma unroll
    for (int dt = 0; dt < kDT; ++dt) {
        const int r = 4 * hf + lane % 16 / 4, d = 32 * dt + 16 * (lane / 16 % 2) + 4 * (lane % 4);
        v_at[dt][0] = r * D + 8 * pk_piece<D>(r, d / 8) + d % 8;
        v_at[dt][1] = (r + 8) * D + 8 * pk_piece<D>(r + 8, d / 8) + d % 8;
    }
    bool odd = false;  // infinities or NaN in V at a place that some column may not attend

    // 32 keys from key0 on, staged at row 32 half of the buffer
    auto compute = [&](int buf, int half, int key0) __attribute__((always_inline)) {
        bf16x8 ka[kKS], va[kDT][2];
        const uint16_t* ks = &sm.st.k[buf][kg][32 * half * D];
        const uint16_t* vs = &sm.st.v[buf][kg][32 * half * D];
#pragma unroll
        for (int kk = 0; kk < kKS; ++kk) ka[kk] = lds_read8(ks + k_at[kk]);
        f32x16 s[NT];
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            s[tt] = f32x16{};
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk)
                s[tt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kk], qreg[tt][kk], s[tt], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);  // V's operands take K's registers
        // V^T operand: dim 32 dt + col, keys 16 c + 4 hf .. +3 and 8 further
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const i16x4 lo = lds_read_tr(vs + v_at[dt][0] + 16 * c * D);
                const i16x4 hi = lds_read_tr(vs + v_at[dt][1] + 16 * c * D);
                va[dt][c] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        const bool edge = a.causal ? key0 + 31 > w_first : key0 + 32 > len;
        if (edge) {
            // a weight of 0 times inf is NaN: such values are cleared here, and added
            // after the walk to the columns that do attend them
            // (an exponent of all ones carries into the sign's place)
            uint32_t any = 0;
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint4 x = __builtin_bit_cast(uint4, va[dt][c]);
                    any |= ((x.x & 0x7f807f80u) + 0x00800080u) | ((x.y & 0x7f807f80u) + 0x00800080u) |
                           ((x.z & 0x7f807f80u) + 0x00800080u) | ((x.w & 0x7f807f80u) + 0x00800080u);
                }
            any &= 0x80008000u;
            if (__ballot(any != 0) != 0) {
                odd = true;
                typedef short s16x8 __attribute__((ext_vector_type(8)));
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s16x8 x = __builtin_bit_cast(s16x8, va[dt][c]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = (x[e] & 0x7f80) == 0x7f80 ? 0 : x[e];
                        va[dt][c] = __builtin_bit_cast(bf16x8, x);
                    }
            }
        }
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            const float neg = ref[tt] == -__builtin_inff() ? 0.0f : -ref[tt];
            bf16x8 pb[2];
            float sum = 0.0f;
            if (edge) {
                const int mine = lim[tt] - key0 - 4 * hf;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][i], a.scale_log2, neg));
                    p = 8 * (i / 4) + i % 4 <= mine ? p : 0.0f;
                    sum += p;
                    pb[i / 8][i % 8] = static_cast<__bf16>(p);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][i], a.scale_log2, neg));
                    sum += p;
                    pb[i / 8][i % 8] = static_cast<__bf16>(p);
                }
            }
            l[tt] += sum;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
                    o[tt][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[dt][c], pb[c], o[tt][dt], 0, 0, 0);
        }
    };

    // A block all of whose keys every column attends, in units of 32 keys x 32
    // columns: while a unit's exponentials are taken, the next one's scores and the
    // last one's output products are on the matrix cores (sched_group_barrier lays
    // the products between the vector instructions).
    auto compute_block = [&](int buf, int next) __attribute__((always_inline)) {
        constexpr int kU = kHalves * NT;
        static_assert(kHalves <= 2, "");
        constexpr int kMfma = kKS + 2 * kDT;                  // products of a unit
        const uint16_t* ks = &sm.st.k[buf][kg][0];
        const uint16_t* vs = &sm.st.v[buf][kg][0];
        bf16x8 ka[kKS], va[2][kDT][2], pb[2][2];                // (two sets of V: NT = 1)
        f32x16 s[2];
        float neg[NT];
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) neg[tt] = ref[tt] == -__builtin_inff() ? 0.0f : -ref[tt];
        auto read_k = [&](int half) __attribute__((always_inline)) {
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk) ka[kk] = lds_read8(ks + k_at[kk] + 32 * half * D);
        };
        auto read_v = [&](int half, bf16x8 (&x)[kDT][2]) __attribute__((always_inline)) {
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const i16x4 lo = lds_read_tr(vs + v_at[dt][0] + (32 * half + 16 * c) * D);
                    const i16x4 hi = lds_read_tr(vs + v_at[dt][1] + (32 * half + 16 * c) * D);
                    x[dt][c] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                }
        };
        auto qk = [&](int u) __attribute__((always_inline)) {
            f32x16 x{};
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk) x = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kk], qreg[u % NT][kk], x, 0, 0, 0);
            s[u & 1] = x;
        };
        auto pv = [&](int u) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
                    o[u % NT][dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[NT == 1 ? u & 1 : 0][dt][c], pb[u & 1][c], o[u % NT][dt], 0, 0, 0);
        };
        read_k(0);
        qk(0);
        read_v(0, va[0]);
        if (NT == 1 && kU > 1) read_k(1);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            __builtin_amdgcn_sched_barrier(0);
            if (u == kU - 1) {
                // the last reads of LDS, then the next block's loads: a read behind them would wait for them
                if (NT == 1 && kU > 1) {
                    read_v(u, va[1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                stage(next, buf ^ 1);
            }
            if (u + 1 < kU) qk(u + 1);
            if (u + 2 < kU && (u + 2) % NT == 0) read_k((u + 2) / NT);  // (its last unit's scores are under way)
            if (u > 0) {
                pv(u - 1);
                if (NT > 1 && u % NT == 0) read_v(u / NT, va[0]);
            }
            // the sum takes the rounded weights, two an instruction: the weights of the product are those
            // that it is divided by
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u & 1][i], a.scale_log2, neg[u % NT]));
                pb[u & 1][i / 8][i % 8] = static_cast<__bf16>(p);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
                const bf16x2 one{static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pb[u & 1][c][e], pb[u & 1][c][e + 1]}, one, sum, false);
            }
            l[u % NT] += sum;
#pragma unroll
            for (int i = 0; i < kMfma; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 48 / kMfma, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        pv(kU - 1);
    };

    // step i: group kg computes block i KG + kg from buffer i & 1 while its next is loaded
    // (first the steps whose blocks every column of the workgroup attends)
    const int steps = (nblk + KG - 1) / KG, whole = (a.causal ? col0 / a.R + 1 : len) / KB / KG;
    // pass 0: against the first block's maxima; 1, after a sum or an output past its guard:
    // against the exact ones; 2, after an output past its guard that 1 did not bring back
    // (a value that is not finite): as 0, so that such a value changes no other output
    int why = 0, past = 0;
    for (int pass = 0;; ++pass) {
        if (threadIdx.x == 0) flag = 0;
        if (kg < nblk) stage(kg, 0);
        clear();
        if (pass != 1) {
            staged_barrier();
            // (group 0's first buffer is written again behind the first step's barrier at the earliest)
            bf16x8 ka[kKS];
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk) ka[kk] = lds_read8(&sm.st.k[0][0][0] + k_at[kk]);
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
                f32x16 s{};
#pragma unroll
                for (int kk = 0; kk < kKS; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kk], qreg[tt][kk], s, 0, 0, 0);
                const int mine = lim[tt] - 4 * hf;
                ref[tt] = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    ref[tt] = fmaxf(ref[tt], 8 * (i / 4) + i % 4 <= mine ? s[i] * a.scale_log2 : -__builtin_inff());
                ref[tt] = pair32_max(ref[tt]);
            }
        } else {
            take_refs(w_end);
            staged_barrier();
        }
        int i = 0;
        for (; i < whole; ++i) {
            const int j = i * KG + kg;
            compute_block(i & 1, j + KG < nblk ? j + KG : j);  // (no next one: a block that nobody reads)
            staged_barrier();
        }
        for (; i < steps; ++i) {
            const int buf = i & 1, j = i * KG + kg, key0 = j * KB;
            if (j + KG < nblk) stage(j + KG, buf ^ 1);
#pragma unroll 1
            for (int hh = 0; hh < kHalves; ++hh)
                if (key0 + 32 * hh < w_end) compute(buf, hh, key0 + 32 * hh);
            staged_barrier();
        }
        if (pass == 2) break;
        bool over = false, far = false;
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            over = over || (live && (!(l[tt] <= kPkGuard) || ref[tt] == -__builtin_inff()));
            far = far || (live && !(l[tt] <= kPkFar));
        }
        int now = 0;                                          // outputs past the guard (wave-uniform)
        if (pass == 1 || __ballot(far) != 0) {
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};          // (infinities and NaN stay in it)
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                    for (int x = 0; x < 16; ++x) sum[x & 3] += __builtin_fabsf(o[tt][dt][x]);
            const float guard = pass == 0 ? kPkOutGuard : 32.0f * kPkOutGuard;  // (2^125 against the exact maxima)
            far = live && !((sum[0] + sum[1]) + (sum[2] + sum[3]) <= guard);
            if (__ballot(far) != 0) {
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                    for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            now += __builtin_popcountll(__ballot(far && !(__builtin_fabsf(o[tt][dt][x]) <= guard)));
            }
        }
        const int mine = pass == 0 ? (__ballot(over) != 0 ? 1 : 0) | (now != 0 ? 2 : 0) : now < past ? 1 : 0;
        if (mine != 0 && lane == 0) atomicOr(&flag, mine);
        past = now;
        __syncthreads();
        const int all = flag;                                 // workgroup-uniform
        if (pass == 0 ? all == 0 : why != 2 || all != 0) break;
        why = all;
        __syncthreads();                                      // (read by all before it is cleared)
    }
    if (__ballot(odd) != 0) {                                 // wave-uniform
        // the values cleared above: a positive weight times inf or NaN is that value
        for (int key = (a.causal ? w_first : len) / 32 * 32; key < w_end; ++key) {
            if (key / KB % KG != kg) continue;
            const uint16_t* vr = vb + static_cast<int64_t>(key) * a.kv_st + 4 * hf;
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const uint2 y = *reinterpret_cast<const uint2*>(vr + 32 * dt + 8 * x);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t h = i < 2 ? y.x : y.y;
                        const float f = __uint_as_float(i % 2 ? h & 0xffff0000u : h << 16);
                        const bool is = !(__builtin_fabsf(f) < __builtin_inff());
#pragma unroll
                        for (int tt = 0; tt < NT; ++tt)
                            if (is && key <= lim[tt]) o[tt][dt][4 * x + i] += f;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) l[tt] = pair32_sum(l[tt]);
    if constexpr (KG > 1) {
        // the groups share their references: plain sums, in group order
        if (kg > 0) {
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) sm.mg.o[kg - 1][wave][(tt * kDT + dt) * 16 + i][lane] = o[tt][dt][i];
                sm.mg.l[kg - 1][wave][tt][lane] = l[tt];
            }
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int x = 0; x < KG - 1; ++x)
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
#pragma unroll
                for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[tt][dt][i] += sm.mg.o[x][wave][(tt * kDT + dt) * 16 + i][lane];
                l[tt] += sm.mg.l[x][wave][tt][lane];
            }
    }
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
        const int c = wcol0 + 32 * tt + col;
        if (c >= ncol) continue;
        const float inv = 1.0f / l[tt];
        uint16_t* op = a.out + (w.row0 + static_cast<int64_t>(tok[tt])) * a.out_st +
                       static_cast<int64_t>(g * a.R + c % a.R) * D + 4 * hf;
#pragma unroll
        for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                bf16x4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = static_cast<__bf16>(o[tt][dt][4 * x + i] * inv);
                *reinterpret_cast<bf16x4*>(op + 32 * dt + 8 * x) = y;
            }
    }
}

// ---------------------------------------------------------------------------
// keys straight from memory: fp32, heads of 16, and bf16 where sequences are short
// ---------------------------------------------------------------------------

namespace {

constexpr int kPdWaves = 4;

struct PackedDirect {
    const void* q;
    int64_t q_st, q_sh;
    const void *k, *v;
    int64_t kv_st, kv_sh;
    const int32_t* cu;
    int n;
    int64_t N;
    int Hkv, R, causal;
    int64_t slots;
    float scale_log2;
    void* out;
    int64_t out_st;
    uint32_t* status;
};

template <int DT>
struct PackedElem {
    typedef float E;
    static constexpr int kTiles = 1;   // 16-key tiles of a step
};
template <>
struct PackedElem<SPARDA_BF16> {
    typedef short E;
    static constexpr int kTiles = 2;
};

__device__ __forceinline__ bool packed_odd(float x) { return !(__builtin_fabsf(x) < __builtin_inff()); }
__device__ __forceinline__ bool packed_odd(short x) { return (x & 0x7f80) == 0x7f80; }
__device__ __forceinline__ float packed_f32(float x) { return x; }
__device__ __forceinline__ float packed_f32(short x) { return bf16_to_f32(static_cast<uint16_t>(x)); }
__device__ __forceinline__ void packed_put(float& o, float x) { o = x; }
__device__ __forceinline__ void packed_put(short& o, float x) { o = __builtin_bit_cast(short, static_cast<__bf16>(x)); }

}  // namespace

// One workgroup of 4 wavefronts per (KV head, window of 16 NT columns of one
// sequence; columns as in the staged kernel). The wavefronts take the steps of 16
// keys (bf16: 32) in turn, each with its own running (m, l, O) of every column, and
// are joined in order at the end: a walk is four times shorter and knows no barrier. K
// and V go straight from memory to the operand registers: the next step's K once the
// scores are taken, its V once the output products are, each under the other's
// products. The score layout of v_mfma_f32_16x16x4_f32 / 16x16x32_bf16 is already that
// of the P operand. Bound in fp32 by the matrix rate (16 keys x 16 columns take D / 2
// products of 32 cycles) and by how evenly the windows fall on the CUs, in bf16 by
// the loads, K and V being read once for every 16 NT columns: hence for short
// sequences, and for heads of 16, which fill no 32-row product. Measured: 37 tokens
// of 12/4 heads of 64 in bf16 4.2 us, three sequences of 1501 tokens in all in fp32 22-24
// us (48-52 TFLOP/s; the matrix cores are busy a third of it), 8000 tokens of 8/2 heads of
// 128 in fp32 1081 us (121 TFLOP/s of the 154 that a large library product reaches).
template <int DT, int D, int NT>
__global__ void __launch_bounds__(kPdWaves* kWave, 2) prefill_packed_direct_kernel(PackedDirect a) {
    typedef typename PackedElem<DT>::E E;
    constexpr bool kF32 = DT == SPARDA_F32;
    constexpr int kTiles = PackedElem<DT>::kTiles, kStep = 16 * kTiles, kBM = 16 * NT;
    constexpr int kV = D / 16, kQ = kF32 ? D / 16 : (D + 31) / 32, kPiece = kF32 ? 4 : 8;  // elements of V a lane holds per key, pieces of K, their elements
    constexpr bool kHalf = !kF32 && D == 16;                  // half of the lanes hold 16 dims (the others' are zero)
    typedef E Row __attribute__((ext_vector_type(kV)));
    __shared__ struct {
        f32x4 o[kPdWaves - 1][NT][kV][kWave];
        float m[kPdWaves - 1][NT][kWave], l[kPdWaves - 1][NT][kWave];
        int odd[kPdWaves];
    } sm;
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int c16 = lane % 16, grp = lane / 16;
    // A sequence's windows grow with their index. Where the chip holds all workgroups at
    // once, no later one evens out the CUs' loads: every other round of 256 runs
    // backwards. us against the plain order, fp32, 12/4 heads of 64: N=1000 25.1 / 27.0, N=1501 42.8 /
    // 47.3, 3 x 500 22.0 / 23.9, 20 x 75 11.5 / 10.8; with more workgroups, N=4000 234 / 229.
    uint32_t at = blockIdx.x;
    if (gridDim.x <= 5 * 256 && at / 256 % 2 == 1 && (at / 256 + 1) * 256 <= gridDim.x) at = at / 256 * 256 + 255 - at % 256;
    const int g = at % a.Hkv;
    const int64_t slot = a.slots - 1 - at / a.Hkv;
    bool bad;
    const PackedWindow w = packed_window(a.cu, a.n, a.N, a.R, kBM, slot, bad);
    if (bad && threadIdx.x == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_SEQUENCE_RANGE));
    if (w.seq < 0) return;                                    // workgroup-uniform
    const int len = w.len, ncol = len * a.R, col0 = static_cast<int>(w.win) * kBM;
    const int w_first = col0 / a.R, w_last = (col0 + kBM <= ncol ? col0 + kBM - 1 : ncol - 1) / a.R;
    const int w_end = a.causal ? w_last + 1 : len;            // keys of the window
    const E* kb = static_cast<const E*>(a.k) + static_cast<int64_t>(w.row0) * a.kv_st + static_cast<int64_t>(g) * a.kv_sh;
    const E* vb = static_cast<const E*>(a.v) + static_cast<int64_t>(w.row0) * a.kv_st + static_cast<int64_t>(g) * a.kv_sh;

    int tok[NT], lim[NT];
    uint4 qr[NT][kQ];                // dims 4 kPiece x + kPiece grp ..
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
        const int c = col0 + 16 * tt + c16 < ncol ? col0 + 16 * tt + c16 : ncol - 1;
        tok[tt] = c / a.R;
        lim[tt] = a.causal ? tok[tt] : len - 1;
        const E* qp = static_cast<const E*>(a.q) + (w.row0 + static_cast<int64_t>(tok[tt])) * a.q_st +
                      static_cast<int64_t>(g * a.R + c % a.R) * a.q_sh + kPiece * grp;
#pragma unroll
        for (int x = 0; x < kQ; ++x) {
            qr[tt][x] = uint4{0, 0, 0, 0};
            if (!kHalf || grp < 2) qr[tt][x] = *reinterpret_cast<const uint4*>(qp + 4 * kPiece * x);
        }
    }
    const int kv_st = static_cast<int>(a.kv_st);
    uint4 kr[kTiles][kQ];            // key 16 t + c16, dims as q
    Row vr[kTiles][4];               // key 16 t + 4 grp + i, dims kV c16 ..
    auto load_k = [&](int u) __attribute__((always_inline)) {
        const int last = len - 1 - kStep * u;                 // rows past the end read the last one
        const E* p = kb + static_cast<int64_t>(kStep * u) * a.kv_st;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            const int key = 16 * t + c16;
            const uint32_t at = static_cast<uint32_t>((key < last ? key : last) * kv_st + kPiece * grp);
#pragma unroll
            for (int x = 0; x < kQ; ++x) {
                kr[t][x] = uint4{0, 0, 0, 0};
                if (!kHalf || grp < 2) kr[t][x] = *reinterpret_cast<const uint4*>(p + at + 4 * kPiece * x);
            }
        }
    };
    auto load_v = [&](int u) __attribute__((always_inline)) {
        const int last = len - 1 - kStep * u;
        const E* p = vb + static_cast<int64_t>(kStep * u) * a.kv_st;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 16 * t + 4 * grp + i;
                vr[t][i] = *reinterpret_cast<const Row*>(p + static_cast<uint32_t>((key < last ? key : last) * kv_st + kV * c16));
            }
    };

    float m[NT], l[NT];                                       // log2 units; this lane's part of the sum
    f32x4 o[NT][kV];
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
        m[tt] = -__builtin_inff();
        l[tt] = 0.0f;
#pragma unroll
        for (int j = 0; j < kV; ++j) o[tt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool odd = false;                                         // V not finite at a place that some column may not attend
    const int steps = (w_end + kStep - 1) / kStep;
    if (wave < steps) {
        load_k(wave);
        load_v(wave);
    }
    for (int u = wave; u < steps; u += kPdWaves) {            // wave-uniform
        const int key0 = kStep * u, next = u + kPdWaves < steps ? u + kPdWaves : u;
        const bool edge = a.causal ? key0 + kStep - 1 > w_first : key0 + kStep > len;
        f32x4 s[NT][kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            // (fp32: two short sums a score, fewer products that wait for the one before and smaller roundings)
            f32x4 s2[NT];
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) s[tt][t] = s2[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < kQ; ++x) {
                if constexpr (kF32) {
                    const f32x4 ka = __builtin_bit_cast(f32x4, kr[t][x]);
#pragma unroll
                    for (int y = 0; y < 4; y += 2)
#pragma unroll
                        for (int tt = 0; tt < NT; ++tt) {
                            const f32x4 qb = __builtin_bit_cast(f32x4, qr[tt][x]);
                            s[tt][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[y], qb[y], s[tt][t], 0, 0, 0);
                            s2[tt] = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[y + 1], qb[y + 1], s2[tt], 0, 0, 0);
                        }
                } else {
#pragma unroll
                    for (int tt = 0; tt < NT; ++tt)
                        s[tt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[t][x]),
                                                                           __builtin_bit_cast(bf16x8, qr[tt][x]), s[tt][t], 0, 0, 0);
                }
            }
            if constexpr (kF32) {
#pragma unroll
                for (int tt = 0; tt < NT; ++tt) s[tt][t] += s2[tt];
            }
        }
        load_k(next);                                         // (the last step: its own again)
        if (edge) {
            // (a weight of 0 times inf is NaN: such values are cleared here, and added at the end to the columns
            // that do attend them)
            bool any = false;
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kV; ++j) any |= packed_odd(vr[t][i][j]);
            if (__ballot(any) != 0) {
                odd = true;
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < kV; ++j) vr[t][i][j] = packed_odd(vr[t][i][j]) ? 0 : vr[t][i][j];
            }
        }
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            const int left = lim[tt] - key0 - 4 * grp;        // this lane's keys 16 t + i up to it are allowed
            float mx = m[tt];
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mx = fmaxf(mx, 16 * t + i <= left ? s[tt][t][i] * a.scale_log2 : -__builtin_inff());
            mx = pair32_max(pair16_max(mx));
            const float ref = mx == -__builtin_inff() ? 0.0f : mx;
            const float alpha = __builtin_amdgcn_exp2f(m[tt] - ref);
            if (__ballot(mx != m[tt]) != 0) {                 // wave-uniform: some column's maximum rose
#pragma unroll
                for (int j = 0; j < kV; ++j) o[tt][j] *= alpha;
                l[tt] *= alpha;
            }
            m[tt] = mx;
            // one rounding between a score and its distance from the reference, which is small where the weight is not
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[tt][t][i] = 16 * t + i <= left ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[tt][t][i], a.scale_log2, -ref)) : 0.0f;
                    l[tt] += s[tt][t][i];
                }
        }
        if constexpr (kF32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kV; ++j)
#pragma unroll
                    for (int tt = 0; tt < NT; ++tt)
                        o[tt][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vr[0][i][j], s[tt][0][i], o[tt][j], 0, 0, 0);
        } else {
            // P is rounded to bf16 for the product (the sum l keeps it in fp32)
            bf16x8 pb[NT];
#pragma unroll
            for (int tt = 0; tt < NT; ++tt)
#pragma unroll
                for (int e = 0; e < 8; ++e) pb[tt][e] = static_cast<__bf16>(s[tt][e / 4][e % 4]);
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                s16x8 va;
#pragma unroll
                for (int e = 0; e < 8; ++e) va[e] = vr[e / 4][e % 4][j];
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
                    o[tt][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), pb[tt], o[tt][j], 0, 0, 0);
            }
        }
        load_v(next);
    }
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) l[tt] = pair32_sum(pair16_sum(l[tt]));

    // ---- join the wavefronts, in order ----
    if (lane == 0) sm.odd[wave] = odd ? 1 : 0;
    if (wave > 0) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
#pragma unroll
            for (int j = 0; j < kV; ++j) sm.o[wave - 1][tt][j][lane] = o[tt][j];
            sm.m[wave - 1][tt][lane] = m[tt];
            sm.l[wave - 1][tt][lane] = l[tt];
        }
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
        float M = m[tt];
#pragma unroll
        for (int x = 0; x < kPdWaves - 1; ++x) M = fmaxf(M, sm.m[x][tt][lane]);
        const float ref = M == -__builtin_inff() ? 0.0f : M;
        float wt = __builtin_amdgcn_exp2f(m[tt] - ref);
        l[tt] *= wt;
#pragma unroll
        for (int j = 0; j < kV; ++j) o[tt][j] *= wt;
#pragma unroll
        for (int x = 0; x < kPdWaves - 1; ++x) {
            wt = __builtin_amdgcn_exp2f(sm.m[x][tt][lane] - ref);
            l[tt] = __builtin_fmaf(wt, sm.l[x][tt][lane], l[tt]);
#pragma unroll
            for (int j = 0; j < kV; ++j) o[tt][j] += sm.o[x][tt][j][lane] * wt;
        }
    }
    if ((sm.odd[0] | sm.odd[1] | sm.odd[2] | sm.odd[3]) != 0) {
        // the values cleared above: a positive weight times inf or NaN is that value
        for (int key = (a.causal ? w_first : len) / kStep * kStep; key < w_end; ++key) {
            const E* vp = vb + static_cast<int64_t>(key) * a.kv_st + 4 * kV * grp;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kV; ++j) {
                    const E f = vp[kV * i + j];
#pragma unroll
                    for (int tt = 0; tt < NT; ++tt)
                        if (packed_odd(f) && key <= lim[tt]) o[tt][j][i] += packed_f32(f);
                }
        }
    }
    // O^T tile j, row 4 grp + i: dim kV (4 grp + i) + j
#pragma unroll
    for (int tt = 0; tt < NT; ++tt) {
        const int c = col0 + 16 * tt + c16;
        if (c >= ncol) continue;
        const float inv = 1.0f / l[tt];
        E* op = static_cast<E*>(a.out) + (w.row0 + static_cast<int64_t>(tok[tt])) * a.out_st +
                static_cast<int64_t>(g * a.R + c % a.R) * D + 4 * kV * grp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            Row y;
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                E e;
                packed_put(e, o[tt][j][i] * inv);
                y[j] = e;
            }
            *reinterpret_cast<Row*>(op + kV * i) = y;
        }
    }
}

int launch_prefill_packed(const void* q, int64_t q_st, int64_t q_sh, const void* k, const void* v, int64_t kv_st,
                          int64_t kv_sh, int dtype, const int32_t* cu, int64_t n, int64_t N, int64_t Hq, int64_t Hkv,
                          int64_t D, int causal, float scale, void* out, int64_t out_st, hipStream_t stream) {
    const int64_t R = Hq / Hkv;
    const float sl = scale * kPkLog2e;
    const bool f32 = dtype == SPARDA_F32;
    // bf16 without staging: where 16-column windows leave every CU at most one workgroup and sequences are short, the
    // walk's latency is all there is. us of this form / the staged ones below, causal: 12/4 heads of 64: N=1
    // 4.0 / 5.4, 37 4.2 / 5.5, 256 5.8 / 6.0, 350 6.5 / 6.5, 512 8.8 / 7.0, 4 x 128 6.7 / 6.1, 16 x 32 5.0 / 5.6;
    // 8/1 heads of 128: N=200 7.4 / 8.4, 400 9.2 / 10.3; 32/8: N=128 6.8 / 7.4, 256 10.3 / 9.3
    if (f32 || D == 16 || (N * Hq <= 16 * 256 && N <= 384 * n)) {
        PackedDirect a{q, q_st, q_sh, k, v, kv_st, kv_sh, cu, static_cast<int>(n), N, static_cast<int>(Hkv),
                       static_cast<int>(R), causal, 0, sl, out, out_st, nullptr};
#define SPARDA_PKD_N(DT_, D_, NT_)                                                                                \
    do {                                                                                                          \
        a.slots = packed_slots(N, n, R, 16 * NT_);                                                                \
        if (!grid_fits(a.slots * Hkv, kPdWaves * kWave)) return set_error(SPARDA_ERR_SHAPE, "prefill_packed: grid too large"); \
        if (const int rc = status_word(&a.status)) return rc;                                                     \
        hipLaunchKernelGGL((prefill_packed_direct_kernel<DT_, D_, NT_>), dim3(static_cast<unsigned>(a.slots * Hkv)), \
                           dim3(kPdWaves * kWave), 0, stream, a);                                                 \
    } while (0)
#define SPARDA_PKD(DT_, D_)                       \
    do {                                          \
        if (wide) SPARDA_PKD_N(DT_, D_, 2);       \
        else SPARDA_PKD_N(DT_, D_, 1);            \
    } while (0)
        // Wider windows read K and V for more columns, narrow ones are more workgroups. us of 16 / 32 columns, fp32, 12/4
        // heads of 64: N=512 12.7 / 16.2, 3 x 500 22.0 / 26.7, N=1501 42.8 / 52.8, N=4000 232 / 225; 8/2 of 128:
        // N=2000 93 / 109, 4 x 750 75 / 76, N=4000 335 / 294, N=8000 1274 / 1081; 12/4 of 32: N=1000 15.3 / 20.1,
        // N=2000 45.9 / 41.6; bf16 heads of 16: N=1000 7.8 / 8.9, N=2000 20.3 / 16.7, N=16384 761 / 579
        const bool wide = N * Hq > 16 * 1536 || (D <= 32 && N * Hq > 16 * 1024);
        if (f32) {
            if (D == 16) SPARDA_PKD(SPARDA_F32, 16);
            else if (D == 32) SPARDA_PKD(SPARDA_F32, 32);
            else if (D == 64) SPARDA_PKD(SPARDA_F32, 64);
            else SPARDA_PKD(SPARDA_F32, 128);
        } else {
            if (D == 16) SPARDA_PKD(SPARDA_BF16, 16);
            else if (D == 32) SPARDA_PKD_N(SPARDA_BF16, 32, 1);
            else if (D == 64) SPARDA_PKD_N(SPARDA_BF16, 64, 1);
            else SPARDA_PKD_N(SPARDA_BF16, 128, 1);
        }
#undef SPARDA_PKD
#undef SPARDA_PKD_N
        return check_hip(hipGetLastError(), "prefill_packed_direct_kernel");
    }
    PackedPrefill a{static_cast<const uint16_t*>(q), q_st, q_sh, static_cast<const uint16_t*>(k),
                    static_cast<const uint16_t*>(v), kv_st, kv_sh, cu, static_cast<int>(n), N, static_cast<int>(Hkv),
                    static_cast<int>(R), causal, 0, sl, static_cast<uint16_t*>(out), out_st, nullptr};
#define SPARDA_PKM(D_, NT_, CW_, KG_, KB_)                                                                        \
    do {                                                                                                          \
        a.slots = packed_slots(N, n, R, 32 * NT_ * CW_);                                                          \
        if (!grid_fits(a.slots * Hkv, CW_ * KG_ * kWave)) return set_error(SPARDA_ERR_SHAPE, "prefill_packed: grid too large"); \
        if (const int rc = status_word(&a.status)) return rc;                                                     \
        hipLaunchKernelGGL((prefill_packed_kernel<D_, NT_, CW_, KG_, KB_>), dim3(static_cast<unsigned>(a.slots * Hkv)), \
                           dim3(CW_ * KG_ * kWave), 0, stream, a);                                                \
    } while (0)
    // W: windows of 128 columns, NB: 64-key blocks of a mean sequence (the host does not know
    // the lengths: a long sequence among short ones goes with the short). Heads of 32 have one
    // form, other calls than causal ones follow the same rule; neither was measured against others. Wide windows
    // stage a block for the most columns; key groups and small windows cut a
    // window's serial walk where windows are few against the 256 CUs (a group's sums
    // cost a merge, so that short walks are not cut). us of (tiles a wavefront, wavefronts,
    // key groups) = (2,4,1) / (1,4,1) / (1,4,2) / (1,2,2) / (1,1,4), 12/4 heads of 64, causal:
    //   N=400 13.3 / 8.8 / 8.9 / 7.4 / 7.0   N=1000 22.8 / 14.9 / 13.4 / 10.7 / 10.1
    //   N=2048 38.7 / 24.9 / 22.4 / 18.3 / 19.5   N=4096 70.5 / 48.5 / 41.0 / 42.0 / 53.1
    //   4 x 1024 24.6 / 20.1 / 20.8 / 20.7 / 24.7   16 x 256 12.7 / 10.2 / 13.7 / 13.2 / 17.8
    //   N=1600 31.1 / 20.2 / 18.6 / 15.6 / 14.4   2 x 700 19.0 / 11.6 / 11.5 / 9.7 / 10.2
    //   2 x 2800 53.0 / 48.0 / 38.6 / 39.1 / 50.8   4 x 1400 32.5 / 27.5 / 28.7 / 25.5 / 37.1
    //   N=8192 152 / 127 / 131 / 133 / 165   16 x 1024 55.5 / 47.7 / 60.3 / 59.5 / 90.4
    //   N=16384 428 / 425 / 480 / 486 / 626   N=32768 1555 / 1630   8 x 8192 847 / 889
    // and of (1,4,1) / (1,4,2) / (1,2,2 of 32 keys), heads of 128:
    //   32/8: N=512 14.5 / 15.1 / 11.8   N=1100 25.0 / 23.7 / 21.6   N=2048 49.2 / 48.9 / 53.4
    //   8 x 250 17.1 / 22.8 / 21.1   8 x 2000 305 / 370 / 400   8/1: N=8192 171 / 144 / 158
    const int64_t W = cdiv(N * Hq, 128), NB = cdiv(cdiv(N, n), 64), cus = 256;
    if (D == 32) {
        SPARDA_PKM(32, 1, 4, 1, 64);
    } else if (D == 64) {
        if (2 * W <= cus || (8 * W <= 5 * cus && NB >= 20)) SPARDA_PKM(64, 1, 1, 4, 32);
        else if (W <= cus && NB >= 8) SPARDA_PKM(64, 1, 2, 2, 64);
        else if ((W <= 2 * cus && NB >= 16) || (5 * W <= 12 * cus && NB >= 32)) SPARDA_PKM(64, 1, 4, 2, 64);
        else if (W <= 8 * cus || NB < 32) SPARDA_PKM(64, 1, 4, 1, 64);
        else SPARDA_PKM(64, 2, 4, 1, 64);
    } else {
        if (2 * W <= cus || (W <= cus && NB >= 8) || (3 * W <= 4 * cus && NB >= 16)) SPARDA_PKM(128, 1, 2, 2, 32);
        else if (W <= 2 * cus && NB >= 64) SPARDA_PKM(128, 1, 4, 2, 64);
        else SPARDA_PKM(128, 1, 4, 1, 64);
    }
#undef SPARDA_PKM
    return check_hip(hipGetLastError(), "prefill_packed_kernel");
}

}  // namespace sparda
