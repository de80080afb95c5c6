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

// One wavefront per (row, query head): lane j takes key j of 64 at a time, the
// running maximum and sum are the wave's, and each lane then holds dims lane and
// lane + 64 of the output. Any head dim up to 128, any strides.
template <int DT>
__global__ void __launch_bounds__(256)
prefill_packed_general_kernel(const void* __restrict__ q, int64_t q_st, int64_t q_sh, const void* __restrict__ k,
                              const void* __restrict__ v, int64_t kv_st, int64_t kv_sh,
                              const int32_t* __restrict__ cu, int n, int64_t N, int Hq, int R, int D, int causal,
                              float scale_log2, void* __restrict__ out, int64_t out_st, uint32_t* __restrict__ status) {
    const int lane = threadIdx.x % kWave;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t slot = item / Hq;
    const int h = static_cast<int>(item % Hq);
    if (slot >= packed_slots(N, n, 1, 1)) return;
    bool bad;
    const PackedWindow w = packed_window(cu, n, N, 1, 1, slot, bad);
    if (bad && lane == 0) atomicOr(status, static_cast<uint32_t>(SPARDA_STATUS_SEQUENCE_RANGE));
    if (w.seq < 0) return;
    const int64_t t = w.row0 + w.win;
    const int keys = causal ? static_cast<int>(w.win) + 1 : w.len;
    const int64_t qo = t * q_st + static_cast<int64_t>(h) * q_sh;
    const int64_t kvo = static_cast<int64_t>(w.row0) * kv_st + static_cast<int64_t>(h / R) * kv_sh;
    float m = -__builtin_inff(), l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int s0 = 0; s0 < keys; s0 += kWave) {
        const int s = s0 + lane;
        float x = -__builtin_inff();
        if (s < keys) {
            float acc = 0.0f;
            const int64_t ko = kvo + s * kv_st;
            for (int d = 0; d < D; ++d) acc = __builtin_fmaf(load_elem<DT>(q, qo + d), load_elem<DT>(k, ko + d), acc);
            x = acc * scale_log2;
        }
        const float mx = fmaxf(m, wave_max(x));
        const float ref = mx == -__builtin_inff() ? 0.0f : mx;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        float p = __builtin_amdgcn_exp2f(x - ref);
        if (s >= keys) p = 0.0f;
        l = l * alpha + wave_sum(p);
        o0 *= alpha;
        o1 *= alpha;
        m = mx;
        const int cnt = keys - s0 < kWave ? keys - s0 : kWave;
        for (int j = 0; j < cnt; ++j) {
            const float pj = __shfl(p, j, kWave);
            const int64_t vo = kvo + static_cast<int64_t>(s0 + j) * kv_st;
            if (lane < D) o0 = __builtin_fmaf(pj, load_elem<DT>(v, vo + lane), o0);
            if (lane + kWave < D) o1 = __builtin_fmaf(pj, load_elem<DT>(v, vo + lane + kWave), o1);
        }
    }
    const float inv = 1.0f / l;
    const int64_t oo = t * out_st + static_cast<int64_t>(h) * D;
    if (lane < D) store_elem<DT>(out, oo + lane, o0 * inv);
    if (lane + kWave < D) store_elem<DT>(out, oo + lane + kWave, o1 * inv);
}

// ---------------------------------------------------------------------------
// bf16, D = 64 and 128, on the matrix cores
// ---------------------------------------------------------------------------

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr float kPkGuard = 18446744073709551616.0f;  // 2^64

// 16-byte piece `c` of row `r` in an LDS tile of D-element rows: pieces are
// exchanged within a row so that both reads of a tile are spread over the banks:
// 16 consecutive rows at one piece (K) take 16 different places of 256 bytes, and
// 4 consecutive rows at 4 consecutive pieces (V, transposed) do too.
template <int D>
__device__ __forceinline__ int pk_piece(int r, int c) {
    if constexpr (D == 64) return c ^ ((r >> 1 & 1) << 2 | (r >> 2 & 1) << 1 | (r >> 3 & 1));
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
// ref[col] is the column's maximum over the sequence's first 32 keys (key 0 is
// allowed to every column), taken before the walk from memory, so that every key
// group has it and nothing is rescaled. A sum past 2^64, or a first tile of -inf
// alone, sends the workgroup over its keys twice more: for the exact maxima, then
// against them.
template <int D, int NT, int CW, int KG, int KB>
__global__ void __launch_bounds__(CW* KG* kWave, 2) prefill_packed_kernel(PackedPrefill a) {
    constexpr int kCols = 32 * NT, kBM = CW * kCols, kThreads = CW * kWave;
    constexpr int kPieces = D / 8, kSR = KB * kPieces / kThreads, kRowStep = kThreads / kPieces;
    constexpr int kKS = D / 16, kDT = D / 32, kHalves = KB / 32;
    __shared__ union {
        PackedStage<D, KB, KG> st;
        PackedMerge<NT * kDT * 16, CW, NT, KG> mg;
        float ref[KG][CW][NT][32];
    } sm;
    __shared__ int flag;
    const int lane = threadIdx.x % kWave;
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int wave = wv % CW, kg = wv / CW;
    const int tid = wave * kWave + lane;
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

    const int srow = tid / kPieces, spiece = tid % kPieces, kv_st = static_cast<int>(a.kv_st);
    typedef unsigned int StageV __attribute__((ext_vector_type(4 * kSR)));
    auto fetch = [&](int j, StageV& nk, StageV& nv) __attribute__((always_inline)) {
        const int row0 = j * KB, last = len - 1 - row0;
        const uint16_t* kr = kb + static_cast<int64_t>(row0) * a.kv_st;
        const uint16_t* vr = vb + static_cast<int64_t>(row0) * a.kv_st;
#pragma unroll
        for (int i = 0; i < kSR; ++i) {
            int r = srow + i * kRowStep;
            r = r < last ? r : last;
            const uint32_t at = static_cast<uint32_t>(r * kv_st + 8 * spiece);
            const uint4 x = *reinterpret_cast<const uint4*>(kr + at);
            const uint4 y = *reinterpret_cast<const uint4*>(vr + at);
            nk[4 * i] = x.x; nk[4 * i + 1] = x.y; nk[4 * i + 2] = x.z; nk[4 * i + 3] = x.w;
            nv[4 * i] = y.x; nv[4 * i + 1] = y.y; nv[4 * i + 2] = y.z; nv[4 * i + 3] = y.w;
        }
    };
    auto stash = [&](int j, int buf, StageV& nk, StageV& nv) __attribute__((always_inline)) {
        const int rows = len - j * KB;
#pragma unroll
        for (int i = 0; i < kSR; ++i) {
            const int r = srow + i * kRowStep, at = r * D + 8 * pk_piece<D>(r, spiece);
            uint4 x{nk[4 * i], nk[4 * i + 1], nk[4 * i + 2], nk[4 * i + 3]};
            uint4 y{nv[4 * i], nv[4 * i + 1], nv[4 * i + 2], nv[4 * i + 3]};
            if (r >= rows) x = y = uint4{0, 0, 0, 0};         // behind the sequence: weightless, and finite
            *reinterpret_cast<uint4*>(&sm.st.k[buf][kg][at]) = x;
            *reinterpret_cast<uint4*>(&sm.st.v[buf][kg][at]) = y;
        }
    };

    // the references: the first 32 keys straight from memory
    float ref[NT], l[NT];
    {
        bf16x8 ka[kKS];
        const uint16_t* kr = kb + static_cast<int64_t>(col < len ? col : len - 1) * a.kv_st + 8 * hf;
#pragma unroll
        for (int kk = 0; kk < kKS; ++kk) ka[kk] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(kr + 16 * kk));
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            f32x16 s{};
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kk], qreg[tt][kk], s, 0, 0, 0);
            float m = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i / 4) + 4 * hf + i % 4 <= lim[tt]) m = fmaxf(m, s[i] * a.scale_log2);
            const float2 r2 = rows32_swap(m);
            ref[tt] = fmaxf(r2.x, r2.y);
        }
    }

    f32x16 o[NT][kDT];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int tt = 0; tt < NT; ++tt) {
            l[tt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt) o[tt][dt] = f32x16{};
        }
    };
    clear();

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
    auto compute = [&](int buf, int half, int key0, bool maxima) __attribute__((always_inline)) {
        bf16x8 ka[kKS], va[kDT][2];
        const uint16_t* ks = &sm.st.k[buf][kg][32 * half * D];
        const uint16_t* vs = &sm.st.v[buf][kg][32 * half * D];
#pragma unroll
        for (int kk = 0; kk < kKS; ++kk) ka[kk] = lds_read8(ks + k_at[kk]);
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
        if (edge && a.causal) {
            // a weight of 0 times inf is NaN: such values are cleared here, and added
            // after the walk to the columns that do attend them
            auto bad2 = [](uint32_t x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; };
            bool any = false;
#pragma unroll
            for (int dt = 0; dt < kDT; ++dt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint4 x = __builtin_bit_cast(uint4, va[dt][c]);
                    any = any || bad2(x.x) || bad2(x.y) || bad2(x.z) || bad2(x.w);
                }
            if (__ballot(any) != 0) {
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
            f32x16 s{};
#pragma unroll
            for (int kk = 0; kk < kKS; ++kk) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[kk], qreg[tt][kk], s, 0, 0, 0);
            if (maxima) {
                float m = ref[tt];
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + 8 * (i / 4) + 4 * hf + i % 4 <= lim[tt]) m = fmaxf(m, s[i] * a.scale_log2);
                ref[tt] = m;
                continue;
            }
            const float neg = ref[tt] == -__builtin_inff() ? 0.0f : -ref[tt];
            bf16x8 pb[2];
            float sum = 0.0f;
            if (edge) {
                const int mine = lim[tt] - key0 - 4 * hf;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, neg));
                    p = 8 * (i / 4) + i % 4 <= mine ? p : 0.0f;
                    sum += p;
                    pb[i / 8][i % 8] = static_cast<__bf16>(p);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, neg));
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

    // step i: group kg computes block i KG + kg from buffer i & 1 while its next is loaded
    const int steps = (nblk + KG - 1) / KG;
    for (int mode = 0;; ++mode) {                             // 0: against ref; 1: the exact maxima; 2: against those
        if (threadIdx.x == 0) flag = 0;
        StageV nk{}, nv{};
        if (kg < nblk) {
            fetch(kg, nk, nv);
            stash(kg, 0, nk, nv);
        }
        if (kg + KG < nblk) fetch(kg + KG, nk, nv);
        __syncthreads();
        for (int i = 0; i < steps; ++i) {
            const int buf = i & 1, j = i * KG + kg;
#pragma unroll 1
            for (int hh = 0; hh < kHalves; ++hh)
                if (j < nblk && j * KB + 32 * hh < w_end) compute(buf, hh, j * KB + 32 * hh, mode == 1);
            if (j + KG < nblk) {
                stash(j + KG, buf ^ 1, nk, nv);
                if (j + 2 * KG < nblk) fetch(j + 2 * KG, nk, nv);
            }
            __syncthreads();
        }
        if (mode == 2) break;
        if (mode == 0) {
            bool over = false;
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) over = over || (live && (!(l[tt] <= kPkGuard) || ref[tt] == -__builtin_inff()));
            if (__ballot(over) != 0 && lane == 0) atomicOr(&flag, 1);
            __syncthreads();
            if (flag == 0) break;                             // workgroup-uniform
            __syncthreads();                                  // (read by all before it is cleared)
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) ref[tt] = -__builtin_inff();
        } else {
#pragma unroll
            for (int tt = 0; tt < NT; ++tt) {
                const float2 r2 = rows32_swap(ref[tt]);
                ref[tt] = fmaxf(r2.x, r2.y);
                if (KG > 1 && hf == 0) sm.ref[kg][wave][tt][col] = ref[tt];
            }
            if constexpr (KG > 1) {
                __syncthreads();
#pragma unroll
                for (int tt = 0; tt < NT; ++tt)
                    for (int x = 0; x < KG; ++x) ref[tt] = fmaxf(ref[tt], sm.ref[x][wave][tt][col]);
                __syncthreads();
            }
            clear();
        }
    }
    if (__ballot(odd) != 0) {                                 // wave-uniform
        // the values cleared above: a positive weight times inf or NaN is that value
        for (int key = w_first / 32 * 32; key < w_end; ++key) {
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

static bool packed_matrix_cores(const void* q, int64_t q_st, int64_t q_sh, const void* k, const void* v, int64_t kv_st,
                                int64_t kv_sh, int dtype, int64_t N, int64_t R, int64_t D, const void* out,
                                int64_t out_st) {
    auto al = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
    return dtype == SPARDA_BF16 && (D == 64 || D == 128) && N * R < (int64_t(1) << 31) - 256 && al(q, 16) && al(k, 16) && al(v, 16) &&
           al(out, 8) && q_st % 8 == 0 && q_sh % 8 == 0 && kv_st >= 0 && kv_st < (1 << 24) && kv_st % 8 == 0 && kv_sh % 8 == 0 && out_st % 4 == 0;
}

int launch_prefill_packed(const void* q, int64_t q_st, int64_t q_sh, const void* k, const void* v, int64_t kv_st,
                          int64_t kv_sh, int dtype, const int32_t* cu, int64_t n, int64_t N, int64_t Hq, int64_t Hkv,
                          int64_t D, int causal, float scale, void* out, int64_t out_st, hipStream_t stream) {
    uint32_t* status;
    if (const int rc = status_word(&status)) return rc;
    const int64_t R = Hq / Hkv;
    const float sl = scale * kPkLog2e;
    if (packed_matrix_cores(q, q_st, q_sh, k, v, kv_st, kv_sh, dtype, N, R, D, out, out_st)) {
        PackedPrefill a{static_cast<const uint16_t*>(q), q_st, q_sh, static_cast<const uint16_t*>(k),
                        static_cast<const uint16_t*>(v), kv_st, kv_sh, cu, static_cast<int>(n), N, static_cast<int>(Hkv),
                        static_cast<int>(R), causal, 0, sl, static_cast<uint16_t*>(out), out_st, status};
        static const int force = getenv("PKV") ? atoi(getenv("PKV")) : 0;
#define SPARDA_PKM(D_, NT_, CW_, KG_, KB_)                                                                        \
    do {                                                                                                          \
        a.slots = packed_slots(N, n, R, 32 * NT_ * CW_);                                                          \
        if (a.slots * Hkv >= (int64_t(1) << 31)) return set_error(SPARDA_ERR_SHAPE, "prefill_packed: grid too large"); \
        hipLaunchKernelGGL((prefill_packed_kernel<D_, NT_, CW_, KG_, KB_>), dim3(static_cast<unsigned>(a.slots * Hkv)), \
                           dim3(CW_ * KG_ * kWave), 0, stream, a);                                                \
    } while (0)
        if (D == 64) {
            if (force == 1) SPARDA_PKM(64, 2, 1, 4, 32);
            else if (force == 2) SPARDA_PKM(64, 1, 1, 4, 32);
            else if (force == 3) SPARDA_PKM(64, 1, 4, 1, 64);
            else if (force == 4) SPARDA_PKM(64, 2, 2, 2, 64);
            else SPARDA_PKM(64, 2, 4, 1, 64);
        } else {
            if (force == 1 || force == 2) SPARDA_PKM(128, 1, 1, 4, 32);
            else if (force == 4) SPARDA_PKM(128, 1, 2, 2, 32);
            else SPARDA_PKM(128, 1, 4, 1, 64);
        }
#undef SPARDA_PKM
        return check_hip(hipGetLastError(), "prefill_packed_kernel");
    }
    const int64_t groups = cdiv(packed_slots(N, n, 1, 1) * Hq, 4);
    if (groups >= (int64_t(1) << 31)) return set_error(SPARDA_ERR_SHAPE, "prefill_packed: too many rows and heads");
#define SPARDA_PKG(DT_)                                                                                            \
    hipLaunchKernelGGL((prefill_packed_general_kernel<DT_>), dim3(static_cast<unsigned>(groups)), dim3(256), 0,    \
                       stream, q, q_st, q_sh, k, v, kv_st, kv_sh, cu, static_cast<int>(n), N, static_cast<int>(Hq), \
                       static_cast<int>(R), static_cast<int>(D), causal, sl, out, out_st, status)
    if (dtype == SPARDA_F32) SPARDA_PKG(SPARDA_F32);
    else SPARDA_PKG(SPARDA_BF16);
#undef SPARDA_PKG
    return check_hip(hipGetLastError(), "prefill_packed_general_kernel");
}

}  // namespace sparda
