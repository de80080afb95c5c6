// A key-value cache in pages (sparda_append_paged, sparda_decode_paged): pages
// of ps rows [ps, Hkv, D], position p of sequence b in row p % ps of page
// table[b, p / ps].
#include "common.h"
#include "kernels.h"
#include "mfma.h"
#include "packed.h"
#include "paged.h"

namespace sparda {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------

// One wavefront per new row: its sequence, its page, then the row's heads in 16-byte
// pieces. Bound by memory, a row read and a row written: 16000 rows of 8 heads of 128
// take 27.7 us a call = 4.7 TB/s where rows and pages change from call to call, 21.5 us =
// 6.1 TB/s where the last-level cache holds them; 64 rows 2.6 us, a launch and three dependent loads.
__global__ void __launch_bounds__(256)
append_paged_kernel(char* __restrict__ k, char* __restrict__ v, Pages pg, int ps, const int32_t* __restrict__ positions,
                    const int32_t* __restrict__ cu, int n, const char* __restrict__ k_new,
                    const char* __restrict__ v_new, int64_t N, int64_t new_st, int64_t new_sh, int Hkv, int row_bytes,
                    int es, uint32_t* __restrict__ status) {
    const int lane = threadIdx.x % kWave;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (t >= N) return;
    const PagedRow r = paged_row(pg, ps, positions, cu, n, N, t, status);
    if (!r.takes || r.page < 0) return;           // (without a page the row is dropped)
    const int64_t to = (r.page * pg.p_st + r.row * pg.s_st) * es;
    const int64_t from = t * new_st * es;
    const int per = row_bytes / 16;               // pieces of a head's row
    for (int c = lane; c < Hkv * per; c += kWave) {
        const int h = c / per, o = (c - h * per) * 16;
        const int64_t src = from + h * new_sh * es + o, dst = to + h * pg.h_st * es + o;
        *reinterpret_cast<uint4*>(k + dst) = *reinterpret_cast<const uint4*>(k_new + src);
        *reinterpret_cast<uint4*>(v + dst) = *reinterpret_cast<const uint4*>(v_new + src);
    }
}

int launch_append_paged(void* k, void* v, int64_t n_pages, int64_t ps, int64_t p_st, int64_t s_st, int64_t h_st,
                        int dtype, const int32_t* table, int64_t t_st, int64_t width, const int32_t* positions,
                        const int32_t* cu, int64_t n, const void* k_new, const void* v_new, int64_t N, int64_t new_st,
                        int64_t new_sh, int64_t Hkv, int64_t D, hipStream_t stream) {
    if (!grid_fits(cdiv(N, 4), 256)) return set_error(SPARDA_ERR_SHAPE, "append_paged: grid too large");
    uint32_t* status;
    if (const int rc = status_word(&status)) return rc;
    const Pages pg{p_st, s_st, h_st, table, t_st, static_cast<int>(width), static_cast<int>(n_pages)};
    const int es = dtype == SPARDA_F32 ? 4 : 2;
    hipLaunchKernelGGL(append_paged_kernel, dim3(static_cast<unsigned>(cdiv(N, 4))), dim3(256), 0, stream,
                       static_cast<char*>(k), static_cast<char*>(v), pg, static_cast<int>(ps), positions, cu,
                       static_cast<int>(n), static_cast<const char*>(k_new), static_cast<const char*>(v_new), N, new_st,
                       new_sh, static_cast<int>(Hkv), static_cast<int>(D * es), es, status);
    return check_hip(hipGetLastError(), "append_paged_kernel");
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------

namespace {

template <int DT>
struct PagedType;
template <>
struct PagedType<SPARDA_BF16> {
    static constexpr int kTiles = 2;   // 16-key tiles of a step
    typedef short E;
};
template <>
struct PagedType<SPARDA_F32> {
    static constexpr int kTiles = 1;
    typedef float E;
};

// The operands of one step, as loaded
template <int DT, int D>
struct PagedStep {
    static constexpr int kTiles = PagedType<DT>::kTiles;
    static constexpr int kQ = DT == SPARDA_F32 ? D / 16 : (D + 31) / 32;   // 16-byte pieces of K a lane holds per tile
    static constexpr int kV = D / 16;                                       // elements of V per key a lane holds
    typedef typename PagedType<DT>::E VRow __attribute__((ext_vector_type(kV)));
    uint4 k[kTiles][kQ];
    VRow v[kTiles][4];
};


}  // namespace

// One output of an item: the sequence's, or the item's partial.
template <int DT, int D>
__device__ __forceinline__ void paged_store(const PagedDecode& a, const Share& sh, int item, int h, int d, float O, float M,
                                            float L, bool bad) {
    if (sh.parts == 1) {
        // (an empty sequence: zeros)
        store_elem<DT>(a.out, sh.seq * a.out_sb + static_cast<int64_t>(h) * D + d, sh.len == 0 && !bad ? 0.0f : O / L);
    } else {
        const int64_t at = static_cast<int64_t>(item) * a.Hq + h;
        a.part_o[at * D + d] = O;
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
    }
}

// One workgroup of W = HG KW wavefronts per (HG head tiles, item): a head tile is
// up to 16 query heads of one KV head, and the HG tiles' wavefronts read the same
// positions at the same time, so that neighbouring heads' rows, which lie side by
// side in a page, are fetched together. The heads of a tile are the 16 columns of
// the matrix products:
//     S^T[key, head] = K[key, :] . Q[head, :]
//     P = exp2(S scale log2 e - m[head])
//     O^T[d, head] += V^T[d, key] . P^T[key, head]
// The KW wavefronts of a tile take the steps of the share in turn, each with its own
// (m, l, O); K and V go straight from the pages to the operand registers, the next
// step's under the present one's arithmetic, and S^T's layout is already that of the
// P operand, so nothing passes through LDS before the wavefronts are joined. A
// tile's 16 keys lie in one page (pages hold a multiple of 16 rows), so that its
// base address is a scalar. Bound by memory where the cache is long: 32 sequences of up to
// 16384 positions, 32/8 heads of 128, 1.43 GB in 246 us = 5.8 TB/s. 131000 positions of 12/4
// heads of 64, 134 MB, take 25.4 us from the last-level cache, of which a launch and the
// chain lengths, table, keys are 4; a call whose cache comes from memory takes 32.0 with the join.
template <int DT, int D, int HG, int KW>
__global__ void __launch_bounds__(HG* KW* kWave, D == 128 ? 2 : DT == SPARDA_F32 ? 3 : 4) decode_paged_kernel(PagedDecode a) {
    typedef PagedStep<DT, D> Step;
    constexpr int kTiles = Step::kTiles, kV = Step::kV, kQ = Step::kQ, kLogStep = kTiles == 1 ? 4 : 5, kStep = 1 << kLogStep, W = KW;
    static_assert(kStep == 16 * kTiles, "steps of 16 or 32 keys");
    extern __shared__ float lds[];
    const int lane = threadIdx.x % kWave;
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int wave = wv / HG;                               // among the wavefronts of a head tile
    const int c16 = lane % 16, grp = lane / 16;
    const int groups = a.Hkv * a.head_tiles / HG;
    const int item = blockIdx.x / groups, gt = blockIdx.x % groups * HG + wv % HG;
    const int g = gt / a.head_tiles, h0 = gt % a.head_tiles * 16;
    const int nh = a.R - h0 < 16 ? a.R - h0 : 16;           // query heads of the tile
    Share sh;
    if (a.whole) {
        const int l = __builtin_amdgcn_readfirstlane(a.len[item]), n = l < 0 ? 0 : l > a.cap ? a.cap : l;
        sh = Share{item, 0, 1, item, paged_steps(l, a.cap, kLogStep), n, l < 0 || l > a.cap};
    } else {
        sh = paged_item(a.len, a.B, a.cap, kLogStep, a.target, a.least, true, item);
    }
    if (sh.seq < 0) return;                                 // workgroup-uniform
    const int b = sh.seq, len = sh.len;
    const int steps = paged_steps(len, a.cap, kLogStep);
    const int s_end = min(steps, (sh.part + 1) * sh.share);
    bool bad = sh.bad;

    // this lane's column of Q
    uint4 qr[kQ];
#pragma unroll
    for (int i = 0; i < kQ; ++i) qr[i] = uint4{0, 0, 0, 0};
    {
        const int64_t qo = b * a.q_sb + static_cast<int64_t>(g * a.R + h0 + c16) * a.q_sh;
#pragma unroll
        for (int i = 0; i < kQ; ++i) {
            const int d = DT == SPARDA_F32 ? 16 * i + 4 * grp : 32 * i + 8 * grp;
            if (c16 < nh && d < D)
                qr[i] = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + (qo + d) * (DT == SPARDA_F32 ? 4 : 2));
        }
    }

    // the walk over the table: tile 2 u (or u) of step u in page `page`, `rem` tiles into it
    const int32_t* row = a.pg.table + b * a.pg.t_st;
    const int tile0 = (sh.part * sh.share + wave) * kTiles;
    int page = tile0 / a.ps16, rem = tile0 % a.ps16;
    const int adv_p = W * kTiles / a.ps16, adv_r = W * kTiles % a.ps16;
    const int last_tile = (len - 1) / 16;
    typedef typename PagedType<DT>::E E;
    const E* kg = static_cast<const E*>(a.k) + g * a.pg.h_st;
    const E* vg = static_cast<const E*>(a.v) + g * a.pg.h_st;
    const int s_st = static_cast<int>(a.pg.s_st);
    auto load = [&](int u, Step& x) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            int tile = u * kTiles + t, p = page, r = rem;
            if (t == 1) {
                if (tile > last_tile) --tile;                // past the end: the step's first tile again, masked
                else if (++r == a.ps16) r = 0, ++p;
            }
            int id = row[p];
            if (id < 0 || id >= a.pg.n_pages) bad = true, id = 0;
            const int last = len - 1 - 16 * tile;            // rows past the end read the last one
            const int64_t base = id * a.pg.p_st + static_cast<int64_t>(16 * r) * a.pg.s_st;
            const E* kb = kg + base;
            const E* vb = vg + base;
            const int kr = c16 < last ? c16 : last;
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
                const int d = DT == SPARDA_F32 ? 16 * i + 4 * grp : 32 * i + 8 * grp;
                x.k[t][i] = uint4{0, 0, 0, 0};
                if (D >= 32 || DT == SPARDA_F32 || d < D)
                    x.k[t][i] = *reinterpret_cast<const uint4*>(kb + (kr * s_st + d));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int vr = 4 * grp + i < last ? 4 * grp + i : last;
                x.v[t][i] = *reinterpret_cast<const typename Step::VRow*>(vb + (vr * s_st + kV * c16));
            }
        }
        rem += adv_r;
        page += adv_p;
        if (rem >= a.ps16) rem -= a.ps16, ++page;
    };

    float m = -__builtin_inff(), l = 0.0f;                   // the column's maximum (log2 units), this lane's part of its sum
    f32x4 o[kV];
#pragma unroll
    for (int j = 0; j < kV; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int u, Step& x) __attribute__((always_inline)) {
        f32x4 s[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
            f32x4 s4[4] = {s[t], s[t], s[t], s[t]};          // (fp32: four short sums, whose roundings are smaller)
#pragma unroll
            for (int i = 0; i < kQ; ++i) {
                if constexpr (DT == SPARDA_F32) {
                    const f32x4 ka = __builtin_bit_cast(f32x4, x.k[t][i]), qb = __builtin_bit_cast(f32x4, qr[i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s4[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[e], qb[e], s4[e], 0, 0, 0);
                } else {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[t][i]),
                                                                   __builtin_bit_cast(bf16x8, qr[i]), s[t], 0, 0, 0);
                }
            }
            if constexpr (DT == SPARDA_F32) s[t] = (s4[0] + s4[1]) + (s4[2] + s4[3]);
        }
        const int left = len - u * kStep - 4 * grp;          // this lane's keys 16 t + i below it are the sequence's
        if (u * kStep + kStep > len) {                       // the last step: the others weigh nothing
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (16 * t + i >= left) {
#pragma unroll
                        for (int j = 0; j < kV; ++j) x.v[t][i][j] = 0;
                    }
        }
        float mx = m;
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, 16 * t + i < left ? s[t][i] * a.scale_log2 : -__builtin_inff());
        mx = pair32_max(pair16_max(mx));
        const float ref = mx == -__builtin_inff() ? 0.0f : mx;
        const float alpha = __builtin_amdgcn_exp2f(m - ref);
        m = mx;
        l *= alpha;
        // one rounding between a score and its distance from the reference, which
        // is small where the weight is not
        float p[kTiles][4];
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[t][i] = 16 * t + i < left ? __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], a.scale_log2, -ref)) : 0.0f;
                l += p[t][i];
            }
#pragma unroll
        for (int j = 0; j < kV; ++j) o[j] *= alpha;
        if constexpr (DT == SPARDA_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kV; ++j)
                    o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[0][i][j], p[0][i], o[j], 0, 0, 0);
        } else {
            // P is rounded to bf16 for the product (the sum l keeps it in fp32)
            bf16x8 pb;
#pragma unroll
            for (int e = 0; e < 8; ++e) pb[e] = static_cast<__bf16>(p[e / 4][e % 4]);
#pragma unroll
            for (int j = 0; j < kV; ++j) {
                typedef short s16x8 __attribute__((ext_vector_type(8)));
                s16x8 va;
#pragma unroll
                for (int e = 0; e < 8; ++e) va[e] = x.v[e / 4][e % 4][j];
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), pb, o[j], 0, 0, 0);
            }
        }
    };

    int u = sh.part * sh.share + wave;
    if (u < s_end) {
        Step x, y;
        load(u, x);
        while (true) {                                       // wave-uniform
            if (u + W < s_end) load(u + W, y);
            compute(u, x);
            u += W;
            if (u >= s_end) break;
            if (u + W < s_end) load(u + W, x);
            compute(u, y);
            u += W;
            if (u >= s_end) break;
        }
    }
    l = pair32_sum(pair16_sum(l));

    const bool any_bad = __ballot(bad) != 0;                  // wave-uniform
    // ---- the wavefronts' partials, joined in order: thread -> (head, dim) ----
    const int hg = wv % HG;
    float* lo = lds + hg * KW * (a.lds_heads * (D + 4) + 33);     // [KW][lds_heads][D + 4]
    float* lm = lo + KW * a.lds_heads * (D + 4);                  // [KW][16][2]
    int* lbad = reinterpret_cast<int*>(lm + KW * 32);             // [KW]
    if (c16 < nh) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kV; ++j) lo[(wave * a.lds_heads + c16) * (D + 4) + kV * (4 * grp + i) + j] = o[j][i];
        if (grp == 0) {
            lm[(wave * 16 + c16) * 2] = m;
            lm[(wave * 16 + c16) * 2 + 1] = l;
        }
    }
    if (lane == 0) lbad[wave] = any_bad ? 1 : 0;
    __syncthreads();
    int bads = 0;
#pragma unroll
    for (int w = 0; w < KW; ++w) bads |= lbad[w];
    if (bads != 0 && wave == 0 && lane == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_PAGE_RANGE));
    for (int e = wave * kWave + lane; e < nh * D; e += KW * kWave) {
        const int c = e / D, d = e % D;
        float mw[KW], M = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            mw[w] = lm[(w * 16 + c) * 2];
            M = fmaxf(M, mw[w]);
        }
        const float ref = M == -__builtin_inff() ? 0.0f : M;
        float L = 0.0f, O = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            const float wt = __builtin_amdgcn_exp2f(mw[w] - ref);
            L = __builtin_fmaf(wt, lm[(w * 16 + c) * 2 + 1], L);
            O = __builtin_fmaf(wt, lo[(w * a.lds_heads + c) * (D + 4) + d], O);
        }
        paged_store<DT, D>(a, sh, item, g * a.R + h0 + c, d, bads ? __builtin_nanf("") : O, M, L, bads != 0);
    }
}

// Joins the items of a sequence, one workgroup per (32 dims of a query head, sequence):
//     M = max m_i, out = sum exp2(m_i - M) O_i / sum exp2(m_i - M) l_i.
// The items' weights once into LDS, then dims over the lanes and the items over the
// thread groups (8 loads in flight each), added in group order. Bound by two
// latencies, the weights' and the partials' (3.7 to 5.4 us): with a whole head a
// workgroup 1 x 20000 positions take 12.8 against 11.7 us, 1 x 131000 31.6 / 30.8,
// with 16 dims 8 x 16384 26.1 / 25.5.
template <int DT, int D, int LOG>
__global__ void __launch_bounds__(kPgJoin) decode_paged_join_kernel(PagedDecode a) {
    constexpr int JD = D < 32 ? D : 32;                       // dims of a workgroup
    constexpr int kG = kPgJoin / JD, kChunk = 1024, kJW = kPgJoin / kWave;
    __shared__ float red[kPgJoin], wts[kChunk], rm[kJW], rl[kJW];
    const int b = blockIdx.y, h = blockIdx.x / (D / JD), d0 = blockIdx.x % (D / JD) * JD, tid = threadIdx.x, wave = tid / kWave;
    const Share sh = paged_item(a.len, a.B, a.cap, LOG, a.target, a.least, false, b);
    if (sh.parts <= 1) return;                                // written by its one item
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + static_cast<int64_t>(sh.first) * a.Hq + h;
    const float* po = a.part_o + (static_cast<int64_t>(sh.first) * a.Hq + h) * D + d0 + tid % JD;
    const int64_t st = static_cast<int64_t>(a.Hq) * D;
    float first[8];                                           // the thread's first items, under the weights' latency
#pragma unroll
    for (int e = 0; e < 8; ++e) first[e] = tid / JD + e * kG < sh.parts ? po[(tid / JD + e * kG) * st] : 0.0f;
    float M = -__builtin_inff();
    for (int i = tid; i < sh.parts; i += kPgJoin) M = fmaxf(M, ml[static_cast<int64_t>(i) * a.Hq].x);
    M = wave_max(M);
    if (tid % kWave == 0) rm[wave] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJW; ++w) M = fmaxf(M, rm[w]);
    const float ref = M == -__builtin_inff() ? 0.0f : M;
    float L = 0.0f, O = 0.0f;
    for (int c0 = 0; c0 < sh.parts; c0 += kChunk) {
        const int n = sh.parts - c0 < kChunk ? sh.parts - c0 : kChunk;
        if (c0 > 0) __syncthreads();                          // the last chunk's weights have been read
        for (int i = tid; i < n; i += kPgJoin) {
            const float2 x = ml[static_cast<int64_t>(c0 + i) * a.Hq];
            const float wt = __builtin_amdgcn_exp2f(x.x - ref);
            wts[i] = wt;
            L = __builtin_fmaf(wt, x.y, L);
        }
        __syncthreads();
        int i = tid / JD;
        if (c0 == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) O = i + e * kG < n ? __builtin_fmaf(wts[i + e * kG], first[e], O) : O;
            i += 8 * kG;
        }
        for (; i + 7 * kG < n; i += 8 * kG) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = po[(c0 + i + e * kG) * st];
#pragma unroll
            for (int e = 0; e < 8; ++e) O = __builtin_fmaf(wts[i + e * kG], x[e], O);
        }
        for (; i < n; i += kG) O = __builtin_fmaf(wts[i], po[(c0 + i) * st], O);
    }
    asm volatile("s_nop 1" : "+v"(L));  // the wait states of the reduction's first DPP, on every way out of the loop
    L = wave_sum(L);
    if (tid % kWave == 0) rl[wave] = L;
    red[tid] = O;
    __syncthreads();
    if (tid >= JD) return;
    float den = 0.0f;
#pragma unroll
    for (int w = 0; w < kJW; ++w) den += rl[w];
#pragma unroll
    for (int i = 1; i < kG; ++i) O += red[i * JD + tid];
    store_elem<DT>(a.out, b * a.out_sb + static_cast<int64_t>(h) * D + d0 + tid, O / den);
}

// The same where sequences have few items in the mean: one thread per (query head,
// dim), items in order, eight in flight. Bound by the launch and two dependent loads: 3.0 us for 1000 positions of 12
// heads of 64.
template <int DT, int D, int LOG>
__global__ void __launch_bounds__(256) decode_paged_join_few_kernel(PagedDecode a) {
    const int b = blockIdx.y, h = blockIdx.x * (256 / D) + threadIdx.x / D, d = threadIdx.x % D;
    const Share sh = paged_item(a.len, a.B, a.cap, LOG, a.target, a.least, false, b);
    if (sh.parts <= 1 || h >= a.Hq) return;                   // written by its one item
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + static_cast<int64_t>(sh.first) * a.Hq + h;
    const float* po = a.part_o + (static_cast<int64_t>(sh.first) * a.Hq + h) * D + d;
    const int64_t st = static_cast<int64_t>(a.Hq) * D;
    float m = -__builtin_inff(), L = 0.0f, O = 0.0f;
    for (int i0 = 0; i0 < sh.parts; i0 += 8) {
        float2 x[8];
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = i0 + e < sh.parts ? i0 + e : sh.parts - 1;
            x[e] = ml[static_cast<int64_t>(i) * a.Hq];
            y[e] = po[i * st];
        }
        float M = m;
#pragma unroll
        for (int e = 0; e < 8; ++e) M = fmaxf(M, x[e].x);
        const float ref = M == -__builtin_inff() ? 0.0f : M, alpha = __builtin_amdgcn_exp2f(m - ref);
        L *= alpha;
        O *= alpha;
        m = M;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i0 + e < sh.parts) {
                const float wt = __builtin_amdgcn_exp2f(x[e].x - ref);
                L = __builtin_fmaf(wt, x[e].y, L);
                O = __builtin_fmaf(wt, y[e], O);
            }
    }
    store_elem<DT>(a.out, b * a.out_sb + static_cast<int64_t>(h) * D + d, O / L);
}

namespace {

// How a launch is cut. us, 12/4 heads of 64 and 32/8 of 128 where named:
//  - A table whose sequences are short, or a batch that gives every CU a workgroup:
//    one item a sequence, written straight to the output, no second launch
//    (B=1, 200 positions 4.6 against 6.3 in shares, 500 6.2 / 6.4; B=4, 600: 6.7 / 7.4; B=16,
//    300: 5.3 / 7.5; 200 of 32/8 heads 5.8 / 7.3; B=64, 1000: 11.3 / 15.0; B=1000, 2000:
//    253 / 269). Fewer and longer sequences are faster in shares (B=1, 1000: 8.7 / 6.4;
//    500 of 32/8 heads 8.3 / 7.5; B=128, 4000: 75.0 / 68.6).
//  - Many (sequence, head) pairs, or several of long sequences: workgroups of 2 or 4
//    neighbouring heads, which fetch whole rows of a page at a time (B=32, 16384, 32/8
//    heads of 128: 257 against 290 with one head a workgroup; 8/8 heads of 64: 137 / 180;
//    caches read from memory, B=8, 16384: 28.3 / 30.4, B=2, 100000: 45.9 / 48.1; but
//    8 x 4000 13.5 / 13.1, 2 x 10000 13.3 / 11.6, 1 x 131000 36.0 / 35.0: lengths from a
//    quarter of the longest up. Where all are as long as the table, neighbouring heads lead
//    from below the limit on: B=8, 4000: 15.3 / 16.5, 6000: 19.5 / 20.4, 8000: 21.9 / 23.3, 12000:
//    27.8 / 29.9; B=2, 20000: 17.1 / 17.8, 50000: 28.4 / 30.5).
//  - Otherwise one head a workgroup: four wavefronts on its keys make four times
//    fewer partials for the join (B=1, 131000: 31.4 / 35). Two workgroups a CU: fewer do
//    not keep the memory busy, more cost a longer join (256 / 512 / 1024 / 2048 with the
//    caches read from memory, B=1, 131000: 41.9 / 35.2 / 36.0 / 37.6, 40000: 17.8 / 16.9 / 18.5 /
//    18.2; B=16, 4000: 20.6 / 18.2 / 18.8 / 19.6; B=1, 50000, 32/8 heads of 128 49.4 / 49.2 /
//    50.9 / 54.2). (Caches that the last-level cache holds would have 256, by 5%.)
//  - The join: one thread a dim where a sequence has 16 items in the mean, items over thread
//    groups where it has more. us of the first / the second, caches read from memory: B=1, 1000:
//    7.1 / 7.9; B=16, 4000: 21.7 / 22.3; B=32 of 16384, 32/8 heads of 128 381 / 395; B=32 of 300 in a
//    table of 131072 12.3 / 14.2; B=4, 3000: 12.1 / 11.4. The host knows the mean alone: one
//    sequence among many short ones gets nearly all items, and one thread a dim then walks
//    hundreds of them (131000 and 31 of 300: 68.0 / 38.0; 32768 and 31 of 200, 32/8 heads of 128
//    57.7 / 56.4).
struct PagedPlan {
    int hg, kw;              // head tiles, and wavefronts for each, of a workgroup
    int64_t target, least;   // items aimed at, steps of the smallest item
    int64_t items, groups;   // items at most, workgroups an item
    bool few;                // a sequence has few items in the mean
};
PagedPlan paged_plan(int64_t B, int64_t cap, int64_t Hq, int64_t Hkv, int64_t D, int dtype) {
    const int64_t R = Hq / Hkv, heads = Hkv * cdiv(R, 16), steps = cdiv(cap, dtype == SPARDA_F32 ? 16 : 32);
    const int even = heads % 4 == 0 ? 4 : heads % 2 == 0 ? 2 : 1;
    const bool eight = (R < 16 ? R : 16) * (D + 4) + 33 <= 2048;  // eight wavefronts' partials fit 64 KB of LDS
    PagedPlan p{1, 4, 1, 4, 0, 0, false};
    if (steps <= (D == 128 ? 12 : B == 1 ? 16 : 20) || (steps <= 64 && B * heads >= 128)) {
        p.least = steps;
        if (eight && steps > 8 && B * heads < 512) p.kw = 8;
    } else if (eight && even > 1 && (B * heads >= 128 || (B * heads >= 8 && B * heads * steps >= 7168))) {
        p.hg = even;
        p.kw = 8 / even;
        // (items are target + B at most: whole rounds of 512 or 256 workgroups, half of one at least beside the B)
        const int64_t round = cdiv(B * heads >= 128 ? 512 : 256, heads / even);
        p.target = cdiv(B + round / 2, round) * round - B;
    } else {
        p.target = 512 / heads - B / 2;
    }
    if (p.target < 1) p.target = 1;
    p.groups = heads / p.hg;
    p.items = p.target + B;
    const int64_t most = B * cdiv(steps, p.least);   // every share the smallest
    if (p.items > most) p.items = most;
    p.few = p.items <= 16 * B;
    return p;
}

}  // namespace

size_t decode_paged_workspace_bytes(int64_t B, int64_t cap, int64_t Hq, int64_t Hkv, int64_t D, int dtype) {
    const PagedPlan p = paged_plan(B, cap, Hq, Hkv, D, dtype);
    // one item a sequence: written by the item itself
    return p.items <= B ? 0 : static_cast<size_t>(p.items * Hq * (D + 2)) * sizeof(float);
}

void launch_paged_join(const PagedDecode& a, int64_t D, int dtype, int log_step, bool few, hipStream_t stream) {
    // (the step is a constant of the kernel: read from its arguments it cost 0.25 us a call)
#define SPARDA_PGJ(DT_, D_, LOG_)                                                                                 \
    if (few)                                                                                                      \
        hipLaunchKernelGGL((decode_paged_join_few_kernel<DT_, D_, LOG_>),                                         \
                           dim3(static_cast<unsigned>(cdiv(a.Hq, 256 / D_)), static_cast<unsigned>(a.B)), dim3(256), 0, stream, a); \
    else                                                                                                          \
        hipLaunchKernelGGL((decode_paged_join_kernel<DT_, D_, LOG_>),                                             \
                           dim3(static_cast<unsigned>(a.Hq * (D_ < 32 ? 1 : D_ / 32)), static_cast<unsigned>(a.B)), dim3(kPgJoin), 0, stream, a)
#define SPARDA_PGJ_D(DT_, LOG_)                     \
    switch (D) {                                    \
        case 16: SPARDA_PGJ(DT_, 16, LOG_); break;  \
        case 32: SPARDA_PGJ(DT_, 32, LOG_); break;  \
        case 64: SPARDA_PGJ(DT_, 64, LOG_); break;  \
        default: SPARDA_PGJ(DT_, 128, LOG_); break; \
    }
    if (dtype != SPARDA_F32) SPARDA_PGJ_D(SPARDA_BF16, 5)
    else if (log_step == 5) SPARDA_PGJ_D(SPARDA_F32, 5)
    else SPARDA_PGJ_D(SPARDA_F32, 4)
#undef SPARDA_PGJ_D
#undef SPARDA_PGJ
}

int launch_decode_paged(const void* q, int64_t q_sb, int64_t q_sh, const void* k, const void* v, int64_t n_pages,
                        int64_t ps, int64_t p_st, int64_t s_st, int64_t h_st, int dtype, const int32_t* table,
                        int64_t t_st, int64_t width, const int32_t* len, int64_t B, int64_t Hq, int64_t Hkv, int64_t D,
                        float scale, void* out, int64_t out_sb, void* workspace, hipStream_t stream) {
    PagedDecode a{};
    const int64_t cap = width * ps, R = Hq / Hkv;
    const PagedPlan p = paged_plan(B, cap, Hq, Hkv, D, dtype);
    if (!grid_fits(p.items * p.groups, p.hg * p.kw * kWave)) return set_error(SPARDA_ERR_SHAPE, "decode_paged: grid too large");
    if (const int rc = status_word(&a.status)) return rc;
    a.q = q, a.q_sb = q_sb, a.q_sh = q_sh, a.k = k, a.v = v;
    a.pg = Pages{p_st, s_st, h_st, table, t_st, static_cast<int>(width), static_cast<int>(n_pages)};
    a.ps16 = static_cast<int>(ps / 16), a.len = len, a.B = static_cast<int>(B), a.cap = static_cast<int>(cap);
    a.Hq = static_cast<int>(Hq), a.Hkv = static_cast<int>(Hkv), a.R = static_cast<int>(R);
    a.head_tiles = static_cast<int>(cdiv(R, 16));
    a.target = static_cast<int>(p.target), a.least = static_cast<int>(p.least);
    a.whole = p.items <= B;
    a.lds_heads = static_cast<int>(R < 16 ? R : 16);
    a.scale_log2 = scale * kPgLog2e, a.out = out, a.out_sb = out_sb;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = workspace ? a.part_o + p.items * Hq * D : nullptr;
    const dim3 grid(static_cast<unsigned>(p.items * p.groups));
#define SPARDA_PGD_W(DT_, D_, HG_, KW_)                                                                           \
    hipLaunchKernelGGL((decode_paged_kernel<DT_, D_, HG_, KW_>), grid, dim3(HG_ * KW_ * kWave),                   \
                       HG_ * KW_ * (a.lds_heads * ((D_) + 4) + 33) * sizeof(float), stream, a)
#define SPARDA_PGD(DT_, D_)                                                                                       \
    do {                                                                                                          \
        if (p.hg == 4) SPARDA_PGD_W(DT_, D_, 4, 2);                                                               \
        else if (p.hg == 2) SPARDA_PGD_W(DT_, D_, 2, 4);                                                          \
        else if (p.kw == 4) SPARDA_PGD_W(DT_, D_, 1, 4);                                                          \
        else SPARDA_PGD_W(DT_, D_, 1, 8);                                                                         \
    } while (0)
#define SPARDA_PGD_D(DT_)                     \
    switch (D) {                              \
        case 16: SPARDA_PGD(DT_, 16); break;  \
        case 32: SPARDA_PGD(DT_, 32); break;  \
        case 64: SPARDA_PGD(DT_, 64); break;  \
        default: SPARDA_PGD(DT_, 128); break; \
    }
    if (dtype == SPARDA_F32) SPARDA_PGD_D(SPARDA_F32)
    else SPARDA_PGD_D(SPARDA_BF16)
#undef SPARDA_PGD_D
#undef SPARDA_PGD_W
#undef SPARDA_PGD
    if (p.items > B) launch_paged_join(a, D, dtype, dtype == SPARDA_F32 ? 4 : 5, p.few, stream);
    return check_hip(hipGetLastError(), "decode_paged_kernel");
}

}  // namespace sparda
