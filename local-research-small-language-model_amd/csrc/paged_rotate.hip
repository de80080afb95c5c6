// The write of new keys and values into a cache in pages with the position
// rotation applied on the way (sparda_rotate_append_paged), queries beside them.
#include "common.h"
#include "kernels.h"
#include "paged.h"
#include "rotate.h"

namespace sparda {

// One wavefront per new row: its sequence, position and page, then the heads in pairs of
// 16-byte pieces (i, i + D/2), the queries' first and the keys' behind them, then the
// values, copied. D/2 holds 1 to 16 pieces, so a lane's piece of the angles is the same
// for every head and is loaded once.
template <int DT, int D>
__global__ void __launch_bounds__(256) rotate_append_paged_kernel(RotateAppend a, char* __restrict__ k, char* __restrict__ v) {
    constexpr int kEs = DT == SPARDA_F32 ? 4 : 2, kVe = 16 / kEs, kPer = D / 2 / kVe, kBatch = 4;
    const int lane = threadIdx.x % kWave;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (t >= a.N) return;
    const PagedRow r = paged_row(a.pg, a.ps, a.positions, a.cu, a.n, a.N, t, a.status);
    if (!r.takes) return;
    const bool off_table = r.pos >= a.rows;                   // the angles end before this position
    if (off_table && lane == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_POSITION_RANGE));
    const bool keep = r.page >= 0 && !off_table;              // otherwise the row is dropped
    const int c = lane % kPer;
    float cs[kVe], sn[kVe];
    load_angles<kVe>(a, r.pos, c * kVe, off_table, cs, sn);
    const char* q = static_cast<const char*>(a.q) + t * a.q_st * kEs + c * 16;
    char* qo = static_cast<char*>(a.q_out) + t * a.qo_st * kEs + c * 16;
    const char* kn = static_cast<const char*>(a.k_new) + t * a.new_st * kEs + c * 16;
    const int64_t to = (r.page * a.pg.p_st + r.row * a.pg.s_st) * kEs;
    const int heads = a.Hq + (keep ? a.Hkv : 0);
    for (int h0 = lane / kPer; h0 < heads; h0 += kBatch * (kWave / kPer)) {
        uint4 x[kBatch], y[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int h = h0 + e * (kWave / kPer);
            if (h < heads) {
                const char* from = h < a.Hq ? q + h * a.q_sh * kEs : kn + (h - a.Hq) * a.new_sh * kEs;
                x[e] = *reinterpret_cast<const uint4*>(from);
                y[e] = *reinterpret_cast<const uint4*>(from + D / 2 * kEs);
            }
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int h = h0 + e * (kWave / kPer);
            if (h < heads) {
                char* dst = h < a.Hq ? qo + h * a.qo_sh * kEs : k + to + (h - a.Hq) * a.pg.h_st * kEs + c * 16;
                turn_pieces<DT>(x[e], y[e], cs, sn);
                *reinterpret_cast<uint4*>(dst) = x[e];
                *reinterpret_cast<uint4*>(dst + D / 2 * kEs) = y[e];
            }
        }
    }
    if (!keep) return;
    const char* vn = static_cast<const char*>(a.v_new) + t * a.new_st * kEs;
    for (int i = lane; i < a.Hkv * 2 * kPer; i += kWave) {
        const int h = i / (2 * kPer), o = i % (2 * kPer) * 16;
        *reinterpret_cast<uint4*>(v + to + h * a.pg.h_st * kEs + o) = *reinterpret_cast<const uint4*>(vn + h * a.new_sh * kEs + o);
    }
}

int launch_rotate_append_paged(const RotateAppend& given, void* k, void* v, int dtype, int64_t D, hipStream_t stream) {
    RotateAppend a = given;
    if (!grid_fits(cdiv(a.N, 4), 256)) return set_error(SPARDA_ERR_SHAPE, "rotate_append_paged: grid too large");
    if (const int rc = status_word(&a.status)) return rc;
    const dim3 grid(static_cast<unsigned>(cdiv(a.N, 4)));
#define SPARDA_RA(DT_, D_)                                                                              \
    hipLaunchKernelGGL((rotate_append_paged_kernel<DT_, D_>), grid, dim3(256), 0, stream, a, static_cast<char*>(k), \
                       static_cast<char*>(v))
#define SPARDA_RA_D(DT_)                      \
    switch (D) {                              \
        case 16: SPARDA_RA(DT_, 16); break;   \
        case 32: SPARDA_RA(DT_, 32); break;   \
        case 64: SPARDA_RA(DT_, 64); break;   \
        default: SPARDA_RA(DT_, 128); break;  \
    }
    if (dtype == SPARDA_F32) SPARDA_RA_D(SPARDA_F32)
    else SPARDA_RA_D(SPARDA_BF16)
#undef SPARDA_RA_D
#undef SPARDA_RA
    return check_hip(hipGetLastError(), "rotate_append_paged_kernel");
}

}  // namespace sparda
