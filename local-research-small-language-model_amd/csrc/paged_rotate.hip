// The write of new keys and values into a cache in pages with the position
// rotation applied on the way (sparda_rotate_append_paged), queries beside them.
#include "common.h"
#include "kernels.h"
#include "paged.h"
#include "rotate.h"

namespace sparda {

// One wavefront per new row: its sequence, position and page, then the heads in pairs of
// 16-byte pieces (i, i + D/2), the queries' first and the keys' behind them, then the
// values, copied. Bound by memory: 16000 rows of 32/8 heads of 128, 393 MB read and written, take 62 us
// = 6.3 TB/s (part of it stays in the last-level cache), 77 in a row of calls = 5.1 TB/s, as large copies do; 64 rows of 12/4 heads of 64 5.0 us a call, of which the
// host's part is 4.5.
template <int DT, int D, bool ONCE>
__global__ void __launch_bounds__(256) rotate_append_paged_kernel(RotateAppend a, char* __restrict__ k, char* __restrict__ v) {
    constexpr int kEs = DT == SPARDA_F32 ? 4 : 2, kPieces = D * kEs / 16;
    const int lane = threadIdx.x % kWave;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (t >= a.N) return;
    const PagedRow r = paged_row(a.pg, a.ps, a.positions, a.cu, a.n, a.N, t, a.status);
    if (!r.takes) return;
    const bool off_table = r.pos >= a.rows;                   // the angles end before this position
    if (off_table && lane == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_POSITION_RANGE));
    const bool keep = r.page >= 0 && !off_table;              // otherwise the row is dropped
    const char* q = static_cast<const char*>(a.q) + t * a.q_st * kEs;
    char* qo = static_cast<char*>(a.q_out) + t * a.qo_st * kEs;
    const char* kn = static_cast<const char*>(a.k_new) + t * a.new_st * kEs;
    const int64_t at = (r.page * a.pg.p_st + r.row * a.pg.s_st) * kEs;
    turn_heads<DT, D, ONCE>(a, r.pos, off_table, a.Hq + (keep ? a.Hkv : 0),
                      [&](int h) { return h < a.Hq ? q + h * a.q_sh * kEs : kn + (h - a.Hq) * a.new_sh * kEs; },
                      [&](int h) { return h < a.Hq ? qo + h * a.qo_sh * kEs : k + at + (h - a.Hq) * a.pg.h_st * kEs; });
    if (!keep) return;
    const char* vn = static_cast<const char*>(a.v_new) + t * a.new_st * kEs;
    for (int i = lane; i < a.Hkv * kPieces; i += kWave) {
        const int h = i / kPieces, o = i % kPieces * 16;
        *reinterpret_cast<uint4*>(v + at + h * a.pg.h_st * kEs + o) = load_row<ONCE>(vn + h * a.new_sh * kEs + o);
    }
}

int launch_rotate_append_paged(const RotateAppend& given, void* k, void* v, int dtype, int64_t D, hipStream_t stream) {
    RotateAppend a = given;
    if (!grid_fits(cdiv(a.N, 4), 256)) return set_error(SPARDA_ERR_SHAPE, "rotate_append_paged: grid too large");
    if (const int rc = status_word(&a.status)) return rc;
    const dim3 grid(static_cast<unsigned>(cdiv(a.N, 4)));
    const bool once = rows_past_cache(a, D, dtype);
#define SPARDA_RA(DT_, D_)                                                                                          \
    do {                                                                                                            \
        if (once) hipLaunchKernelGGL((rotate_append_paged_kernel<DT_, D_, true>), grid, dim3(256), 0, stream, a,    \
                                     static_cast<char*>(k), static_cast<char*>(v));                                 \
        else hipLaunchKernelGGL((rotate_append_paged_kernel<DT_, D_, false>), grid, dim3(256), 0, stream, a,        \
                                static_cast<char*>(k), static_cast<char*>(v));                                      \
    } while (0)
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
