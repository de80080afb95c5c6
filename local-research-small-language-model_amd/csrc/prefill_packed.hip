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

int launch_prefill_packed(const void* q, int64_t q_st, int64_t q_sh, const void* k, const void* v, int64_t kv_st,
                          int64_t kv_sh, int dtype, const int32_t* cu, int64_t n, int64_t N, int64_t Hq, int64_t Hkv,
                          int64_t D, int causal, float scale, void* out, int64_t out_st, hipStream_t stream) {
    uint32_t* status;
    if (const int rc = status_word(&status)) return rc;
    const int64_t R = Hq / Hkv;
    const float sl = scale * kPkLog2e;
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
