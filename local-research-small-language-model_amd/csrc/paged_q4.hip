// A key-value cache in pages of 4-bit codes (sparda_append_paged_q4,
// sparda_gather_paged_q4, sparda_decode_paged_q4).
//
// Dims are taken in groups of 32 (a head of 16 dims is half a group). A group of
// a row x, in bf16, is held as h (2 c - 15), c in 0 .. 15 a dim and h = max|x| / 15 in
// fp16: the odd multiples of h, of which the nearest to x is that of
// c = floor(x / 2h) + 8. 4.5 bits a dim; a row of N(0,1) comes back with a relative error
// of 9%. One number a group (no offset) costs the products no second sum: the
// levels' middle, 7.5, is the same for all.
//
// 16 positions of a head (a tile) lie together, 576 bytes a group, G groups a head:
//   keys' codes    [16 positions][4 quarters][G][4 bytes]: quarter p of group i holds dims
//                  32 i + 8 p + e, e = 0 .. 7, in nibble e/2 + 4 (e % 2), so that nibbles four apart
//                  are neighbouring dims
//   values' codes  [4 fours of positions][16 pairs w][G][4 bytes]: byte s is position
//                  {0, 2, 1, 3}[s] of the four, its nibbles dims 32 g + 2 w and + 1
//   keys' h        [16 positions][G], then the values' h
// Both are what a lane of the matrix products takes (decode below), and a wavefront reads
// a tile's codes as one block of memory.
#include "common.h"
#include "kernels.h"
#include "mfma.h"
#include "paged.h"
#include "rotate.h"

#include <type_traits>

namespace sparda {

namespace {

constexpr int q4_groups(int D) { return D < 32 ? 1 : D / 32; }

// h of a group from the bits of its largest magnitude. A value that is not finite makes the
// group NaN; magnitudes above 15 * 65504 are cut off.
__device__ __forceinline__ _Float16 q4_scale(uint32_t top) {
    if (top >= 0x7f800000u) return __builtin_bit_cast(_Float16, static_cast<uint16_t>(0x7e00));
    const float h = __uint_as_float(top) / 15.0f;
    return static_cast<_Float16>(h < 65504.0f ? h : 65504.0f);
}

// floor(x / 2h) + 8 in 0 .. 15, exactly: the rounded quotient is within half of the
// true one, so that one of its neighbours is the floor, and x - n 2h, on a grid of
// at most 14 bits, has no rounding to hide its sign.
__device__ __forceinline__ uint32_t q4_code(float x, float h2, float inv) {
    const float n = fminf(fmaxf(__builtin_rintf(x * inv), -9.0f), 8.0f);   // (where h is cut off, x / 2h may be any number)
    const float e = __builtin_fmaf(-n, h2, x);
    const int c = static_cast<int>(n) - (e < 0.0f ? 1 : 0) + 8;
    return static_cast<uint32_t>(c < 0 ? 0 : c > 15 ? 15 : c);
}

// Eight codes of a group of one number h.
__device__ __forceinline__ void q4_codes(const float (&x)[8], _Float16 h, uint32_t (&c)[8]) {
    const float h2 = 2.0f * static_cast<float>(h);
    if (!(h2 > 0.0f)) {                            // zeros, or NaN: any code
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = 8;
        return;
    }
    const float inv = 1.0f / h2;
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = q4_code(x[e], h2, inv);
}

// Eight elements of a row, as bf16 values in fp32 (round: fp32 rows are rounded)
template <int DT, bool ONCE>
__device__ __forceinline__ void q4_load8(const char* p, float (&x)[8]) {
    auto load = [](const char* at) { return load_row<ONCE>(at); };
    const uint4 a = load(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    if constexpr (DT == SPARDA_F32) {
        const uint4 b = load(p + 16);
        const uint32_t r[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(w[e]), x[4 + e] = __uint_as_float(r[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = __uint_as_float(w[e] << 16), x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
}
template <int DT>
__device__ __forceinline__ void q4_store8(char* p, const float (&x)[8]) {
    if constexpr (DT == SPARDA_F32) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 16) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
__device__ __forceinline__ uint32_t q4_top(float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = static_cast<float>(static_cast<__bf16>(x[e]));
        m = max(m, __float_as_uint(x[e]) & 0x7fffffffu);
    }
    return m;
}
// the largest over neighbouring lanes: 2 or 4 of them
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32_max(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, false)));
}
template <int LANES>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    if constexpr (LANES >= 2) asm volatile("s_nop 1" : "+v"(v));  // the wait states of the first DPP, on every way here
    if constexpr (LANES >= 2) v = dpp_u32_max<kDppXor1>(v);
    if constexpr (LANES >= 4) v = dpp_u32_max<kDppXor2>(v);
    return v;
}

// byte offsets in a tile
template <int G>
__device__ __forceinline__ int q4_key_word(int key, int dim) { return key * 16 * G + dim % 32 / 8 * 4 * G + dim / 32 * 4; }
template <int G>
__device__ __forceinline__ int q4_value_byte(int key, int dim) {
    const int i = key % 4, slot = i == 1 ? 2 : i == 2 ? 1 : i;
    return 256 * G + (key / 4 * 16 + dim % 32 / 2) * 4 * G + dim / 32 * 4 + slot;
}
template <int G>
__device__ __forceinline__ int q4_scale_at(int which, int key, int group) { return 512 * G + which * 32 * G + (key * G + group) * 2; }

__device__ __forceinline__ uint32_t q4_key_pack(const uint32_t (&c)[8]) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= c[e] << (4 * (e / 2 + 4 * (e % 2)));
    return w;
}

}  // namespace

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------

// One wavefront per new row. A lane takes eight dims and the eight that they are paired
// with; the largest magnitude of a group comes from up to four neighbouring lanes. The queries are rotated
// as for 16-bit pages, four heads at a time. Bound by memory: 16000 rows of 32/8 heads of 128 (196.6 MB read,
// 149.4 written) take 65.5 us = 5.3 TB/s (counted: 158 MB written, a row holding single bytes of the values' words). 64 rows of 12/4 heads of 64 take 5.2 us, a chain of five dependent
// loads. Neighbouring rows on one XCD: 77.5 against 78.2 us (then), not taken.
template <int DT, int D, bool ROT, bool ONCE>
__global__ void __launch_bounds__(256) append_paged_q4_kernel(RotateAppend a, char* __restrict__ pages) {
    constexpr int G = q4_groups(D), kEs = DT == SPARDA_F32 ? 4 : 2, kPer = D / 16;
    const int lane = threadIdx.x % kWave;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (t >= a.N) return;
    const PagedRow r = paged_row(a.pg, a.ps, a.positions, a.cu, a.n, a.N, t, a.status);
    if (!r.takes) return;
    const bool off_table = ROT && r.pos >= a.rows;
    if (off_table && lane == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_POSITION_RANGE));
    const bool keep = r.page >= 0 && !off_table;
    if constexpr (ROT) {
        const char* q = static_cast<const char*>(a.q) + t * a.q_st * kEs;
        char* qo = static_cast<char*>(a.q_out) + t * a.qo_st * kEs;
        turn_heads<DT, D, ONCE>(a, r.pos, off_table, a.Hq, [&](int h) { return q + h * a.q_sh * kEs; }, [&](int h) { return qo + h * a.qo_sh * kEs; });
    }
    if (!keep) return;
    const int key = static_cast<int>(r.row % 16);
    char* tiles = pages + r.page * a.pg.p_st + r.row / 16 * (576 * G);
    const int c = lane % kPer;
    float cs[8], sn[8];
    if constexpr (ROT) load_angles<8>(a, r.pos, c * 8, false, cs, sn);
    for (int h = lane / kPer; h < a.Hkv; h += kWave / kPer) {
        const char* from = static_cast<const char*>(a.k_new) + (t * a.new_st + h * a.new_sh + c * 8) * kEs;
        char* tile = tiles + h * a.pg.h_st;
        float x[2][8];
        q4_load8<DT, ONCE>(from, x[0]);
        q4_load8<DT, ONCE>(from + D / 2 * kEs, x[1]);
        if constexpr (ROT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) turn(x[0][e], x[1][e], cs[e], sn[e]);
        }
        uint32_t top[2] = {q4_top(x[0]), q4_top(x[1])};
        if constexpr (D < 64) top[0] = top[1] = max(top[0], top[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const _Float16 hh = q4_scale(lanes_max<(D >= 64 ? 4 : D == 32 ? 2 : 1)>(top[i]));
            const int dim = i * (D / 2) + c * 8;
            uint32_t code[8];
            q4_codes(x[i], hh, code);
            *reinterpret_cast<uint32_t*>(tile + q4_key_word<G>(key, dim)) = q4_key_pack(code);
            if (dim % 32 == 0) *reinterpret_cast<_Float16*>(tile + q4_scale_at<G>(0, key, dim / 32)) = hh;
        }
    }
    for (int i = lane; i < a.Hkv * 2 * kPer; i += kWave) {
        const int h = i / (2 * kPer), dim = i % (2 * kPer) * 8;
        char* tile = tiles + h * a.pg.h_st;
        float x[8];
        q4_load8<DT, ONCE>(static_cast<const char*>(a.v_new) + (t * a.new_st + h * a.new_sh + dim) * kEs, x);
        const _Float16 hh = q4_scale(lanes_max<(D >= 32 ? 4 : 2)>(q4_top(x)));
        uint32_t code[8];
        q4_codes(x, hh, code);
#pragma unroll
        for (int e = 0; e < 8; e += 2)
            *reinterpret_cast<uint8_t*>(tile + q4_value_byte<G>(key, dim + e)) = static_cast<uint8_t>(code[e] | code[e + 1] << 4);
        if (dim % 32 == 0) *reinterpret_cast<_Float16*>(tile + q4_scale_at<G>(1, key, dim / 32)) = hh;
    }
}

// ---------------------------------------------------------------------------
// gather
// ---------------------------------------------------------------------------

// One wavefront per row, eight dims a lane: the values that the codes stand for. Bound by memory: 17486
// rows of 8 heads of 128 (20.1 MB of codes, 71.6 written) take 19.0-23.1 us = 4.0-4.8 TB/s; the codes of a row
// lie in a third of a tile's lines, and other rows read the same lines again (counted: 37 MB read).
template <int DT, int D>
__global__ void __launch_bounds__(256)
gather_paged_q4_kernel(RotateAppend a, const char* __restrict__ pages, char* __restrict__ k, char* __restrict__ v) {
    constexpr int G = q4_groups(D), kEs = DT == SPARDA_F32 ? 4 : 2, kPer = D / 8;
    const int lane = threadIdx.x % kWave;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (t >= a.N) return;
    const PagedRow r = paged_row(a.pg, a.ps, a.positions, a.cu, a.n, a.N, t, a.status);
    if (!r.takes) return;
    const int key = static_cast<int>(r.row % 16);
    const char* tiles = pages + r.page * a.pg.p_st + r.row / 16 * (576 * G);
    for (int i = lane; i < a.Hkv * kPer; i += kWave) {
        const int h = i / kPer, dim = i % kPer * 8;
        float x[8], y[8];
        if (r.page >= 0) {
            const char* tile = tiles + h * a.pg.h_st;
            const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + q4_key_word<G>(key, dim));
            const float hk = *reinterpret_cast<const _Float16*>(tile + q4_scale_at<G>(0, key, dim / 32));
            const float hv = *reinterpret_cast<const _Float16*>(tile + q4_scale_at<G>(1, key, dim / 32));
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint32_t b = *reinterpret_cast<const uint8_t*>(tile + q4_value_byte<G>(key, dim + e));
                x[e] = hk * static_cast<float>(static_cast<int>(w >> (2 * e) & 15) * 2 - 15);
                x[e + 1] = hk * static_cast<float>(static_cast<int>(w >> (2 * e + 16) & 15) * 2 - 15);
                y[e] = hv * static_cast<float>(static_cast<int>(b & 15) * 2 - 15);
                y[e + 1] = hv * static_cast<float>(static_cast<int>(b >> 4) * 2 - 15);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e] = __builtin_nanf("");
        }
        const int64_t at = (t * a.new_st + h * a.new_sh + dim) * kEs;
        q4_store8<DT>(k + at, x);
        q4_store8<DT>(v + at, y);
    }
}

int launch_append_paged_q4(const RotateAppend& given, void* pages, int dtype, int64_t D, hipStream_t stream) {
    RotateAppend a = given;
    if (!grid_fits(cdiv(a.N, 4), 256)) return set_error(SPARDA_ERR_SHAPE, "append_paged_q4: grid too large");
    if (const int rc = status_word(&a.status)) return rc;
    const dim3 grid(static_cast<unsigned>(cdiv(a.N, 4)));
    const bool once = rows_past_cache(a, D, dtype);
#define SPARDA_AQ_O(DT_, D_, ROT_)                                                                                     \
    do {                                                                                                               \
        if (once) hipLaunchKernelGGL((append_paged_q4_kernel<DT_, D_, ROT_, true>), grid, dim3(256), 0, stream, a, static_cast<char*>(pages)); \
        else hipLaunchKernelGGL((append_paged_q4_kernel<DT_, D_, ROT_, false>), grid, dim3(256), 0, stream, a, static_cast<char*>(pages));     \
    } while (0)
#define SPARDA_AQ(DT_, D_)                        \
    do {                                          \
        if (a.cos) SPARDA_AQ_O(DT_, D_, true);    \
        else SPARDA_AQ_O(DT_, D_, false);         \
    } while (0)
#define SPARDA_AQ_D(DT_)                      \
    switch (D) {                              \
        case 16: SPARDA_AQ(DT_, 16); break;   \
        case 32: SPARDA_AQ(DT_, 32); break;   \
        case 64: SPARDA_AQ(DT_, 64); break;   \
        default: SPARDA_AQ(DT_, 128); break;  \
    }
    if (dtype == SPARDA_F32) SPARDA_AQ_D(SPARDA_F32)
    else SPARDA_AQ_D(SPARDA_BF16)
#undef SPARDA_AQ_D
#undef SPARDA_AQ
#undef SPARDA_AQ_O
    return check_hip(hipGetLastError(), "append_paged_q4_kernel");
}

int launch_gather_paged_q4(const RotateAppend& given, const void* pages, int dtype, int64_t D, void* k, void* v,
                           hipStream_t stream) {
    RotateAppend a = given;
    if (!grid_fits(cdiv(a.N, 4), 256)) return set_error(SPARDA_ERR_SHAPE, "gather_paged_q4: grid too large");
    if (const int rc = status_word(&a.status)) return rc;
    const dim3 grid(static_cast<unsigned>(cdiv(a.N, 4)));
#define SPARDA_GQ(DT_, D_)                                                                                            \
    hipLaunchKernelGGL((gather_paged_q4_kernel<DT_, D_>), grid, dim3(256), 0, stream, a, static_cast<const char*>(pages), \
                       static_cast<char*>(k), static_cast<char*>(v))
#define SPARDA_GQ_D(DT_)                      \
    switch (D) {                              \
        case 16: SPARDA_GQ(DT_, 16); break;   \
        case 32: SPARDA_GQ(DT_, 32); break;   \
        case 64: SPARDA_GQ(DT_, 64); break;   \
        default: SPARDA_GQ(DT_, 128); break;  \
    }
    if (dtype == SPARDA_F32) SPARDA_GQ_D(SPARDA_F32)
    else SPARDA_GQ_D(SPARDA_BF16)
#undef SPARDA_GQ_D
#undef SPARDA_GQ
    return check_hip(hipGetLastError(), "gather_paged_q4_kernel");
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// N words of codes; STREAM: read once, not to stay in the caches
template <int N, bool STREAM>
__device__ __forceinline__ void q4_load_words(const char* p, uint32_t (&w)[N]) {
    typedef uint32_t words __attribute__((ext_vector_type(N)));
    words x;
    if constexpr (STREAM) x = __builtin_nontemporal_load(reinterpret_cast<const words*>(p));
    else x = *reinterpret_cast<const words*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = x[i];
}
// four positions' numbers, [4][G]
template <int G>
__device__ __forceinline__ void q4_load_scales(const char* p, _Float16 (&h)[4][G]) {
    if constexpr (G == 1) {
        const auto x = __builtin_bit_cast(__attribute__((ext_vector_type(4))) _Float16, *reinterpret_cast<const uint2*>(p));
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i][0] = x[i];
    } else {
#pragma unroll
        for (int j = 0; j < G / 2; ++j) {
            const auto x = __builtin_bit_cast(f16x8, *reinterpret_cast<const uint4*>(p + 16 * j));
#pragma unroll
            for (int e = 0; e < 8; ++e) h[(j * 8 + e) / G][(j * 8 + e) % G] = x[e];
        }
    }
}

// Codes go to the matrix products as bf16 16.5 + c: a code at bits 3 .. 6 of the mantissa over a
// half below it. The middle level is then 24, a bf16 value, and is taken off by a product with the
// constant -24 (128 + c would need one shift less, and a middle of 135.5, which bf16 does not hold).
// The masks are held in registers, so that the and and the or of a word are one instruction (of
// two literals the compiler makes two).
struct Q4Masks {
    uint32_t bits, magic;
};
__device__ __forceinline__ Q4Masks q4_masks() {
    Q4Masks m{0x00780078u, 0x41844184u};
    asm("" : "+s"(m.bits));
    asm("" : "+v"(m.magic));
    return m;
}
// bits n .. n + 3 of both halves of a word
template <int N>
__device__ __forceinline__ uint32_t q4_pair(uint32_t w, const Q4Masks& m) {
    return ((N < 3 ? w << (3 - N) : w >> (N > 3 ? N - 3 : 0)) & m.bits) | m.magic;
}
// the eight codes of a key word: nibbles n and n + 4 are the halves of register n
__device__ __forceinline__ bf16x8 q4_key_operand(uint32_t w, const Q4Masks& m) {
    return __builtin_bit_cast(bf16x8, make_uint4(q4_pair<0>(w, m), q4_pair<4>(w, m), q4_pair<8>(w, m), q4_pair<12>(w, m)));
}
// nibble J of the eight positions of two tiles' words
template <int J>
__device__ __forceinline__ bf16x8 q4_value_operand(uint32_t w0, uint32_t w1, const Q4Masks& m) {
    return __builtin_bit_cast(bf16x8, make_uint4(q4_pair<4 * J>(w0, m), q4_pair<4 * J + 8>(w0, m), q4_pair<4 * J>(w1, m),
                                                 q4_pair<4 * J + 8>(w1, m)));
}

// x as a sum of TERMS bf16 values (1: rounded; 3: all 24 bits of it)
template <int TERMS>
__device__ __forceinline__ void q4_split(const float (&x)[8], bf16x8 (&out)[TERMS]) {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = x[e];
#pragma unroll
    for (int n = 0; n < TERMS; ++n) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = pack_bf16(rest[2 * e], rest[2 * e + 1]);
            if (n + 1 < TERMS) {
                rest[2 * e] -= __uint_as_float(w[e] << 16);
                rest[2 * e + 1] -= __uint_as_float(w[e] & 0xffff0000u);
            }
        }
        out[n] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    }
}

// a lane permutation without lanes outside (bound_ctrl, so that it is taken into the operation that uses it)
template <int CTRL>
__device__ __forceinline__ float q4_dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// x times lane E of the quad's h
template <int E>
__device__ __forceinline__ float q4_by_quad(float x, float h) {
    return x * q4_dpp<E * 0x55>(h);
}
// sums over the lanes 16 / G apart in a row of 16, in an order and with roundings (no fused multiply-add)
// that make them equal in all of those
template <int G>
__device__ __forceinline__ float q4_group_sum(float v) {
#pragma clang fp contract(off)
    if constexpr (G >= 2) v = v + q4_dpp<0x128>(v);   // row_ror:8
    if constexpr (G >= 4) v = v + q4_dpp<0x124>(v);   // row_ror:4
    return v;
}

// pages and tiles of the two tiles of a step
struct Q4Place {
    int id[2], tile[2];
};

// wavefronts of a SIMD
constexpr int q4_waves(int DT, int D, int NF, int NR) {
    return (D == 128 && NF > 0 ? 3 : 4) - (DT == SPARDA_F32 ? 1 : 0) - (NF + NR > 1 ? 1 : 0);
}

}  // namespace

// One workgroup of KW wavefronts per (16 NC columns, item). The columns are the (token, query
// head) pairs of a KV head, token-major; token t of T sees the positions below
// len - T + 1 + t. The numbers h stay outside of the products with the codes:
//     S^T[key, col] = 2 sum_g h_g[key] sum_{d in g} ((16.5 + c) - 24) q[d]
//     O^T[d, col]  += 2 sum_key ((16.5 + c) - 24) P_g[key, col],  P_g = exp2(S - m) h_g[key] in bf16
// so that the levels, odd multiples of h, enter without rounding. The rounding of P_g, half a step of 2^-8 as that
// of the weights over 16-bit pages, keeps the product on the bf16 matrix cores; fp32 calls take P_g and q in three
// bf16 terms each.
//
// A lane's keys of a step (positions 4 grp .. 4 grp + 3 of two tiles) are the same in S^T's rows and in
// the operand that P^T becomes, so P never leaves its lanes, and the order of the codes in memory is that
// of the operands: no LDS but for the join of the wavefronts.
//
// A tile whose columns fit 16 / G of its 16 (NR = 1; beside NF full ones) holds every column once for each of its G groups: column
// h + kCols g takes the scores of group g alone (Q's operand is zero elsewhere) and carries the weights of
// group g alone. The products of all groups then go into one accumulator, which starts at the
// middle's share of the column (a constant), h is one number a lane and key, and the groups' sums are added
// across lanes: 16 products a step of 32 keys instead of 32, and 210 vector instructions instead of 307 (D =
// 128). Unpacking is 128 of them.
//
// 32 sequences of up to 16384, 32/8 heads of 128 (401 MB): 74.7 us a call = 5.4 TB/s; without a repeated tile and
// STREAM 87.6, without STREAM 84.2. Loads alone took 74.5, arithmetic alone 72.9 before. 8 x 16384, 12/4 heads of 64 (29
// MB): 12.3 of 14.8 us a call, a chain of three steps' reads under load; 16 x 5 tokens at up to 8000, 32/8 of
// 128 (20 columns: a full tile and a repeated one): 32.6 of 36.5, vector issue; in two full tiles 35.5 of 41. 1 x
// 1000: 4.9 of 8, a launch and four dependent loads. Steps staged through LDS one or two ahead took 97 and 105 us where this took 95.
template <int DT, int D, int KW, int NF, int NR, bool STREAM>
__global__ void __launch_bounds__(KW* kWave, q4_waves(DT, D, NF, NR))
decode_paged_q4_kernel(PagedDecode a) {
    constexpr int G = q4_groups(D), kTerms = DT == SPARDA_F32 ? 3 : 1, kLogStep = 5, kStep = 1 << kLogStep, kEs = DT == SPARDA_F32 ? 4 : 2;
    constexpr int NC = NF + NR, kCols = 16 / G;              // tiles; columns of a repeated one
    static_assert(NR == 0 || (NR == 1 && G > 1), "one repeated tile, of several groups");
    constexpr bool REP = NR > 0;
    constexpr int kRep = REP ? NF : 0;                       // the repeated tile (tiles before it are full)
    extern __shared__ float lds[];
    const int lane = threadIdx.x % kWave;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
    const int c16 = lane % 16, grp = lane / 16;
    const int groups = a.Hkv * a.head_tiles;
    const int item = blockIdx.x / groups, gt = blockIdx.x % groups;
    const int g = gt / a.head_tiles, col0 = gt % a.head_tiles * (16 * NC);
    const int ncol = a.R * a.T - col0 < 16 * NC ? a.R * a.T - col0 : 16 * NC;   // columns of the workgroup (all, where one is repeated)
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

    bf16x8 middle;
#pragma unroll
    for (int e = 0; e < 8; ++e) middle[e] = static_cast<__bf16>(-24.0f);
    // this lane's columns of Q (a repeated tile's column h of group g in lane h + kCols g, in the product with that group's codes alone)
    const int mine = c16 / kCols;
    int lim[NC];                                             // positions a column sees
    bf16x8 qr[NC][G][kTerms];
    f32x4 start{0.f, 0.f, 0.f, 0.f};                         // repeated tile: -24 times the sum of the column's q in its group
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const bool repeated = REP && c == kRep;
        const int at = 16 * c + (repeated ? c16 % kCols : c16), col = col0 + (at < ncol ? at : ncol - 1), tok = col / a.R, head = g * a.R + col % a.R;
        lim[c] = len - a.T + 1 + tok;
        const char* q = static_cast<const char*>(a.q) + (b * a.q_sb + tok * a.q_st + head * a.q_sh) * kEs;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            float x[8];
            if (at < ncol && 32 * i + 8 * grp < D && (!repeated || mine == i)) {
                q4_load8<DT, false>(q + (32 * i + 8 * grp) * kEs, x);
                if (a.negate) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = -x[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = 0.0f;
            }
            q4_split<kTerms>(x, qr[c][i]);
            if (repeated) {
#pragma unroll
                for (int n = 0; n < kTerms; ++n) start = __builtin_amdgcn_mfma_f32_16x16x32_bf16(middle, qr[c][i][n], start, 0, 0, 0);
            }
        }
    }

    // The walk over the table: tile 2 u is `rem` tiles into page `page`. The page numbers of a step are
    // read a step before its codes, through the scalar cache.
    const auto* row = (const __attribute__((address_space(4))) int32_t*)(a.pg.table + b * a.pg.t_st);
    const char* kv = static_cast<const char*>(a.k) + g * a.pg.h_st;
    const int last_tile = (len - 1) / 16;
    const int o_keys = (c16 * 4 + grp) * 4 * G, o_values = 256 * G + lane * 4 * G;
    const int o_scales = 512 * G + grp * 8 * G, o_own = o_scales + (c16 % 4 * G + mine) * 2;
    int u = sh.part * sh.share + wave;
    int page = 2 * u / a.ps16, rem = 2 * u % a.ps16;
    const int adv_p = 2 * KW / a.ps16, adv_r = 2 * KW % a.ps16;
    auto places = [&](int v) __attribute__((always_inline)) {
        Q4Place at;
        const bool two = 2 * v + 1 <= last_tile, next = rem + 1 == a.ps16;   // (past the end: the first tile again, masked)
        at.tile[0] = rem, at.tile[1] = !two ? rem : next ? 0 : rem + 1;
        at.id[0] = row[page], at.id[1] = row[two && next ? page + 1 : page];
        rem += adv_r;
        page += adv_p;
        if (rem >= a.ps16) rem -= a.ps16, ++page;
        return at;
    };
    uint32_t xk[2][G], xv[2][G];                             // the codes of a step, as loaded
    _Float16 hk[2][4][G], hv[2][4][G];                       // full tiles: positions 4 grp .. 4 grp + 3
    _Float16 rk[2], rv[2];                                   // the repeated one: position 4 grp + c16 % 4, the lane's group
    const char* base[2];
    auto locate = [&](const Q4Place& at) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            int id = at.id[t];
            if (id < 0 || id >= a.pg.n_pages) bad = true, id = 0;
            base[t] = kv + id * a.pg.p_st + static_cast<int64_t>(at.tile[t]) * (576 * G);
        }
    };
    // (keys: position c16, quarter grp; values: four grp, pair c16)
    auto load_keys = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            q4_load_words<G, STREAM>(base[t] + o_keys, xk[t]);
            if constexpr (REP) rk[t] = *reinterpret_cast<const _Float16*>(base[t] + o_own);
            if constexpr (NF > 0) q4_load_scales<G>(base[t] + o_scales, hk[t]);
        }
    };
    auto load_values = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            q4_load_words<G, STREAM>(base[t] + o_values, xv[t]);
            if constexpr (REP) rv[t] = *reinterpret_cast<const _Float16*>(base[t] + o_own + 32 * G);
            if constexpr (NF > 0) q4_load_scales<G>(base[t] + o_scales + 32 * G, hv[t]);
        }
    };

    // m: the columns' references, in the scores' own units, l: this lane's part of their sums
    float m[NC], ref[NC], l[NC];
    const float slack = 16.0f / a.scale_log2;
    f32x4 o[NC][G][2], less{0.f, 0.f, 0.f, 0.f};             // less: repeated tile: -24 times the sum of the column's weights, not yet in o
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        m[c] = -__builtin_inff(), ref[c] = l[c] = 0.0f;
#pragma unroll
        for (int i = 0; i < G; ++i) o[c][i][0] = o[c][i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // The repeated tile's sums of (16.5 + c) P and of -24 P cancel where values average out, so they must not grow long
    // apart: 256 steps of a wavefront with flat scores left an fp32 output off by 5.8e-4, now 2.0e-6. fp32 calls join them
    // in every step (138.5 / 144 us for 32 x 16384, 32/8 heads of 128), the smaller terms first, which the sums hold
    // better before they are large. bf16 calls, off by 2.4e-3 by their weights' rounding, join them every 64 steps.
    constexpr bool kEach = DT == SPARDA_F32;
    constexpr int kFold = 64;
    int fold = kFold;
    const Q4Masks masks = q4_masks();
    f32x4 s[NC][2];
    auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 all = start;                               // the repeated tile's
#pragma unroll
            for (int c = 0; c < NF; ++c) s[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const bf16x8 ka = q4_key_operand(xk[t][i], masks);
                if constexpr (REP) {
#pragma unroll
                    for (int n = 0; n < kTerms; ++n) all = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, qr[kRep][i][n], all, 0, 0, 0);
                }
#pragma unroll
                for (int c = 0; c < NF; ++c) {
                    f32x4 y{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int n = 0; n < kTerms; ++n) y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(middle, qr[c][i][n], y, 0, 0, 0);
#pragma unroll
                    for (int n = 0; n < kTerms; ++n) y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, qr[c][i][n], y, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[c][t][e] = __builtin_fmaf(y[e], static_cast<float>(hk[t][e][i]), s[c][t][e]);
                }
                if constexpr (NF > 0) __builtin_amdgcn_sched_barrier(0);   // (operands of one group at a time: registers)
            }
            if constexpr (REP) {
                const float h = static_cast<float>(rk[t]);
                s[kRep][t][0] = q4_group_sum<G>(q4_by_quad<0>(all[0], h));
                s[kRep][t][1] = q4_group_sum<G>(q4_by_quad<1>(all[1], h));
                s[kRep][t][2] = q4_group_sum<G>(q4_by_quad<2>(all[2], h));
                s[kRep][t][3] = q4_group_sum<G>(q4_by_quad<3>(all[3], h));
            }
        }
    };
    auto attend = [&](auto masked, int v) __attribute__((always_inline)) {
        constexpr bool kMask = decltype(masked)::value;
        float p[NC][8];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int left = lim[c] - v * kStep - 4 * grp;   // this lane's keys 16 t + e below it are the column's
            float mx = -__builtin_inff();
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, !kMask || 16 * t + e < left ? s[c][t][e] : -__builtin_inff());
            // The reference follows the maximum only where a weight would pass 2^16: weights keep their
            // relative precision whatever they are measured against, and most steps rescale nothing.
            if (__ballot(!(mx <= m[c] + slack)) != 0) {      // (scale 0: -inf + inf, no order)
                const float top = fmaxf(m[c], pair32_max(pair16_max(mx)));
                const float to = top == -__builtin_inff() ? 0.0f : top * a.scale_log2;
                const float alpha = m[c] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ref[c] - to);
                m[c] = top, ref[c] = to;
                l[c] *= alpha;
#pragma unroll
                for (int i = 0; i < G; ++i) o[c][i][0] *= alpha, o[c][i][1] *= alpha;
                if (REP && c == kRep) less *= alpha;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[c][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][e / 4][e % 4], a.scale_log2, -ref[c]));
                if (kMask) p[c][e] = 16 * (e / 4) + e % 4 < left ? p[c][e] : 0.0f;
                l[c] += p[c][e];
            }
        }
        bf16x8 own[kTerms];                                  // the repeated tile's weights, of the lane's group
        if constexpr (REP) {
            const int left = lim[kRep] - v * kStep - 4 * grp;
            float ph[8];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const float h = static_cast<float>(rv[t]);
                ph[4 * t] = q4_by_quad<0>(p[kRep][4 * t], h);
                ph[4 * t + 1] = q4_by_quad<1>(p[kRep][4 * t + 1], h);
                ph[4 * t + 2] = q4_by_quad<2>(p[kRep][4 * t + 2], h);
                ph[4 * t + 3] = q4_by_quad<3>(p[kRep][4 * t + 3], h);
            }
            if constexpr (kMask) {
#pragma unroll
                for (int e = 0; e < 8; ++e) ph[e] = 16 * (e / 4) + e % 4 < left ? ph[e] : 0.0f;   // (a number behind the column's positions may be anything)
            }
            q4_split<kTerms>(ph, own);
            if (kEach) less = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = kTerms - 1; n >= 0; --n) less = __builtin_amdgcn_mfma_f32_16x16x32_bf16(middle, own[n], less, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const bf16x8 v0 = q4_value_operand<0>(xv[0][i], xv[1][i], masks), v1 = q4_value_operand<1>(xv[0][i], xv[1][i], masks);
            if constexpr (REP) {
#pragma unroll
                for (int n = kTerms - 1; n >= 0; --n) {
                    o[kRep][i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, own[n], o[kRep][i][0], 0, 0, 0);
                    o[kRep][i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, own[n], o[kRep][i][1], 0, 0, 0);
                }
                if constexpr (kEach) o[kRep][i][0] += less, o[kRep][i][1] += less;
            }
#pragma unroll
            for (int c = 0; c < NF; ++c) {
                const int left = lim[c] - v * kStep - 4 * grp;
                float ph[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    ph[e] = __builtin_fmaf(p[c][e], static_cast<float>(hv[e / 4][e % 4][i]), 0.0f);
                    if (kMask) ph[e] = 16 * (e / 4) + e % 4 < left ? ph[e] : 0.0f;   // (as above)
                }
                bf16x8 pb[kTerms];
                q4_split<kTerms>(ph, pb);
#pragma unroll
                for (int n = 0; n < kTerms; ++n) {
                    o[c][i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(middle, pb[n], o[c][i][0], 0, 0, 0);
                    o[c][i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(middle, pb[n], o[c][i][1], 0, 0, 0);
                    o[c][i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pb[n], o[c][i][0], 0, 0, 0);
                    o[c][i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pb[n], o[c][i][1], 0, 0, 0);
                }
            }
            if constexpr (NF > 0) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (REP && !kEach) {
            if (--fold == 0) {                               // (wave-uniform)
                fold = kFold;
#pragma unroll
                for (int i = 0; i < G; ++i) o[kRep][i][0] += less, o[kRep][i][1] += less;
                less = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    };
    if (u < s_end) {
        locate(places(u));
        load_keys();
        load_values();
        Q4Place at{};
        if (u + KW < s_end) at = places(u + KW);
        // The next step's keys go into the registers that the scores leave free, its values behind the
        // sums. `until`: wave-uniform
        auto walk = [&](auto masked, int until) __attribute__((always_inline)) {
            while (u < until) {
                const bool more = u + KW < s_end;
                scores();
                if (more) {
                    locate(at);
                    load_keys();
                    if (u + 2 * KW < s_end) at = places(u + 2 * KW);
                }
                attend(masked, u);
                if (more) load_values();
                u += KW;
            }
        };
        const int seen = len - a.T + 1;                      // positions that every token sees
        walk(std::false_type{}, seen < 0 ? 0 : min(s_end, seen / kStep));
        walk(std::true_type{}, s_end);
    }

    const bool any_bad = __ballot(bad) != 0;                  // wave-uniform
    // ---- the wavefronts' partials, joined in order: thread -> (column, dim), 16 columns at a time ----
    float* lo = lds;                                          // [KW][lds_heads][D + 4]
    float* lm = lo + KW * a.lds_heads * (D + 4);              // [KW][16][2]
    int* lbad = reinterpret_cast<int*>(lm + KW * 32);         // [KW]
    if (lane == 0) lbad[wave] = any_bad ? 1 : 0;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int nh = ncol - 16 * c < 16 ? ncol - 16 * c : 16;
        if (nh <= 0) break;                                   // workgroup-uniform
        if (c > 0) __syncthreads();                           // the last ones have been read
        l[c] = pair32_sum(pair16_sum(l[c]));
        const bool repeated = REP && c == kRep;
        const int cc16 = repeated ? c16 % kCols : c16;        // the lane's column
        if (cc16 < nh) {
#pragma unroll
            for (int i = 0; i < G; ++i) {
                if (repeated && mine != i) continue;          // (other groups' weights)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int d = 32 * i + 2 * (4 * grp + e) + j;
                        if (d < D) lo[(wave * a.lds_heads + cc16) * (D + 4) + d] = 2.0f * (repeated && !kEach ? o[c][i][j][e] + less[e] : o[c][i][j][e]);
                    }
            }
            if (grp == 0 && (!repeated || mine == 0)) {
                lm[(wave * 16 + c16) * 2] = m[c] == -__builtin_inff() ? m[c] : ref[c];   // (log2 units from here)
                lm[(wave * 16 + c16) * 2 + 1] = l[c];
            }
        }
        __syncthreads();
        int bads = 0;
#pragma unroll
        for (int w = 0; w < KW; ++w) bads |= lbad[w];
        if (c == 0 && bads != 0 && wave == 0 && lane == 0) atomicOr(a.status, static_cast<uint32_t>(SPARDA_STATUS_PAGE_RANGE));
        for (int e = wave * kWave + lane; e < nh * D; e += KW * kWave) {
            const int cc = e / D, d = e % D;
            float mw[KW], M = -__builtin_inff();
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                mw[w] = lm[(w * 16 + cc) * 2];
                M = fmaxf(M, mw[w]);
            }
            const float top = M == -__builtin_inff() ? 0.0f : M;
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const float wt = __builtin_amdgcn_exp2f(mw[w] - top);
                L = __builtin_fmaf(wt, lm[(w * 16 + cc) * 2 + 1], L);
                O = __builtin_fmaf(wt, lo[(w * a.lds_heads + cc) * (D + 4) + d], O);
            }
            if (bads) O = __builtin_nanf("");
            const int col = col0 + 16 * c + cc, t = col / a.R, h = t * a.heads + g * a.R + col % a.R;
            if (sh.parts == 1) {
                // (a token before the sequence's first position: zeros)
                store_elem<DT>(a.out, b * a.out_sb + static_cast<int64_t>(h) * D + d,
                               len - a.T + 1 + t <= 0 && !bads ? 0.0f : O / L);
            } else {
                const int64_t to = static_cast<int64_t>(item) * a.Hq + h;
                a.part_o[to * D + d] = O;
                if (d == 0) *reinterpret_cast<float2*>(a.part_ml + to * 2) = make_float2(M, L);
            }
        }
    }
}

namespace {

// How the work is cut, and what was measured on either side of each rule:
// - Two tiles of 16 columns share the unpacked codes where there are more than 16 columns and the products
//   are single: 16 x 5 tokens of 32/8 heads of 128 at 8000 (20 columns) 41 us, 47 with a tile a workgroup. In
//   fp32 the terms of two tiles do not fit the registers.
// - Columns that fit 16 / G of a tile stand in it G times, and so do those that are left of a full tile (one token of
//   32/8 heads of 128 88 / 84 us at 32 x 16384; five tokens 41 / 36.5 at 16 x 8000). More would take several such tiles, at 76
//   vector instructions a step each where a full tile takes 120.
// - A sequence is one item, with no join, up to 16 steps of 32 keys, or up to 64 where the sequences fill
//   half of the chip by themselves; otherwise there are as many items as workgroups run at a time (256 CUs
//   times the wavefronts that a SIMD holds), so that all shares are done in one round: one too many
//   costs a second. The target is below that by B / 2, since ceil adds half an item a sequence in the mean, and
//   by two standard deviations of that sum. Over 24 draws of 32 lengths up to 16384, 32/8 heads of 128: 79.9 us in
//   the mean and 89.7 at most, without the deviations 84.6 and 101.2, with B below 81.3 and 95.8; half as
//   many items 109.6 where all took 80.5, twice as many 85.0. 16 x 5 tokens: 43.9 and 47.4, 44.3 and 57.2.
// - A share is four steps at least, one for each wavefront. (A sequence of several items, the only kind that is joined,
//   therefore holds more than 128 positions: all of its tokens, 64 at most, see some.)
// - A call over more than the last-level cache holds (256 MB of codes at the tables' capacity) finds nothing there from the
//   last call and loads past it: 32 x 16384 84.2 / 74.4 us. Smaller ones may: 16 x 5 tokens at 8000 repeated over few
//   caches 40.9 / 44.2 with such loads, over twelve 49.4 / 48.2; 20 x 9000 32.0 / 33.2 and 36.7 / 33.5.
struct Q4Plan {
    int nf, nr;              // column tiles of a workgroup: full ones, one with its columns once for every group
    int64_t target, least;   // items aimed at, steps of the smallest item
    int64_t items, groups;   // items at most, workgroups an item
    bool few;                // a sequence has few items in the mean
    bool stream;             // the codes do not stay in the last-level cache from call to call
};
Q4Plan q4_plan(int64_t B, int64_t T, int64_t cap, int64_t Hq, int64_t Hkv, int64_t D, int dtype) {
    const int64_t cols = Hq / Hkv * T, steps = cdiv(cap, 32);
    Q4Plan p{dtype == SPARDA_BF16 && cols > 16 ? 2 : 1, 0, 1, 4, 0, 0, false, false};
    const int64_t few = D >= 64 ? 16 / (D / 32) : 0;   // columns of a repeated tile
    if (cols <= few) p.nf = 0, p.nr = 1;
    else if (dtype == SPARDA_BF16 && cols > 16 && cols <= 16 + few) p.nf = 1, p.nr = 1;
    p.groups = Hkv * cdiv(cols, 16 * (p.nf + p.nr));
    if (steps <= 16 || (steps <= 64 && B * p.groups >= 128)) {
        p.least = steps;
    } else {
        // (items are target + B at most, target + B / 2 in the mean, sqrt(B / 12) to either side)
        const int64_t slots = 256 * q4_waves(dtype, static_cast<int>(D), p.nf, p.nr);
        int64_t margin = 0;                          // ceil(0.6 sqrt(B))
        while (margin * margin * 25 < B * 9) ++margin;
        p.target = slots / p.groups - B / 2 - margin;
    }
    if (p.target < 1) p.target = 1;
    p.items = p.target + B;
    const int64_t most = B * cdiv(steps, p.least);   // every share the smallest
    if (p.items > most) p.items = most;
    p.few = p.items <= 16 * B;
    p.stream = B * cap * Hkv * q4_groups(static_cast<int>(D)) * 36 > (256ll << 20);
    return p;
}

}  // namespace

size_t decode_paged_q4_workspace_bytes(int64_t B, int64_t T, int64_t cap, int64_t Hq, int64_t Hkv, int64_t D, int dtype) {
    const Q4Plan p = q4_plan(B, T, cap, Hq, Hkv, D, dtype);
    return p.items <= B ? 0 : static_cast<size_t>(p.items * T * Hq * (D + 2)) * sizeof(float);
}

int launch_decode_paged_q4(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, const void* pages,
                           int64_t n_pages, int64_t ps, int64_t p_st, int64_t h_st, const int32_t* table, int64_t t_st,
                           int64_t width, const int32_t* len, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                           float scale, void* out, int64_t out_sb, void* workspace, hipStream_t stream) {
    PagedDecode a{};
    const int64_t cap = width * ps, R = Hq / Hkv;
    const Q4Plan p = q4_plan(B, T, cap, Hq, Hkv, D, dtype);
    if (!grid_fits(p.items * p.groups, 4 * kWave)) return set_error(SPARDA_ERR_SHAPE, "decode_paged_q4: grid too large");
    if (const int rc = status_word(&a.status)) return rc;
    a.q = q, a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh, a.k = pages;
    a.pg = Pages{p_st, 0, h_st, table, t_st, static_cast<int>(width), static_cast<int>(n_pages)};
    a.T = static_cast<int>(T), a.heads = static_cast<int>(Hq);
    a.ps16 = static_cast<int>(ps / 16), a.len = len, a.B = static_cast<int>(B), a.cap = static_cast<int>(cap);
    a.Hq = static_cast<int>(T * Hq), a.Hkv = static_cast<int>(Hkv), a.R = static_cast<int>(R);
    a.head_tiles = static_cast<int>(cdiv(R * T, 16 * (p.nf + p.nr)));
    a.target = static_cast<int>(p.target), a.least = static_cast<int>(p.least);
    a.whole = p.items <= B;
    a.lds_heads = static_cast<int>(R * T < 16 ? R * T : 16);
    a.negate = scale < 0.0f;
    a.scale_log2 = 2.0f * fabsf(scale) * kPgLog2e, a.out = out, a.out_sb = out_sb;   // (h (2 c - 15) = 2 h (c - 7.5))
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = workspace ? a.part_o + p.items * a.Hq * D : nullptr;
    const dim3 grid(static_cast<unsigned>(p.items * p.groups));
#define SPARDA_DQ_S(DT_, D_, NF_, NR_, S_)                                                        \
    hipLaunchKernelGGL((decode_paged_q4_kernel<DT_, D_, 4, NF_, NR_, S_>), grid, dim3(4 * kWave), \
                       4 * (a.lds_heads * ((D_) + 4) + 33) * sizeof(float), stream, a)
#define SPARDA_DQ_C(DT_, D_, NF_, NR_)                                                            \
    do {                                                                                          \
        if (p.stream) SPARDA_DQ_S(DT_, D_, NF_, NR_, true);                                       \
        else SPARDA_DQ_S(DT_, D_, NF_, NR_, false);                                               \
    } while (0)
#define SPARDA_DQ(DT_, D_)                                                                        \
    do {                                                                                          \
        if constexpr (D_ >= 64) {                                                                 \
            if (p.nr > 0 && p.nf == 0) {                                                          \
                SPARDA_DQ_C(DT_, D_, 0, 1);                                                       \
                break;                                                                            \
            }                                                                                     \
        }                                                                                         \
        if constexpr (D_ >= 64 && DT_ == SPARDA_BF16) {                                           \
            if (p.nr > 0) {                                                                       \
                SPARDA_DQ_C(DT_, D_, 1, 1);                                                       \
                break;                                                                            \
            }                                                                                     \
        }                                                                                         \
        if constexpr (DT_ == SPARDA_BF16) {                                                       \
            if (p.nf == 2) SPARDA_DQ_C(DT_, D_, 2, 0);                                            \
            else SPARDA_DQ_C(DT_, D_, 1, 0);                                                      \
        } else {                                                                                  \
            SPARDA_DQ_C(DT_, D_, 1, 0);                                                           \
        }                                                                                         \
    } while (0)
#define SPARDA_DQ_D(DT_)                      \
    switch (D) {                              \
        case 16: SPARDA_DQ(DT_, 16); break;   \
        case 32: SPARDA_DQ(DT_, 32); break;   \
        case 64: SPARDA_DQ(DT_, 64); break;   \
        default: SPARDA_DQ(DT_, 128); break;  \
    }
    if (dtype == SPARDA_F32) SPARDA_DQ_D(SPARDA_F32)
    else SPARDA_DQ_D(SPARDA_BF16)
#undef SPARDA_DQ_D
#undef SPARDA_DQ
#undef SPARDA_DQ_C
#undef SPARDA_DQ_S
    if (p.items > B) launch_paged_join(a, D, dtype, 5, p.few, stream);
    return check_hip(hipGetLastError(), "decode_paged_q4_kernel");
}

}  // namespace sparda
