// The rotation of queries and keys by their positions, as the writes into pages
// apply it (paged_rotate.hip, paged_q4.hip): pairs (i, i + D/2),
//     y[i] = x[i] cos - x[i + D/2] sin,  y[i + D/2] = x[i + D/2] cos + x[i] sin,
// products, sum and difference each rounded to fp32 (no fused multiply-add, so that the
// result is that of the same formula in fp32 torch operations, and the 4-bit codes
// made from it are the same), and once to the rows' type.
#pragma once

#include "common.h"
#include "paged.h"

namespace sparda {

// New rows and their places; strides in elements.
struct RotateAppend {
    Pages pg;
    int ps;
    const int32_t *positions, *cu;
    int n;
    int64_t N;
    const void* q;                 // [N, Hq, D]; Hq 0: none
    int64_t q_st, q_sh;
    const void *k_new, *v_new;     // [N, Hkv, D]
    int64_t new_st, new_sh;
    const float *cos, *sin;        // [rows, D/2]
    int64_t cs_st, rows;
    int Hq, Hkv;
    void* q_out;
    int64_t qo_st, qo_sh;
    uint32_t* status;
};

// 16 bytes of a new row. ONCE: loaded past the caches, which nothing reads it from again. Calls that read and
// write more than the last-level cache holds (256 MB) do so: 16000 rows of 32/8 heads of 128, cold, 76.5 / 63.3 us for
// the kernel, just written by another one 70.4 / 66.3; in a row of such calls, where what earlier ones wrote still
// goes to memory, no difference. Smaller ones find their rows in the caches, where the projection has just put
// them: 4096 rows 32.3 / 33.6, 1501 of 12/4 heads of 64 in fp32 5.5 / 6.1. (What is written here is read next and stays in
// the caches: stores past them make a write of 65 MB 3 us shorter and its reader 11 longer.)
template <bool ONCE>
__device__ __forceinline__ uint4 load_row(const char* p) {
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    if constexpr (ONCE) return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const words*>(p)));
    else return *reinterpret_cast<const uint4*>(p);
}
// whether a call does: queries and new rows, each read and (at most) written once
inline bool rows_past_cache(const RotateAppend& a, int64_t D, int dtype) {
    return 2 * a.N * (a.Hq + 2 * static_cast<int64_t>(a.Hkv)) * D * (dtype == SPARDA_F32 ? 4 : 2) > (256ll << 20);
}

// N angles of position pos from dim `at` on; NaN behind the tables (whose first row is loaded then: with the
// loads on one way of a branch the compiler kept a part of them in scratch memory)
template <int N>
__device__ __forceinline__ void load_angles(const RotateAppend& a, int64_t pos, int at, bool off_table, float (&c)[N], float (&s)[N]) {
    const int64_t from = off_table ? 0 : pos * a.cs_st;
#pragma unroll
    for (int e = 0; e < N; e += 4) {
        const float4 x = *reinterpret_cast<const float4*>(a.cos + from + at + e);
        const float4 y = *reinterpret_cast<const float4*>(a.sin + from + at + e);
        c[e] = x.x, c[e + 1] = x.y, c[e + 2] = x.z, c[e + 3] = x.w;
        s[e] = y.x, s[e + 1] = y.y, s[e + 2] = y.z, s[e + 3] = y.w;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        c[e] = off_table ? __builtin_nanf("") : c[e];
        s[e] = off_table ? __builtin_nanf("") : s[e];
    }
}

__device__ __forceinline__ void turn(float& x, float& y, float c, float s) {
#pragma clang fp contract(off)
    const float xc = x * c, ys = y * s, yc = y * c, xs = x * s;
    x = xc - ys;
    y = yc + xs;
}

// two fp32 values as bf16, rounded to the nearest even
__device__ __forceinline__ uint32_t pack_bf16(float x, float y) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    bf16x2 v;
    v[0] = static_cast<__bf16>(x), v[1] = static_cast<__bf16>(y);
    return __builtin_bit_cast(uint32_t, v);
}

// 16 bytes of a row's first half and the 16 that they are paired with
template <int DT, int N>
__device__ __forceinline__ void turn_pieces(uint4& x, uint4& y, const float (&c)[N], const float (&s)[N]) {
    uint32_t a[4] = {x.x, x.y, x.z, x.w}, b[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if constexpr (DT == SPARDA_F32) {
            float u = __uint_as_float(a[w]), v = __uint_as_float(b[w]);
            turn(u, v, c[w], s[w]);
            a[w] = __float_as_uint(u), b[w] = __float_as_uint(v);
        } else {
            float u0 = __uint_as_float(a[w] << 16), u1 = __uint_as_float(a[w] & 0xffff0000u);
            float v0 = __uint_as_float(b[w] << 16), v1 = __uint_as_float(b[w] & 0xffff0000u);
            turn(u0, v0, c[2 * w], s[2 * w]);
            turn(u1, v1, c[2 * w + 1], s[2 * w + 1]);
            a[w] = pack_bf16(u0, u1), b[w] = pack_bf16(v0, v1);
        }
    }
    x = make_uint4(a[0], a[1], a[2], a[3]);
    y = make_uint4(b[0], b[1], b[2], b[3]);
}

// Rotates `heads` heads of row t: head h from from(h) to to(h), both at its first element. A lane takes 16
// bytes and the 16 that they are paired with, of four heads at a time; D/2 holds 1 to 16
// such pieces, so that a lane's piece of the angles is the same for every head and is loaded once.
template <int DT, int D, bool ONCE, class From, class To>
__device__ __forceinline__ void turn_heads(const RotateAppend& a, int64_t pos, bool off_table, int heads, From from, To to) {
    constexpr int kEs = DT == SPARDA_F32 ? 4 : 2, kVe = 16 / kEs, kPer = D / 2 / kVe, kAtOnce = kWave / kPer, kBatch = 4;
    const int lane = threadIdx.x % kWave, c = lane % kPer;
    float cs[kVe], sn[kVe];
    load_angles<kVe>(a, pos, c * kVe, off_table, cs, sn);
    for (int h0 = lane / kPer; h0 < heads; h0 += kBatch * kAtOnce) {
        uint4 x[kBatch], y[kBatch];
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int h = h0 + e * kAtOnce;
            if (h < heads) {
                const char* p = from(h) + c * 16;
                x[e] = load_row<ONCE>(p);
                y[e] = load_row<ONCE>(p + D / 2 * kEs);
            }
        }
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
            const int h = h0 + e * kAtOnce;
            if (h < heads) {
                char* p = to(h) + c * 16;
                turn_pieces<DT>(x[e], y[e], cs, sn);
                *reinterpret_cast<uint4*>(p) = x[e];
                *reinterpret_cast<uint4*>(p + D / 2 * kEs) = y[e];
            }
        }
    }
}

}  // namespace sparda
