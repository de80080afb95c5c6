// C entries of the serving operators beyond 16-bit pages: the rotated write, the
// 4-bit pages, drafted tokens. Every argument is checked here, before any HIP call.
#include "common.h"
#include "kernels.h"
#include "paged.h"
#include "rotate.h"

using namespace sparda;

namespace sparda {

int launch_rotate_append_paged(const RotateAppend& a, void* k, void* v, int dtype, int64_t D, hipStream_t stream);
int launch_append_paged_q4(const RotateAppend& a, void* pages, int dtype, int64_t D, hipStream_t stream);
int launch_gather_paged_q4(const RotateAppend& a, const void* pages, int dtype, int64_t D, void* k, void* v, hipStream_t stream);
size_t decode_paged_q4_workspace_bytes(int64_t B, int64_t T, int64_t cap, int64_t Hq, int64_t Hkv, int64_t D, int dtype);
int launch_decode_paged_q4(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype, const void* pages,
                           int64_t n_pages, int64_t ps, int64_t p_st, int64_t h_st, const int32_t* table, int64_t t_st,
                           int64_t width, const int32_t* len, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                           float scale, void* out, int64_t out_sb, void* workspace, hipStream_t stream);
size_t verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V, int dtype);
int launch_verify_drafts(const void* logits, int dtype, int64_t l_sb, int64_t l_st, const int32_t* drafts, int64_t d_sb,
                         const float* uniform, int64_t u_sb, const float* probs, int64_t p_sb, int64_t p_st,
                         const int32_t* counts, const float* temperature, float all_temperature, int64_t B, int64_t K,
                         int64_t V, int32_t* tokens, int32_t* accepted, void* workspace, hipStream_t stream);

}  // namespace sparda

namespace {

bool dtype_ok(int dt) { return dt == SPARDA_F32 || dt == SPARDA_BF16; }
bool head_dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int64_t piece(int dtype) { return dtype == SPARDA_F32 ? 4 : 8; }   // elements of 16 bytes

// sizes of pages and table, common to all of them
int check_cache(const char* who, int64_t n_pages, int64_t page_size, int64_t t_st, int64_t width, int64_t Hkv, int64_t D) {
    SPARDA_REQUIRE(n_pages > 0 && width > 0 && Hkv > 0, SPARDA_ERR_SHAPE, "%s: sizes must be positive", who);
    SPARDA_REQUIRE(page_size >= 16 && page_size % 16 == 0, SPARDA_ERR_SHAPE,
                   "%s: page size %lld is no positive multiple of 16", who, (long long)page_size);
    SPARDA_REQUIRE(head_dim_ok(D), SPARDA_ERR_SHAPE, "%s: head dim %lld not in {16,32,64,128}", who, (long long)D);
    SPARDA_REQUIRE(n_pages < (1ll << 31) && Hkv <= 65535 && page_size < (1ll << 31) && width <= 0x7fffffff / page_size,
                   SPARDA_ERR_SHAPE, "%s: 2^31 pages, or 2^31 positions in a row of the table", who);
    SPARDA_REQUIRE(t_st >= 0, SPARDA_ERR_STRIDE, "%s: negative stride", who);
    return 0;
}
int check_q4(const char* who, const void* pages, int64_t n_pages, int64_t page_size, int64_t p_st, int64_t h_st, int64_t t_st,
             int64_t width, int64_t Hkv, int64_t D) {
    if (const int rc = check_cache(who, n_pages, page_size, t_st, width, Hkv, D)) return rc;
    SPARDA_REQUIRE(p_st >= 0 && h_st >= 0, SPARDA_ERR_STRIDE, "%s: negative stride", who);
    SPARDA_REQUIRE(aligned16(pages) && p_st % 16 == 0 && h_st % 16 == 0, SPARDA_ERR_STRIDE,
                   "%s: the pages' heads must be 16-byte aligned", who);
    return 0;
}
// the new rows of a write or the rows of a read, and their sequences
int check_rows(const char* who, const void* a, const void* b, int dtype, const int32_t* cu, int64_t n_seqs, int64_t N,
               int64_t st, int64_t sh) {
    SPARDA_REQUIRE(dtype_ok(dtype), SPARDA_ERR_DTYPE, "%s: dtype %d unsupported", who, dtype);
    SPARDA_REQUIRE(n_seqs > 0 && N > 0 && N < (1ll << 31) && (n_seqs <= (1ll << 30) || !cu), SPARDA_ERR_SHAPE,
                   "%s: bad numbers of sequences or rows", who);
    SPARDA_REQUIRE(cu || N == n_seqs, SPARDA_ERR_SHAPE,
                   "%s: without offsets every sequence takes one row (%lld rows, %lld sequences)", who, (long long)N,
                   (long long)n_seqs);
    SPARDA_REQUIRE(aligned16(a) && aligned16(b) && st % piece(dtype) == 0 && sh % piece(dtype) == 0, SPARDA_ERR_STRIDE,
                   "%s: the rows must be 16-byte aligned", who);
    return 0;
}
// rows [N, H, D] that a kernel writes must not overlap: tokens outside heads, or heads outside tokens
bool rows_apart(int64_t N, int64_t H, int64_t D, int64_t st, int64_t sh) {
    if (st < 0 || sh < 0) return false;
    const bool heads = H == 1 || sh >= D, tokens = N == 1 || st >= D;
    return heads && tokens && (N == 1 || H == 1 || st >= (H - 1) * sh + D || sh >= (N - 1) * st + D);
}
int check_rotation(const char* who, const void* q, int64_t q_st, int64_t q_sh, int64_t Hq, int dtype, int64_t N, int64_t D,
                   const float* cos, const float* sin, int64_t cs_st, int64_t rows, const void* q_out, int64_t qo_st,
                   int64_t qo_sh) {
    SPARDA_REQUIRE(cos && sin, SPARDA_ERR_NULL, "%s: null pointer", who);
    SPARDA_REQUIRE(Hq >= 0 && Hq <= 65535, SPARDA_ERR_SHAPE, "%s: query heads must be in [0, 65535]", who);
    SPARDA_REQUIRE(Hq == 0 || (q && q_out), SPARDA_ERR_NULL, "%s: null pointer", who);
    SPARDA_REQUIRE(rows > 0, SPARDA_ERR_SHAPE, "%s: empty tables of angles", who);
    SPARDA_REQUIRE(aligned16(cos) && aligned16(sin) && cs_st % 4 == 0 && cs_st >= 0, SPARDA_ERR_STRIDE,
                   "%s: rows of the angles must be 16-byte aligned", who);
    if (Hq > 0) {
        const int64_t ve = piece(dtype);
        SPARDA_REQUIRE(aligned16(q) && aligned16(q_out) && q_st % ve == 0 && q_sh % ve == 0 && qo_st % ve == 0 && qo_sh % ve == 0,
                       SPARDA_ERR_STRIDE, "%s: the rows must be 16-byte aligned", who);
        SPARDA_REQUIRE(rows_apart(N, Hq, D, qo_st, qo_sh), SPARDA_ERR_STRIDE, "%s: output rows overlap", who);
    }
    return 0;
}

}  // namespace

SPARDA_API int sparda_rotate_append_paged(void* k_pages, void* v_pages, int dtype, int64_t n_pages, int64_t page_size,
                                          int64_t p_st, int64_t s_st, int64_t h_st, const int32_t* page_table,
                                          int64_t t_st, int64_t width, const int32_t* positions,
                                          const int32_t* cu_seqlens, int64_t n_seqs, const void* q, int64_t q_st,
                                          int64_t q_sh, int64_t Hq, const void* k_new, const void* v_new, int64_t N,
                                          int64_t new_st, int64_t new_sh, int64_t Hkv, int64_t D, const float* cos,
                                          const float* sin, int64_t cs_st, int64_t rows, void* q_out, int64_t qo_st,
                                          int64_t qo_sh, void* stream) {
    const char* who = "rotate_append_paged";
    SPARDA_REQUIRE(k_pages && v_pages && page_table && positions && k_new && v_new, SPARDA_ERR_NULL, "%s: null pointer", who);
    if (const int rc = check_rows(who, k_new, v_new, dtype, cu_seqlens, n_seqs, N, new_st, new_sh)) return rc;
    if (const int rc = check_cache(who, n_pages, page_size, t_st, width, Hkv, D)) return rc;
    const int64_t ve = piece(dtype);
    SPARDA_REQUIRE(p_st >= 0 && s_st >= 0 && h_st >= 0, SPARDA_ERR_STRIDE, "%s: negative stride", who);
    SPARDA_REQUIRE(aligned16(k_pages) && aligned16(v_pages) && p_st % ve == 0 && s_st % ve == 0 && h_st % ve == 0,
                   SPARDA_ERR_STRIDE, "%s: the rows of the pages must be 16-byte aligned", who);
    if (const int rc = check_rotation(who, q, q_st, q_sh, Hq, dtype, N, D, cos, sin, cs_st, rows, q_out, qo_st, qo_sh)) return rc;
    RotateAppend a{};
    a.pg = Pages{p_st, s_st, h_st, page_table, t_st, static_cast<int>(width), static_cast<int>(n_pages)};
    a.ps = static_cast<int>(page_size), a.positions = positions, a.cu = cu_seqlens, a.n = static_cast<int>(n_seqs), a.N = N;
    a.q = q, a.q_st = q_st, a.q_sh = q_sh, a.k_new = k_new, a.v_new = v_new, a.new_st = new_st, a.new_sh = new_sh;
    a.cos = cos, a.sin = sin, a.cs_st = cs_st, a.rows = rows, a.Hq = static_cast<int>(Hq), a.Hkv = static_cast<int>(Hkv);
    a.q_out = q_out, a.qo_st = qo_st, a.qo_sh = qo_sh;
    return launch_rotate_append_paged(a, k_pages, v_pages, dtype, D, static_cast<hipStream_t>(stream));
}

SPARDA_API int sparda_append_paged_q4(void* pages, int64_t n_pages, int64_t page_size, int64_t p_st, int64_t h_st,
                                      const int32_t* page_table, int64_t t_st, int64_t width, const int32_t* positions,
                                      const int32_t* cu_seqlens, int64_t n_seqs, const void* q, int64_t q_st,
                                      int64_t q_sh, int64_t Hq, const void* k_new, const void* v_new, int dtype,
                                      int64_t N, int64_t new_st, int64_t new_sh, int64_t Hkv, int64_t D,
                                      const float* cos, const float* sin, int64_t cs_st, int64_t rows, void* q_out,
                                      int64_t qo_st, int64_t qo_sh, void* stream) {
    const char* who = "append_paged_q4";
    SPARDA_REQUIRE(pages && page_table && positions && k_new && v_new, SPARDA_ERR_NULL, "%s: null pointer", who);
    if (const int rc = check_rows(who, k_new, v_new, dtype, cu_seqlens, n_seqs, N, new_st, new_sh)) return rc;
    if (const int rc = check_q4(who, pages, n_pages, page_size, p_st, h_st, t_st, width, Hkv, D)) return rc;
    if (cos || sin) {
        if (const int rc = check_rotation(who, q, q_st, q_sh, Hq, dtype, N, D, cos, sin, cs_st, rows, q_out, qo_st, qo_sh)) return rc;
    } else {
        SPARDA_REQUIRE(Hq == 0, SPARDA_ERR_NULL, "%s: queries are rotated: they need the angles", who);
    }
    RotateAppend a{};
    a.pg = Pages{p_st, 0, h_st, page_table, t_st, static_cast<int>(width), static_cast<int>(n_pages)};
    a.ps = static_cast<int>(page_size), a.positions = positions, a.cu = cu_seqlens, a.n = static_cast<int>(n_seqs), a.N = N;
    a.q = q, a.q_st = q_st, a.q_sh = q_sh, a.k_new = k_new, a.v_new = v_new, a.new_st = new_st, a.new_sh = new_sh;
    a.cos = cos, a.sin = sin, a.cs_st = cs_st, a.rows = rows, a.Hq = static_cast<int>(Hq), a.Hkv = static_cast<int>(Hkv);
    a.q_out = q_out, a.qo_st = qo_st, a.qo_sh = qo_sh;
    return launch_append_paged_q4(a, pages, dtype, D, static_cast<hipStream_t>(stream));
}

SPARDA_API int sparda_gather_paged_q4(const void* pages, int64_t n_pages, int64_t page_size, int64_t p_st, int64_t h_st,
                                      const int32_t* page_table, int64_t t_st, int64_t width, const int32_t* positions,
                                      const int32_t* cu_seqlens, int64_t n_seqs, void* k, void* v, int dtype, int64_t N,
                                      int64_t st, int64_t sh, int64_t Hkv, int64_t D, void* stream) {
    const char* who = "gather_paged_q4";
    SPARDA_REQUIRE(pages && page_table && positions && k && v, SPARDA_ERR_NULL, "%s: null pointer", who);
    if (const int rc = check_rows(who, k, v, dtype, cu_seqlens, n_seqs, N, st, sh)) return rc;
    if (const int rc = check_q4(who, pages, n_pages, page_size, p_st, h_st, t_st, width, Hkv, D)) return rc;
    SPARDA_REQUIRE(rows_apart(N, Hkv, D, st, sh), SPARDA_ERR_STRIDE, "%s: output rows overlap", who);
    RotateAppend a{};
    a.pg = Pages{p_st, 0, h_st, page_table, t_st, static_cast<int>(width), static_cast<int>(n_pages)};
    a.ps = static_cast<int>(page_size), a.positions = positions, a.cu = cu_seqlens, a.n = static_cast<int>(n_seqs), a.N = N;
    a.new_st = st, a.new_sh = sh, a.Hkv = static_cast<int>(Hkv);
    return launch_gather_paged_q4(a, pages, dtype, D, k, v, static_cast<hipStream_t>(stream));
}

SPARDA_API size_t sparda_decode_paged_q4_workspace_bytes(int64_t B, int64_t T, int64_t width, int64_t page_size,
                                                         int64_t Hq, int64_t Hkv, int64_t D, int dtype) {
    if (B <= 0 || T <= 0 || !dtype_ok(dtype) || width <= 0 || page_size <= 0 || Hkv <= 0 || Hq < Hkv || D <= 0) return 0;
    return decode_paged_q4_workspace_bytes(B, T, width * page_size, Hq, Hkv, D, dtype);
}

SPARDA_API int sparda_decode_paged_q4(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, int dtype,
                                      const void* pages, int64_t n_pages, int64_t page_size, int64_t p_st, int64_t h_st,
                                      const int32_t* page_table, int64_t t_st, int64_t width, const int32_t* lengths,
                                      int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, float scale, void* out,
                                      int64_t out_sb, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "decode_paged_q4";
    SPARDA_REQUIRE(q && pages && page_table && lengths && out, SPARDA_ERR_NULL, "%s: null pointer", who);
    SPARDA_REQUIRE(dtype_ok(dtype), SPARDA_ERR_DTYPE, "%s: dtype %d unsupported", who, dtype);
    if (const int rc = check_q4(who, pages, n_pages, page_size, p_st, h_st, t_st, width, Hkv, D)) return rc;
    SPARDA_REQUIRE(T >= 1 && T <= 64, SPARDA_ERR_SHAPE, "%s: tokens of a sequence must be in [1, 64]", who);
    SPARDA_REQUIRE(B > 0 && B <= 65535 && Hq > 0 && T * Hq <= 65535, SPARDA_ERR_SHAPE,
                   "%s: sequences, and query heads times tokens, must be in [1, 65535]", who);
    SPARDA_REQUIRE(Hq % Hkv == 0, SPARDA_ERR_SHAPE, "%s: Hq must be a multiple of Hkv", who);
    // (the kernels add steps of the whole batch and shares of it, and positions and a step, in 32 bits)
    SPARDA_REQUIRE(width * page_size <= (1ll << 31) - 64 && B * cdiv(width * page_size, 16) < (1ll << 30), SPARDA_ERR_SHAPE,
                   "%s: too many positions", who);
    const int64_t ve = piece(dtype);
    SPARDA_REQUIRE(aligned16(q) && q_sb % ve == 0 && q_st % ve == 0 && q_sh % ve == 0, SPARDA_ERR_STRIDE,
                   "%s: the rows of q must be 16-byte aligned", who);
    SPARDA_REQUIRE(B == 1 || out_sb >= T * Hq * D, SPARDA_ERR_STRIDE, "%s: output rows overlap", who);
    const size_t need = decode_paged_q4_workspace_bytes(B, T, width * page_size, Hq, Hkv, D, dtype);
    SPARDA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)), SPARDA_ERR_WORKSPACE,
                   "%s: workspace of %zu bytes needed, 16-byte aligned", who, need);
    return launch_decode_paged_q4(q, q_sb, q_st, q_sh, dtype, pages, n_pages, page_size, p_st, h_st, page_table, t_st, width,
                                  lengths, B, T, Hq, Hkv, D, scale, out, out_sb, need ? workspace : nullptr,
                                  static_cast<hipStream_t>(stream));
}

namespace {
bool verify_sizes_ok(int64_t B, int64_t K, int64_t V) {
    return B > 0 && K >= 0 && K <= 64 && B <= 65535 / (K + 1) && V > 0 && V <= (1ll << 20) - 8;
}
}  // namespace

SPARDA_API size_t sparda_verify_drafts_workspace_bytes(int64_t B, int64_t K, int64_t V, int dtype) {
    return verify_sizes_ok(B, K, V) && dtype_ok(dtype) ? verify_drafts_workspace_bytes(B, K, V, dtype) : 0;
}

SPARDA_API int sparda_verify_drafts(const void* logits, int dtype, int64_t l_sb, int64_t l_st, const int32_t* drafts,
                                    int64_t d_sb, const float* uniform, int64_t u_sb, const float* draft_probs,
                                    int64_t p_sb, int64_t p_st, const int32_t* n_drafts, const float* temperatures,
                                    float temperature, int64_t B, int64_t K, int64_t V, int32_t* tokens,
                                    int32_t* n_accepted, void* workspace, size_t workspace_bytes, void* stream) {
    const char* who = "verify_drafts";
    SPARDA_REQUIRE(logits && uniform && tokens && n_accepted && (drafts || K == 0), SPARDA_ERR_NULL, "%s: null pointer", who);
    SPARDA_REQUIRE(dtype_ok(dtype), SPARDA_ERR_DTYPE, "%s: dtype %d unsupported", who, dtype);
    SPARDA_REQUIRE(verify_sizes_ok(B, K, V), SPARDA_ERR_SHAPE,
                   "%s: %lld sequences of %lld drafts of a vocabulary of %lld: at most 64 drafts, 65535 rows, 2^20 - 8 tokens", who,
                   (long long)B, (long long)K, (long long)V);
    SPARDA_REQUIRE(temperatures || (temperature >= 0.0f && temperature <= 3.4e38f), SPARDA_ERR_SHAPE,
                   "%s: the temperature must be finite and not negative", who);
    const uintptr_t es = dtype == SPARDA_F32 ? 4 : 2;
    SPARDA_REQUIRE(reinterpret_cast<uintptr_t>(logits) % es == 0 && l_sb >= 0 && l_st >= 0 && d_sb >= 0 && u_sb >= 0 &&
                       p_sb >= 0 && p_st >= 0, SPARDA_ERR_STRIDE, "%s: negative strides, or logits off their elements", who);
    const size_t need = verify_drafts_workspace_bytes(B, K, V, dtype);
    SPARDA_REQUIRE(workspace && workspace_bytes >= need && aligned16(workspace), SPARDA_ERR_WORKSPACE,
                   "%s: workspace of %zu bytes needed, 16-byte aligned", who, need);
    return launch_verify_drafts(logits, dtype, l_sb, l_st, drafts, d_sb, uniform, u_sb, K > 0 ? draft_probs : nullptr, p_sb, p_st,
                                n_drafts, temperatures, temperature, B, K, V, tokens, n_accepted, workspace,
                                static_cast<hipStream_t>(stream));
}
