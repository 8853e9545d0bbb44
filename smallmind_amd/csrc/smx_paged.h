// smx_paged.h -- layout of the paged KV cache (smx_paged_cache_*), shared by its writer, its reader, the attention
// over it and the eviction from it.
//
// A cache is a pool of pages of `page` positions (a power of two from 16 to 1024).  A row is the head_dim values of one
// position's K or V in one KV head, fp16 or bf16.  Memory is [page][kv head][K rows, then V rows], a row W values wide
// (W = head_dim rounded up to a width that the attention is built for; what lies beyond head_dim stays 0).
//
// Within a row the 16-byte units of 8 values change places by the row's number (pg_unit): pages go to LDS as they
// are, straight from memory, and there eight rows' units at one place of the row, or four rows' pairs of units, which is what the
// attention's matrix operands are read as, lie on different banks.
//
// Every value kept is finite but for one case: where a position's K or V (after rounding) holds a NaN or an infinity, its K row is NaN
// throughout and its V row 0.  A score of it is NaN, so whoever sees the position gets NaN; for whoever does not, its
// weight is 0 and 0 times V is 0, whatever was written.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace smx {

constexpr int kPgMaxHead = 256;   // largest head_dim
constexpr int kPgGroup = 16;      // positions that a page has whole multiples of

__host__ __device__ constexpr int pg_width(int hd) { return hd <= 128 ? (hd + 31) / 32 * 32 : hd <= 192 ? 192 : 256; }

// Where unit u of row r is.  Rows of whole 128 bytes (8 units) start on the same banks: eight permutations, such that
// pairs of units of four rows stay apart too; the others start on different ones, and four do.
__host__ __device__ constexpr int pg_turn(int w, int r) { return w % 64 == 0 ? 2 * (r & 3) + ((r >> 2) & 1) : (r >> 2) & 3; }
__host__ __device__ constexpr int pg_unit(int w, int u, int r) { return u ^ pg_turn(w, r); }

// What the kernels see of a cache.
struct PgView {
    uint8_t *base;
    int n_pages, n_kv, hd, w, page, bf16;

    __host__ __device__ size_t head_bytes() const { return (size_t)page * w * 4; }   // K and V of one page's head
    __host__ __device__ uint8_t *k_row(int pg, int head, int r) const
    {
        return base + ((size_t)pg * n_kv + head) * head_bytes() + (size_t)r * w * 2;
    }
    __host__ __device__ size_t v_off() const { return (size_t)page * w * 2; }        // from a K row to its V row
    __host__ __device__ size_t bytes() const { return (size_t)n_pages * n_kv * head_bytes(); }
};

// Element types at the entry points.
enum PgType { PG_F32 = 0, PG_F16 = 1, PG_BF16 = 2 };

// Rotation by position (smx_rotation, checked).
struct PgRotation {
    const float *cos, *sin;       // [n_pos][half]
    const int32_t *pos;           // [n_axes][n_tok]
    int n_pos, half, halves;      // half: pairs; halves: (j, j + half), otherwise (2 j, 2 j + 1)
    int ends[4];                  // pairs below ends[a] (and not below ends[a - 1]) turn by axis a
    int vec;                      // the tables can be read 16 bytes at a time
};

// Arguments of the write of rows (k_paged_write.hip).
struct PgWriteArgs {
    PgView c;                     // c.base null: K goes to k_out
    const void *q, *k, *v;        // token t's rows at t * stride (in elements); q, k, v may be null
    int64_t q_stride, k_stride, v_stride;
    const float *q_gamma, *k_gamma;
    float eps, inv_hd;
    PgRotation rot;               // half = 0: none
    const int32_t *places;
    void *q_out, *k_out;
    int n_tok, n_head, n_kv, hd;
    int out_type;                 // of q_out and k_out
    int vec;                      // rows can be read and written 16 bytes at a time
    int splits, q_parts;          // waves that share a token's rows; the first of them that take queries only (0: all take both)
    int group_shift;              // log2 of the lanes of a row
};

// Arguments of the eviction (k_paged_evict.hip).
struct PgEvictArgs {
    PgView c;
    const float *mass;            // [n_seq * n_kv] rows, mass_stride apart
    const int32_t *lens, *tables, *new_tables;
    int32_t *kept, *new_lens;     // [n_seq][n_kv][n_keep], [n_seq]
    float *new_mass;              // as kept
    int64_t mass_stride;
    int table_stride, new_stride;
    int n_keep, n_recent, max_len;
};

}  // namespace smx
