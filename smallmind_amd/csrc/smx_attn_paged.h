// smx_attn_paged.h -- arguments of the attention over the paged KV cache and of the weights that positions receive.
// The kernels are built once per row width and element type (k_attn_paged.hip); the plan, the dispatch and the joining
// of parts are in k_attn_paged_join.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smx_paged.h"

namespace smx {

constexpr int kPgTile = 64;      // positions that are gone through at once
constexpr int kPgRows = 32;      // rows (a query head of a token) of a wave

struct AttnPgArgs {
    PgView c;
    const void *q;               // token t, head h at t * q_stride + h * hd (elements)
    void *out;                   // [n_tok][n_head][hd]
    float *lse;                  // [n_tok][n_head] or null
    const int32_t *starts;       // [n_seq + 1]
    const int32_t *lens;         // [n_seq]
    const int32_t *tables;       // [n_seq][table_stride]
    const float *slopes;         // [n_head] or null
    const int32_t *prefix;       // [n_seq] or null
    float *part_ml, *part_acc;   // [parts][n_tok * n_head][2], [..][hd]
    // weights received: mass [n_seq * n_kv] rows of mass_width floats, mass_stride apart (or null), mass_out rows of max_len;
    // lse_in [n_tok][n_head]; with mass_parts > 1 part p goes to mass_part + p * n_seq * n_kv * max_len
    const float *mass, *lse_in;
    float *mass_out, *mass_part;
    int64_t mass_stride;
    int mass_width, mass_parts, mass_per;   // mass_per: rows' blocks of a part
    int64_t q_stride;
    double inv_group;            // n_kv / n_head
    float scale_log2e;           // of plain scores, as exponents of 2
    float cap_in, cap_out;       // scores * cap_in -> tanh -> * cap_out is an exponent of 2; cap_in 0: not capped
    int window;                  // 0: none
    int q_vec, out_vec;          // q, out may be read and written 16 bytes at a time
    int page_shift, table_stride;
    int n_tok, n_head, group, n_seq, max_q, max_len;
    int io;                      // PgType of q and out
    int tile_wgs, tile_blocks;   // workgroups (blocks of rows) of the many-row path; the rest take short sequences
    int short_rows;              // sequences of up to this many rows go the short way (0: none do)
    int chunk, parts;            // tiles that a part has at least; parts (1: the outputs are written at once)
    int ranked;                  // few rows: the longest sequences first
    float q_least;               // fp32 queries over F16: a row counts as no smaller, so that its unit times scale_log2e is not 0
};

// How blocks of 128 rows are gone through: by four waves, or by two groups of four that take tiles in turn; in PG_SPARE by
// four waves that leave registers for more blocks on a compute unit.  PG_SHORT: no sequence has more than 32 rows per KV head.
enum PgMode { PG_SHORT, PG_ONE_GROUP, PG_TWO_GROUPS, PG_SPARE };

// How a call is cut up.
struct AttnPgPlan {
    PgMode mode;
    int chunk, parts, tile_blocks, ranked;
    int64_t tile_wgs, blocks;
    int64_t work_bytes;
};

struct MassPgPlan {
    bool few;                    // every sequence has up to 32 rows per KV head
    int parts, per, ranked;
    int64_t blocks, work_bytes;
};

}  // namespace smx
