// smx_attn_q8.h -- arguments of the attention over the 8-bit KV cache.  The kernel is built once per
// row width (k_attn_q8.hip); the plan, the dispatch and the joining of parts are in k_attn_q8_join.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "smx_kvcache.h"

namespace smx {

// How the rows go through the prefix (k_attn_q8.hip).
enum AttnQ8Pre { PRE_NONE, PRE_STREAM, PRE_ROWS };

struct AttnQ8Args {
    const float *q;             // token t, head h at t * q_stride + h * hd
    float *out;                 // [n_seq * n_q][n_head][hd]
    const uint8_t *cache;
    size_t head_bytes;          // of one (slot, KV head)
    const int32_t *slots, *lens;
    float *part_ml, *part_acc;  // [parts][n_rows][2], [parts][n_rows][hd]
    int64_t q_stride, n_rows;   // n_rows = n_seq * n_q * n_head
    double inv_group;           // n_kv / n_head
    // Scores are held as q . k / 16, no larger than what they stand for (hd <= 256), which spares them fp32's end;
    // log2(e) 16 / sqrt(hd) makes them exponents.
    float scale_log2e;
    int q_vec, out_vec;         // q, out may be read and written as float4
    int n_slots, n_seq, n_q, n_head, n_kv, hd;
    int max_len, own_chunk, own_splits, own_blocks;
    int prefix_slot, prefix_len, pre_chunk, pre_splits, pre_wgs;
    int parts;                  // pre_splits + own_splits
    int direct;                 // a single part of the sequences' own positions: it writes the outputs
};

// How a call is cut up.
struct AttnQ8Plan {
    AttnQ8Pre pre;
    bool past_caches;           // the sequences' positions are read past the caches (PRE_NONE)
    int own_chunk, own_splits, own_blocks;
    int pre_chunk, pre_splits, pre_blocks;
    int parts;
    int64_t blocks, pre_wgs;    // workgroups of the launch
    int64_t work_bytes;         // of the parts (0 where none are kept)
};

}  // namespace smx
