// smx_kvcache.h -- layout of the 8-bit KV cache (smx_kv_cache_*), shared by its writer, its reader
// and the attention over it.
//
// A cache holds n_slots sequences of up to ctx positions.  One row is the head_dim values of one
// position's K or V in one KV head: 8-bit codes with one fp32 scale (a Q8Tensor block of head_dim
// elements, Q8Tensor.cs:72-128), value = (byte - 128) * scale.
//
// Memory is [slot][kv head][tile of 64 positions], each tile one contiguous record:
//   K codes  [64 positions][W]       W = head_dim rounded up to a multiple of 32
//   V codes  [W dims][64 positions]  position p of the tile at byte 16 ((p / 4) % 4) + 4 (p / 16) + p % 4
//   K scales [64] fp32, V scales [64] fp32
// so that a wave streams records front to back, and both operands of the attention's products come
// out of 16-byte loads in the order of the matrix instructions' lanes: of 64 positions the products
// q K^T leave lane 16 g + c the positions 16 t + 4 g + i (t, i < 4), and those are the 16 bytes that
// the lane loads of a V row.  The offset of 128 lets two instructions per two bytes turn codes into
// fp16 (k_attn_q8.hip).  What lies beyond head_dim or beyond the written positions is never used.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace smx {

constexpr int kKvTile = 64;      // positions per tile
constexpr int kKvMaxHead = 256;  // largest head_dim
constexpr int kKvZero = 128;     // the byte that stands for 0

__host__ __device__ constexpr int kv_width(int head_dim) { return (head_dim + 31) / 32 * 32; }
__host__ __device__ constexpr size_t kv_tile_bytes(int w) { return (size_t)2 * kKvTile * w + 2 * kKvTile * 4; }
// byte of position p (0..63) in a dim's V row
__host__ __device__ constexpr int kv_v_byte(int p) { return 16 * ((p >> 2) & 3) + 4 * (p >> 4) + (p & 3); }

// What the kernels see of a cache.
struct KvView {
    uint8_t *base;
    int n_slots, n_kv, hd, w, ctx, tiles;   // tiles: per (slot, head)

    __host__ __device__ size_t tile_off(int slot, int head, int tile) const
    {
        return (((size_t)slot * n_kv + head) * tiles + tile) * kv_tile_bytes(w);
    }
    __host__ __device__ size_t bytes() const { return (size_t)n_slots * n_kv * tiles * kv_tile_bytes(w); }
};

}  // namespace smx
