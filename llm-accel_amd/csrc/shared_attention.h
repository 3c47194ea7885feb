// shared_attention.h -- attention of a batch whose sequences share a prefix
// (internal to the library).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llm {

struct SharedAttnArgs {
    const int16_t* q;        // [sequences][kv_heads * group][d], after RoPE
    const int16_t* kcache;   // this layer's pages (attention.h)
    const int16_t* vcache;
    uint32_t pages;          // per KV head
    const int16_t *k_own, *v_own;  // [sequences][kv_heads][own_cap][d]
    const uint32_t* own_len;       // [sequences], at most own_cap count
    int16_t* out;            // as q
    uint32_t sequences, prefix, own_cap;
    uint32_t kv_heads, group, head_dim;
    int32_t qk_scale;
    const int16_t* exp14;
    // Tiles of 64 positions: `whole` lie in the prefix and are every row's,
    // then each sequence has up to own_tiles of its own (the first may begin
    // with the prefix's last positions); rows of a KV head are rho =
    // sequence * group + query head, padded to 16.
    uint32_t whole, own_tiles, tiles, rows, rows_pad;
    // scratch: scores, their maximum per tile, and per tile the factor of
    // what came before, the probabilities' sum, and the values
    int16_t* scores;  // [kv_heads][tiles][rows_pad][64]
    int16_t* tmax;    // [kv_heads][tiles][rows_pad]
    int32_t* old;     // [kv_heads][tiles][rows_pad]
    int32_t* tsum;    // [kv_heads][tiles][rows_pad]
    int16_t* tval;    // [kv_heads][tiles][rows_pad][d]
    uint32_t inv_group;  // 2^16 / group, rounded up: rho / group = rho inv_group >> 16
    // workgroups of the launches over tiles: row groups per shared tile, and
    // how many
    uint32_t groups, shared_jobs, own_jobs;
};
// Fills the derived sizes (whole .. own_jobs).
void shared_attention_shape(SharedAttnArgs& a);
// Bytes of the scratch (0: few tiles, none used), and its parts laid out from
// `base`.
size_t shared_attention_bytes(const SharedAttnArgs& a);
void shared_attention_scratch(SharedAttnArgs& a, uint8_t* base);
hipError_t launch_shared_attention(const SharedAttnArgs& a, hipStream_t st);

}  // namespace llm
