// Parameters of the block operations (block_ops.hip) and of the attention over shared blocks
// (shared_attn.hip).
#pragma once

#include "fa2_common.h"

namespace mi_fa2 {

struct BlockOpParams {
  const uint8_t* src;
  uint8_t* dst;
  int64_t src_plane, dst_plane;  // bytes between planes
  int32_t src_blocks, dst_blocks, planes;
  int64_t block_bytes;
  const int32_t* pairs;          // copy, move: [n][2] source, destination
  const int32_t* children;       // fork: [n][4] parent slot, child slot, tokens, new block
  int32_t n;
  int32_t* tables;               // fork, move: [max_seqs][table_stride]
  int64_t table_stride;
  int32_t table_width, max_seqs;
  int32_t* seq_lens;             // fork
  int32_t block_size;            // fork: tokens of a block
  int64_t token_bytes;
  const int32_t* rows;           // move: [n_rows][2] slot, blocks held
  int32_t n_rows;
  const int32_t* new_ids;        // move: [src_blocks]
};
enum BlockOp { kCopy = 0, kFork = 1, kMove = 2 };
hipError_t launch_block_op(const BlockOpParams& p, int op, hipStream_t stream);

// Rows per call of the attention.
constexpr int kShMaxRows = 512;

struct SharedParams {
  const uint16_t* q;    // [total_q][Hq][128], token and head strides
  const uint16_t* k;    // pools: slot and head strides
  const uint16_t* v;
  uint16_t* o;
  float* lse;           // or NULL
  const int32_t* cu_q;  // [B + 1]
  const int32_t* table; // [B][bt_stride]
  int64_t bt_stride;
  const int32_t* kv_lens;      // [B]
  const int32_t* cu_rows;      // [G + 1]
  const int32_t* prefix_lens;  // [G]
  int64_t q_st, q_sh, kv_st, kv_sh, o_st, o_sh, l_sh, l_st;
  int32_t G, B, total_q, Hq, Hkv, group;
  int32_t max_kv, bs_shift, num_blocks, causal;
  float scale_log2;
  // filled by launch_shared
  FastDiv group_div, heads_div;
  float* ws_o;          // parts: [column][128] fp32, unnormalised
  float* ws_ml;         // [column][2]: maximum (of the unscaled scores) and sum
  int32_t* ws_where;    // [2][total_q][Hq][2]: where a pair's parts stand, of the prefix and its own keys
  int32_t columns;      // of the workspace
  int32_t narrow_base;  // the first column of the waves' parts
};

// The workspace.  In each of two areas (the work-groups' parts and the waves') an item's parts begin at
// the number of pairs before the item (prefixes first, total_q * heads_q of them, then rows) and worker
// w's part of it stands w tiles further: from one (item, worker) to the next either number grows, so no
// two parts meet.
constexpr int kSharedWgs = 256, kSharedWaves = 8, kSharedTile = 128, kSharedNarrow = 32;
struct SharedSpace {
  int32_t columns, narrow;
  size_t ml, where, total;   // byte offsets after the O parts
};
inline SharedSpace shared_space(int64_t total_q, int64_t heads_q) {
  const int64_t pairs = 2 * total_q * heads_q;
  const int64_t narrow = pairs + kSharedTile * kSharedWgs;
  const int64_t columns = narrow + pairs + kSharedNarrow * kSharedWgs * kSharedWaves;
  SharedSpace s{};
  s.columns = (int32_t)columns;
  s.narrow = (int32_t)narrow;
  s.ml = (size_t)columns * kHeadDim * sizeof(float);
  s.where = s.ml + (size_t)columns * 2 * sizeof(float);
  s.total = s.where + (size_t)pairs * 2 * sizeof(int32_t);
  return s;
}
hipError_t launch_shared(SharedParams p, int dtype, int n_cus, void* workspace, hipStream_t stream);

}  // namespace mi_fa2
