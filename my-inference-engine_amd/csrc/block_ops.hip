// Blocks of a paged cache copied, forked and moved together.
//
// All of it is moving bytes: block j of every plane (a layer's K or V) is one contiguous run (16 tokens
// x 2 kv heads x 128 x 2 bytes = 8 KB in the engine's cache).  One work-group copies one piece of one
// block of one plane; the table rows of a fork or a move are further work-groups of the same launch.
#include "cache_ops.h"

namespace mi_fa2 {

constexpr int kBoThreads = 256;
constexpr int kBoPiece = 16384;  // bytes of a block per work-group

// bytes [0, n) of src to dst by the work-group, U at a time.
template <typename U>
__device__ __forceinline__ void copy_span(uint8_t* dst, const uint8_t* src, int64_t n) {
  U* d = reinterpret_cast<U*>(dst);
  const U* s = reinterpret_cast<const U*>(src);
  for (int64_t i = threadIdx.x; i < n / (int64_t)sizeof(U); i += kBoThreads) d[i] = s[i];
}

template <typename U, int OP>
__global__ __launch_bounds__(kBoThreads) void block_op_kernel(const BlockOpParams p, int pieces) {
  const int copies = p.n * pieces;
  if ((int)blockIdx.x >= copies) {
    // table rows
    if (blockIdx.y != 0) return;
    const int i = blockIdx.x - copies;
    if constexpr (OP == kMove) {
      const int slot = p.rows[2 * i], held = min(p.rows[2 * i + 1], p.table_width);
      if (slot < 0 || slot >= p.max_seqs) return;
      int32_t* t = p.tables + slot * p.table_stride;
      for (int j = threadIdx.x; j < held; j += kBoThreads) {
        const int b = t[j];
        if ((unsigned)b < (unsigned)p.src_blocks) t[j] = p.new_ids[b];
      }
    }
    if constexpr (OP == kFork) {
      const int parent = p.children[4 * i], child = p.children[4 * i + 1];
      const int len = p.children[4 * i + 2], fresh = p.children[4 * i + 3];
      if ((unsigned)parent >= (unsigned)p.max_seqs || (unsigned)child >= (unsigned)p.max_seqs ||
          parent == child || len < 0)
        return;
      const int whole = len / p.block_size, rest = len - whole * p.block_size;
      if (whole + (rest > 0) > p.table_width) return;
      const int32_t* from = p.tables + parent * p.table_stride;
      int32_t* to = p.tables + child * p.table_stride;
      if (rest > 0 && ((unsigned)fresh >= (unsigned)p.src_blocks ||
                       (unsigned)from[whole] >= (unsigned)p.src_blocks))
        return;
      for (int j = threadIdx.x; j < whole; j += kBoThreads) to[j] = from[j];
      if (threadIdx.x == 0) {
        if (rest > 0) to[whole] = fresh;
        p.seq_lens[child] = len;
      }
    }
    return;
  }
  const int i = blockIdx.x / pieces;
  const int64_t at = (int64_t)(blockIdx.x - i * pieces) * kBoPiece;
  int from, to;
  int64_t bytes = p.block_bytes;
  if constexpr (OP == kFork) {
    const int parent = p.children[4 * i], child = p.children[4 * i + 1];
    const int len = p.children[4 * i + 2];
    if ((unsigned)parent >= (unsigned)p.max_seqs || (unsigned)child >= (unsigned)p.max_seqs ||
        parent == child || len < 0)
      return;
    const int whole = len / p.block_size, rest = len - whole * p.block_size;
    if (rest == 0 || whole + 1 > p.table_width) return;
    from = p.tables[parent * p.table_stride + whole];
    to = p.children[4 * i + 3];
    bytes = rest * p.token_bytes;
  } else {
    from = p.pairs[2 * i];
    to = p.pairs[2 * i + 1];
  }
  if ((unsigned)from >= (unsigned)p.src_blocks || (unsigned)to >= (unsigned)p.dst_blocks) return;
  if (at >= bytes) return;
  const int64_t plane = blockIdx.y;
  copy_span<U>(p.dst + plane * p.dst_plane + to * p.block_bytes + at,
               p.src + plane * p.src_plane + from * p.block_bytes + at,
               min(bytes - at, (int64_t)kBoPiece));
}

template <typename U>
static hipError_t launch_block_op_t(const BlockOpParams& p, int op, hipStream_t stream) {
  const int pieces = (int)((p.block_bytes + kBoPiece - 1) / kBoPiece);
  const int rows = op == kMove ? p.n_rows : op == kFork ? p.n : 0;
  const dim3 grid(p.n * pieces + rows, p.planes);
  if (op == kCopy)
    hipLaunchKernelGGL((block_op_kernel<U, kCopy>), grid, dim3(kBoThreads), 0, stream, p, pieces);
  else if (op == kFork)
    hipLaunchKernelGGL((block_op_kernel<U, kFork>), grid, dim3(kBoThreads), 0, stream, p, pieces);
  else
    hipLaunchKernelGGL((block_op_kernel<U, kMove>), grid, dim3(kBoThreads), 0, stream, p, pieces);
  return hipGetLastError();
}

hipError_t launch_block_op(const BlockOpParams& p, int op, hipStream_t stream) {
  // 16 bytes at a time where every run starts on a 16-byte boundary and is a multiple of it
  const uint64_t all = reinterpret_cast<uint64_t>(p.src) | reinterpret_cast<uint64_t>(p.dst) |
                       (uint64_t)p.src_plane | (uint64_t)p.dst_plane | (uint64_t)p.block_bytes |
                       (op == kFork ? (uint64_t)p.token_bytes : 0);
  return all % 16 == 0 ? launch_block_op_t<u32x4>(p, op, stream)
                       : launch_block_op_t<uint8_t>(p, op, stream);
}

}  // namespace mi_fa2
