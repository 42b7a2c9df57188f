// Blocks of a paged cache copied, forked and moved together.
//
// All of it is moving bytes: block j of every plane (a layer's K or V) is one contiguous run (16 tokens
// x 2 kv heads x 128 x 2 bytes = 8 KB in the engine's cache).  One work-group copies one piece of one
// block of one plane; the table rows of a fork or a move are further work-groups of the same launch.
#include "cache_ops.h"

namespace mi_fa2 {

constexpr int kBoThreads = 256;
constexpr int kBoPiece = 16384;  // bytes of a block per work-group

// bytes [0, n) of src to dst by the work-group, U at a time, four loads of a thread in flight.  What is
// written goes past the caches (non-temporal): blocks copied or moved are not read soon.  (A fork's started
// block is, by the child's next step: at most 8 KB a child and plane with the engine's blocks, from the last-level
// cache or memory.)  NT: what is read goes past them too.
template <typename U, bool NT>
__device__ __forceinline__ void copy_span(uint8_t* dst, const uint8_t* src, int n) {
  constexpr int kFlight = 4;
  U* d = reinterpret_cast<U*>(dst);
  const U* s = reinterpret_cast<const U*>(src);
  const int m = n / (int)sizeof(U);
  for (int i = threadIdx.x; i < m; i += kFlight * kBoThreads) {
    U x[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i + k * kBoThreads < m)
        x[k] = NT ? __builtin_nontemporal_load(s + i + k * kBoThreads) : s[i + k * kBoThreads];
#pragma unroll
    for (int k = 0; k < kFlight; ++k)
      if (i + k * kBoThreads < m) __builtin_nontemporal_store(x[k], d + i + k * kBoThreads);
  }
}

// A fork's child, if everything it names is in range.
struct Child {
  int parent, slot, length, fresh, whole, rest;
  bool ok;
};
__device__ __forceinline__ Child child_of(const BlockOpParams& p, int i) {
  const int4 c = *reinterpret_cast<const int4*>(p.children + 4 * i);
  Child r{c.x, c.y, c.z, c.w, 0, 0, false};
  if ((unsigned)r.parent >= (unsigned)p.max_seqs || (unsigned)r.slot >= (unsigned)p.max_seqs ||
      r.parent == r.slot || r.length < 0)
    return r;
  r.whole = r.length / p.block_size;
  r.rest = r.length - r.whole * p.block_size;
  r.ok = r.whole + (r.rest > 0) <= p.table_width &&
         (r.rest == 0 || (unsigned)r.fresh < (unsigned)p.src_blocks);
  return r;
}

// Work-groups [0, rows) rewrite tables (fork: a child each, move: a row each); the others copy a piece of a
// block in a plane each, plane by plane (blocks that lie together are copied together: 1,500 blocks of 8 KB
// in 56 planes 227 us, 6.1 TB/s read and written; with the planes of a block side by side 267).
template <typename U, int OP, bool NT>
__global__ __launch_bounds__(kBoThreads) void block_op_kernel(const BlockOpParams p, int pieces, int rows,
                                                              FastDiv jobs) {
  if ((int)blockIdx.x < rows) {
    const int i = blockIdx.x;
    if constexpr (OP == kMove) {
      const int slot = p.rows[2 * i], held = min(p.rows[2 * i + 1], p.table_width);
      if ((unsigned)slot >= (unsigned)p.max_seqs) return;
      int32_t* t = p.tables + slot * p.table_stride;
      for (int j = threadIdx.x; j < held; j += kBoThreads) {
        const int b = t[j];
        if ((unsigned)b < (unsigned)p.src_blocks) t[j] = p.new_ids[b];
      }
    }
    if constexpr (OP == kFork) {
      const Child c = child_of(p, i);
      if (!c.ok) return;
      const int32_t* from = p.tables + c.parent * p.table_stride;
      int32_t* to = p.tables + c.slot * p.table_stride;
      if (c.rest > 0 && (unsigned)from[c.whole] >= (unsigned)p.src_blocks) return;
      for (int j = threadIdx.x; j < c.whole; j += kBoThreads) to[j] = from[j];
      if (threadIdx.x == 0) {
        if (c.rest > 0) to[c.whole] = c.fresh;
        p.seq_lens[c.slot] = c.length;
      }
    }
    return;
  }
  const int work = blockIdx.x - rows;
  const int plane = fdiv(work, jobs), job = work - plane * (int)jobs.d;
  const int i = job / pieces;
  const int64_t at = (int64_t)(job - i * pieces) * kBoPiece;
  int from, to;
  int64_t bytes = p.block_bytes;
  if constexpr (OP == kFork) {
    const Child c = child_of(p, i);
    if (!c.ok || c.rest == 0) return;
    from = p.tables[c.parent * p.table_stride + c.whole];
    to = c.fresh;
    bytes = c.rest * p.token_bytes;
  } else {
    from = p.pairs[2 * i];
    to = p.pairs[2 * i + 1];
  }
  if ((unsigned)from >= (unsigned)p.src_blocks || (unsigned)to >= (unsigned)p.dst_blocks) return;
  if (at >= bytes) return;
  copy_span<U, NT>(p.dst + plane * p.dst_plane + to * p.block_bytes + at,
                   p.src + plane * p.src_plane + from * p.block_bytes + at,
                   (int)min(bytes - at, (int64_t)kBoPiece));
}

// Copies of at least 16 MB read past the caches.  A source that was not touched lately is faster so at any
// size (150 blocks of 8 KB in 56 planes, 69 MB: 33 us, 47 through the caches; 1,500: 241 and 313), one that
// the caches still hold is slower while it is small (20 blocks, 9 MB: 5.0 and 3.5).
constexpr int64_t kBoStream = int64_t(1) << 24;

template <typename U, int OP, bool NT>
static hipError_t launch_block_op_t(const BlockOpParams& p, hipStream_t stream) {
  const int pieces = (int)((p.block_bytes + kBoPiece - 1) / kBoPiece);
  const int rows = OP == kMove ? p.n_rows : OP == kFork ? p.n : 0, jobs = p.n * pieces;
  hipLaunchKernelGGL((block_op_kernel<U, OP, NT>), dim3(rows + jobs * p.planes), dim3(kBoThreads), 0, stream,
                     p, pieces, rows, make_fastdiv(jobs > 0 ? jobs : 1));
  return hipGetLastError();
}

template <typename U>
static hipError_t launch_block_op_u(const BlockOpParams& p, int op, hipStream_t stream) {
  const bool nt = p.n * p.block_bytes >= kBoStream / p.planes;
  if (op == kFork) return launch_block_op_t<U, kFork, false>(p, stream);
  if (op == kMove)
    return nt ? launch_block_op_t<U, kMove, true>(p, stream) : launch_block_op_t<U, kMove, false>(p, stream);
  return nt ? launch_block_op_t<U, kCopy, true>(p, stream) : launch_block_op_t<U, kCopy, false>(p, stream);
}

hipError_t launch_block_op(const BlockOpParams& p, int op, hipStream_t stream) {
  // 16 bytes at a time where every run starts on a 16-byte boundary and is a multiple of it
  const uint64_t all = reinterpret_cast<uint64_t>(p.src) | reinterpret_cast<uint64_t>(p.dst) |
                       (uint64_t)p.src_plane | (uint64_t)p.dst_plane | (uint64_t)p.block_bytes |
                       (op == kFork ? (uint64_t)p.token_bytes : 0);
  return all % 16 == 0 ? launch_block_op_u<u32x4>(p, op, stream)
                       : launch_block_op_u<uint8_t>(p, op, stream);
}

}  // namespace mi_fa2
