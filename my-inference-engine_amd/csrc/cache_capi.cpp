// C ABI of libmi_cache.so: argument checks and launches of the block operations and of the attention
// over shared blocks.  The contract of every entry point is in include/mi_cache.h.
#include "mi_cache.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "cache_ops.h"

namespace {

using mi_fa2::BlockOpParams;
using mi_fa2::SharedParams;

enum Status { kOk = 0, kInvalid = 1, kUnsupported = 2, kWorkspace = 3, kLaunch = 4 };

thread_local char g_err[256] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int ok() {
  g_err[0] = '\0';
  return kOk;
}

int launched(hipError_t err) {
  if (err != hipSuccess) return fail(kLaunch, "kernel launch failed: %s", hipGetErrorString(err));
  return ok();
}

// The current device's compute units, read once per device.
int compute_units(int* out) {
  static std::atomic<int> known[64];
  int dev = -1;
  *out = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err == hipSuccess && dev >= 0 && dev < 64) *out = known[dev].load(std::memory_order_relaxed);
  if (err == hipSuccess && *out == 0) {
    err = hipDeviceGetAttribute(out, hipDeviceAttributeMultiprocessorCount, dev);
    if (err == hipSuccess && dev < 64) known[dev].store(*out, std::memory_order_relaxed);
  }
  if (err != hipSuccess || *out <= 0)
    return fail(kLaunch, "reading the device's CU count failed: %s", hipGetErrorString(err));
  return kOk;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A pool's sizes: planes go into a grid dimension, and a plane must hold its blocks.
int check_pool(const char* name, const void* p, int64_t plane_bytes, int32_t num_blocks,
               int32_t planes, int64_t block_bytes) {
  if (!p) return fail(kInvalid, "%s is NULL", name);
  if (num_blocks < 0 || planes < 0 || block_bytes <= 0)
    return fail(kInvalid, "%s: bad sizes: %d blocks of %lld bytes in %d planes", name, num_blocks,
                (long long)block_bytes, planes);
  if (planes > 65535) return fail(kUnsupported, "%s: %d planes, at most 65535", name, planes);
  if (block_bytes > (int64_t(1) << 40) || plane_bytes / block_bytes < num_blocks)
    return fail(kInvalid, "%s: planes of %lld bytes do not hold %d blocks of %lld", name,
                (long long)plane_bytes, num_blocks, (long long)block_bytes);
  return kOk;
}

// A launch stays below 2^31 threads: one work-group of 256 for each 16 KB of a block and plane, and for
// each table row.
int check_count(int64_t n, int64_t rows, int64_t block_bytes, int64_t planes) {
  if (n < 0 || rows < 0) return fail(kInvalid, "bad counts: %lld, %lld", (long long)n, (long long)rows);
  const int64_t pieces = (block_bytes + 16383) / 16384;
  if (n >= int64_t(1) << 23 || pieces >= int64_t(1) << 23 ||
      n * pieces >= (int64_t(1) << 23) / std::max<int64_t>(planes, 1) - rows / std::max<int64_t>(planes, 1) - 1)
    return fail(kUnsupported, "%lld blocks of %lld bytes in %lld planes, %lld rows in one call",
                (long long)n, (long long)block_bytes, (long long)planes, (long long)rows);
  return kOk;
}

int check_table(const int32_t* tables, int64_t stride, int32_t width, int32_t max_seqs) {
  if (!tables) return fail(kInvalid, "tables is NULL");
  if (width < 0 || max_seqs < 0 || stride < width)
    return fail(kInvalid, "bad tables: %d rows of %d entries, %lld apart", max_seqs, width,
                (long long)stride);
  return kOk;
}

// (token, head) pairs of a call: a wave each in the merge, below 2^32 threads.
constexpr int64_t kMaxPairs = int64_t(1) << 25;

int check_tensor(const char* name, const void* p, const int64_t* strides) {
  if (!p) return fail(kInvalid, "%s is NULL", name);
  if (!aligned16(p)) return fail(kInvalid, "%s is not 16-byte aligned", name);
  if (!strides) return fail(kInvalid, "%s strides are NULL", name);
  for (int i = 0; i < 2; ++i)
    if (strides[i] % 8 != 0)
      return fail(kInvalid, "%s stride[%d] = %lld is not a multiple of 8 elements", name, i,
                  (long long)strides[i]);
  return kOk;
}

}  // namespace

extern "C" {

const char* mi_cache_last_error(void) { return g_err; }

int mi_cache_copy_blocks(const void* src, int64_t src_plane_bytes, int32_t src_num_blocks,
                         void* dst, int64_t dst_plane_bytes, int32_t dst_num_blocks,
                         int32_t planes, int64_t block_bytes, const int32_t* pairs, int32_t n,
                         void* stream) {
  if (int rc = check_pool("src", src, src_plane_bytes, src_num_blocks, planes, block_bytes)) return rc;
  if (int rc = check_pool("dst", dst, dst_plane_bytes, dst_num_blocks, planes, block_bytes)) return rc;
  if (int rc = check_count(n, 0, block_bytes, planes)) return rc;
  if (n == 0 || planes == 0) return ok();
  if (!pairs) return fail(kInvalid, "pairs is NULL");
  BlockOpParams p{};
  p.src = static_cast<const uint8_t*>(src);
  p.dst = static_cast<uint8_t*>(dst);
  p.src_plane = src_plane_bytes, p.dst_plane = dst_plane_bytes;
  p.src_blocks = src_num_blocks, p.dst_blocks = dst_num_blocks;
  p.planes = planes;
  p.block_bytes = block_bytes;
  p.pairs = pairs;
  p.n = n;
  return launched(mi_fa2::launch_block_op(p, mi_fa2::kCopy, static_cast<hipStream_t>(stream)));
}

int mi_cache_fork_rows(void* pool, int64_t plane_bytes, int32_t num_blocks, int32_t planes,
                       int32_t block_size, int64_t token_bytes, int32_t* tables,
                       int64_t table_stride, int32_t table_width, int32_t* seq_lens,
                       int32_t max_seqs, const int32_t* children, int32_t n, void* stream) {
  if (block_size <= 0 || token_bytes <= 0 || token_bytes > int64_t(1) << 32 || block_size > 1 << 20)
    return fail(kInvalid, "bad block: %d tokens of %lld bytes", block_size, (long long)token_bytes);
  const int64_t block_bytes = block_size * token_bytes;
  if (int rc = check_pool("pool", pool, plane_bytes, num_blocks, planes, block_bytes)) return rc;
  if (int rc = check_table(tables, table_stride, table_width, max_seqs)) return rc;
  if (int rc = check_count(n, n, block_bytes, planes)) return rc;
  if (!seq_lens) return fail(kInvalid, "seq_lens is NULL");
  if (planes == 0) return fail(kInvalid, "pool: no planes");
  if (n == 0) return ok();
  if (!children) return fail(kInvalid, "children is NULL");
  if (!aligned16(children)) return fail(kInvalid, "children is not 16-byte aligned");
  BlockOpParams p{};
  p.src = p.dst = static_cast<uint8_t*>(pool);
  p.src_plane = p.dst_plane = plane_bytes;
  p.src_blocks = p.dst_blocks = num_blocks;
  p.planes = planes;
  p.block_bytes = block_bytes;
  p.block_size = block_size;
  p.token_bytes = token_bytes;
  p.children = children;
  p.n = n;
  p.tables = tables;
  p.table_stride = table_stride;
  p.table_width = table_width;
  p.seq_lens = seq_lens;
  p.max_seqs = max_seqs;
  return launched(mi_fa2::launch_block_op(p, mi_fa2::kFork, static_cast<hipStream_t>(stream)));
}

int mi_cache_move_blocks(void* pool, int64_t plane_bytes, int32_t num_blocks, int32_t planes,
                         int64_t block_bytes, const int32_t* pairs, int32_t n, int32_t* tables,
                         int64_t table_stride, int32_t table_width, int32_t max_seqs,
                         const int32_t* rows, int32_t n_rows, const int32_t* new_ids,
                         void* stream) {
  if (int rc = check_pool("pool", pool, plane_bytes, num_blocks, planes, block_bytes)) return rc;
  if (int rc = check_count(n, n_rows, block_bytes, planes)) return rc;
  if (planes == 0) return fail(kInvalid, "pool: no planes");
  if (n > 0 && !pairs) return fail(kInvalid, "pairs is NULL");
  if (n_rows > 0) {
    if (int rc = check_table(tables, table_stride, table_width, max_seqs)) return rc;
    if (!rows) return fail(kInvalid, "rows is NULL");
    if (!new_ids) return fail(kInvalid, "new_ids is NULL");
  }
  if (n == 0 && n_rows == 0) return ok();
  BlockOpParams p{};
  p.src = p.dst = static_cast<uint8_t*>(pool);
  p.src_plane = p.dst_plane = plane_bytes;
  p.src_blocks = p.dst_blocks = num_blocks;
  p.planes = planes;
  p.block_bytes = block_bytes;
  p.pairs = pairs;
  p.n = n;
  p.tables = tables;
  p.table_stride = table_stride;
  p.table_width = table_width;
  p.max_seqs = max_seqs;
  p.rows = rows;
  p.n_rows = n_rows;
  p.new_ids = new_ids;
  return launched(mi_fa2::launch_block_op(p, mi_fa2::kMove, static_cast<hipStream_t>(stream)));
}

size_t mi_cache_attend_workspace_size(int32_t total_q, int32_t heads_q) {
  if (total_q <= 0 || heads_q <= 0 || int64_t(total_q) * heads_q > kMaxPairs) return 0;
  return mi_fa2::shared_space(total_q, heads_q).total;
}

int mi_cache_attend(int32_t dtype, const void* q, const void* k_pool, const void* v_pool, void* o,
                    float* lse, const int32_t* cu_seqlens_q, const int32_t* block_table,
                    int64_t block_table_stride, const int32_t* kv_lens, const int32_t* cu_rows,
                    const int32_t* prefix_lens, int32_t n_groups, int32_t batch, int32_t total_q,
                    int32_t heads_q, int32_t heads_kv, int32_t max_kv_len, int32_t head_dim,
                    int32_t block_size, int32_t num_blocks, const int64_t* q_strides,
                    const int64_t* pool_strides, const int64_t* o_strides,
                    const int64_t* lse_strides, int32_t is_causal, float sm_scale, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (dtype != 0 && dtype != 1)
    return fail(kUnsupported, "dtype %d is not bf16 (0) or fp16 (1)", dtype);
  if (head_dim != mi_fa2::kHeadDim)
    return fail(kUnsupported, "head_dim %d: the kernel is built for head_dim 128", head_dim);
  if (batch < 0 || heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv || total_q < 0)
    return fail(kInvalid, "bad sizes: batch=%d total_q=%d heads_q=%d heads_kv=%d", batch, total_q,
                heads_q, heads_kv);
  if (batch > mi_fa2::kShMaxRows || heads_q > 65535)
    return fail(kUnsupported, "batch %d (at most %d), heads_q %d (at most 65535)", batch,
                mi_fa2::kShMaxRows, heads_q);
  if (int64_t(total_q) * heads_q > kMaxPairs)
    return fail(kUnsupported, "%d tokens of %d heads: at most 2^25 pairs", total_q, heads_q);
  // the shares of work are counted in 32 bits: (tiles of 128 pairs, at most one more per range and
  // head) x (64-key units, and what an item costs beside them)
  if ((int64_t(total_q) * heads_q / 64 + 4 * int64_t(batch) * heads_kv) *
          (max_kv_len / 64 + int64_t(4)) >= int64_t(1) << 31)
    return fail(kUnsupported, "%d tokens over %d keys in one call", total_q, max_kv_len);
  if (n_groups < 0 || n_groups > batch)
    return fail(kInvalid, "n_groups %d: 0 to batch (%d)", n_groups, batch);
  if (max_kv_len < 0) return fail(kInvalid, "max_kv_len %d < 0", max_kv_len);
  // a step ends up to 128 keys behind the last one; positions are 32-bit
  if (max_kv_len > INT32_MAX - 8192)
    return fail(kUnsupported, "max_kv_len %d: at most 2^31 - 8193", max_kv_len);
  if (block_size < 16 || (block_size & (block_size - 1)))
    return fail(kUnsupported, "block_size %d is not a power of two >= 16", block_size);
  if (num_blocks < 0) return fail(kInvalid, "num_blocks %d < 0", num_blocks);
  if (!(sm_scale > 0.f) || !(sm_scale < 3.0e38f))
    return fail(kInvalid, "sm_scale is not a positive finite number");
  if (batch == 0 || total_q == 0) return ok();
  if (!cu_seqlens_q) return fail(kInvalid, "cu_seqlens_q is NULL");
  if (!kv_lens) return fail(kInvalid, "kv_lens is NULL");
  if (n_groups > 0 && (!cu_rows || !prefix_lens))
    return fail(kInvalid, "cu_rows or prefix_lens is NULL");
  if (max_kv_len > 0 && !block_table) return fail(kInvalid, "block_table is NULL");
  if (block_table_stride < 0)
    return fail(kInvalid, "block_table stride %lld < 0", (long long)block_table_stride);
  if (int rc = check_tensor("q", q, q_strides)) return rc;
  if (int rc = check_tensor("o", o, o_strides)) return rc;
  if (int rc = check_tensor("k_pool", k_pool, pool_strides)) return rc;
  if (int rc = check_tensor("v_pool", v_pool, pool_strides)) return rc;
  if (pool_strides[0] < head_dim || pool_strides[0] >= int64_t(1) << 24)
    return fail(pool_strides[0] < head_dim ? kInvalid : kUnsupported,
                "pool slot stride %lld: from head_dim to 2^24 - 8", (long long)pool_strides[0]);
  if (lse && !lse_strides) return fail(kInvalid, "lse strides are NULL");
  const size_t need = mi_cache_attend_workspace_size(total_q, heads_q);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(kWorkspace, "workspace: %zu bytes given, %zu needed, 16-byte aligned",
                workspace ? workspace_bytes : size_t(0), need);

  SharedParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k_pool);
  p.v = static_cast<const uint16_t*>(v_pool);
  p.o = static_cast<uint16_t*>(o);
  p.lse = lse;
  p.cu_q = cu_seqlens_q;
  p.table = block_table;
  p.bt_stride = block_table_stride;
  p.kv_lens = kv_lens;
  p.cu_rows = cu_rows;
  p.prefix_lens = prefix_lens;
  p.q_st = q_strides[0], p.q_sh = q_strides[1];
  p.kv_st = pool_strides[0], p.kv_sh = pool_strides[1];
  p.o_st = o_strides[0], p.o_sh = o_strides[1];
  if (lse) p.l_sh = lse_strides[0], p.l_st = lse_strides[1];
  p.G = n_groups;
  p.B = batch;
  p.total_q = total_q;
  p.Hq = heads_q;
  p.Hkv = heads_kv;
  p.group = heads_q / heads_kv;
  p.max_kv = max_kv_len;
  p.bs_shift = __builtin_ctz(block_size);
  p.num_blocks = num_blocks;
  p.causal = is_causal ? 1 : 0;
  p.scale_log2 = sm_scale * mi_fa2::kLog2e;
  int cus = 0;
  if (int rc = compute_units(&cus)) return rc;
  return launched(
      mi_fa2::launch_shared(p, dtype, cus, workspace, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
