// Copies within the paged KV cache: whole or partly filled pages (forks,
// copies on write, compaction of the pool) and the rows of an accepted path of
// drafted tokens.  No counterpart in the reference, whose pages only ever move
// by recomputing them (engine/block_manager.py:58-120).
//
// The pool is `slabs` arrays (layers x K/V) of [num_blocks, block_size, row]
// bytes; a call moves the same pages or rows in every one of them, in one
// launch.  Bound by HBM: every moved byte is read and written once.
#include <algorithm>

#include "nq_device.hpp"

namespace nq {
namespace {

// ---------------------------------------------------------------- pages
// One workgroup copies kChunk bytes of one page of one slab, four 16-byte
// loads per lane in flight.  48 pages of 256 tokens in 16 layers (8 kv heads, D =
// 128, bf16; 1.6 GB moved) 307 us, 5.2 TB/s, what a plain copy of that size
// reaches; two partly filled pages 10 us, 5.5 TB/s (some of it from the L2s).
constexpr int kCopyThreads = 256, kCopyUnroll = 4;
constexpr int kChunk = kCopyThreads * kCopyUnroll * 16;

__global__ __launch_bounds__(kCopyThreads) void copy_blocks_kernel(uint8_t *pool, const int32_t *src, const int32_t *dst,
                                                                   const int32_t *tokens, int64_t num_blocks,
                                                                   int block_size, int64_t row_bytes, int chunks) {
  // chunk fastest, then slab, then pair
  const int64_t unit = blockIdx.x;
  const int chunk = static_cast<int>(unit % chunks);
  const int pair = static_cast<int>(unit / chunks);
  const int64_t slab = blockIdx.y;
  const int32_t from = ld_const(src + pair), to = ld_const(dst + pair);
  if (from < 0 || to < 0 || from >= num_blocks || to >= num_blocks || from == to) return;
  const int rows = tokens ? min(max(ld_const(tokens + pair), 0), block_size) : block_size;
  const int64_t bytes = rows * row_bytes, page = block_size * row_bytes;
  const uint8_t *s = pool + (slab * num_blocks + from) * page;
  uint8_t *d = pool + (slab * num_blocks + to) * page;
  const int64_t at = static_cast<int64_t>(chunk) * kChunk + threadIdx.x * 16;
  u32x4 x[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (at + u * kCopyThreads * 16 < bytes) x[u] = load16(s + at + u * kCopyThreads * 16);
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (at + u * kCopyThreads * 16 < bytes) store16(d + at + u * kCopyThreads * 16, x[u]);
}

// The scales of pages (of a cache with a scale for each block of tokens and head):
// `per` floats a page and slab, one per thread.
__global__ __launch_bounds__(kCopyThreads) void copy_scales_kernel(float *pool, const int32_t *src, const int32_t *dst,
                                                                   int64_t num_blocks, int per, int parts) {
  const int pair = static_cast<int>(blockIdx.x / parts);
  const int i = static_cast<int>(blockIdx.x % parts) * kCopyThreads + threadIdx.x;
  const int32_t from = ld_const(src + pair), to = ld_const(dst + pair);
  if (from < 0 || to < 0 || from >= num_blocks || to >= num_blocks || from == to || i >= per) return;
  float *slab = pool + static_cast<int64_t>(blockIdx.y) * num_blocks * per + i;
  slab[to * static_cast<int64_t>(per)] = slab[from * static_cast<int64_t>(per)];
}

// ---------------------------------------------------------------- trees
// Every wave walks its sequence's tree itself (nodes lane, lane + 64, ... in
// registers, one ballot per 64 nodes and step) and then moves its columns.  A
// node comes after its parent, so path[r] rises and path[r] >= r: in the order
// r = 1, 2, ... no row is read after it was written.  Walking once per wave
// costs no launch and no wait for another workgroup's path: 4.5 us for one
// sequence, 8 for 64 (a call is 12.5, the host's work for it).
constexpr int kMaxNodes = 256, kNodeRegs = kMaxNodes / 64;
constexpr int kCommitThreads = 256, kRowUnroll = 8;

struct CommitArgs {
  uint8_t *pool;
  int64_t num_blocks, row_bytes;
  int block_size, slabs;
  const int32_t *block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t *cu_q, *cu_k;
  int total_q, max_q;
  const int32_t *parents;
  const int64_t *tokens, *targets;
  int32_t *path;  // [num_seqs, max_q]
  int32_t *count;
  int64_t *next;
  int given;  // path and count are inputs
};

__global__ __launch_bounds__(kCommitThreads) void commit_tree_kernel(const CommitArgs a) {
  const int s = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int q0 = max(0, min(ld_const(a.cu_q + s), a.total_q));
  const int n = max(0, min(min(ld_const(a.cu_q + s + 1), a.total_q) - q0, a.max_q));
  const int C = ld_const(a.cu_k + s + 1) - ld_const(a.cu_k + s) - n;  // tokens before the tree
  int path[kNodeRegs];  // lane l: path[64 i + l]
  int len = 0;
  if (a.given) {
    const int want = min(max(ld_const(a.count + s), 0), n);
#pragma unroll
    for (int i = 0; i < kNodeRegs; ++i) {
      const int r = 64 * i + lane;
      path[i] = r < want ? a.path[static_cast<int64_t>(s) * a.max_q + r] : -1;
    }
    // up to the first entry that does not rise or names no node
    uint64_t wrong = 0;
    len = want;
    int before = -1;
#pragma unroll
    for (int i = 0; i < kNodeRegs; ++i) {
      const int up = __shfl_up(path[i], 1);
      const int prev = lane == 0 ? before : up;
      wrong = __builtin_amdgcn_ballot_w64(64 * i + lane < want && (path[i] <= prev || path[i] >= n));
      if (wrong != 0) len = min(len, 64 * i + static_cast<int>(__builtin_ctzll(wrong)));
      before = __builtin_amdgcn_readlane(path[i], 63);
    }
  } else {
    int parent[kNodeRegs];
    int64_t token[kNodeRegs], target[kNodeRegs];
#pragma unroll
    for (int i = 0; i < kNodeRegs; ++i) {
      const int v = 64 * i + lane;
      path[i] = -1;
      parent[i] = -1;
      token[i] = target[i] = 0;
      if (v < n) {
        parent[i] = a.parents[q0 + v];
        token[i] = a.tokens[q0 + v];
        target[i] = a.targets[q0 + v];
      }
    }
    int cur = 0;
    int64_t want = -1;
    while (cur >= 0 && cur < n) {
      int child = -1;
#pragma unroll
      for (int i = 0; i < kNodeRegs; ++i) {
        if (len >> 6 == i && lane == (len & 63)) path[i] = cur;
        if (cur >> 6 == i) {
          const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(target[i]), cur & 63);
          const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(target[i] >> 32), cur & 63);
          want = static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
        }
      }
      ++len;
#pragma unroll
      for (int i = kNodeRegs - 1; i >= 0; --i) {
        const int v = 64 * i + lane;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(v < n && v > cur && parent[i] == cur && token[i] == want);
        if (hit != 0) child = 64 * i + static_cast<int>(__builtin_ctzll(hit));
      }
      cur = child;
    }
    if (blockIdx.x == 0 && threadIdx.x < 64) {
#pragma unroll
      for (int i = 0; i < kNodeRegs; ++i) {
        const int r = 64 * i + lane;
        if (r < a.max_q) a.path[static_cast<int64_t>(s) * a.max_q + r] = path[i];
      }
      if (lane == 0) {
        a.count[s] = len;
        a.next[s] = want;
      }
    }
  }
  // Cache rows of the path's nodes and of their places (lane l: path[64 i + l]).
  const int32_t *bt = a.block_tables + static_cast<int64_t>(s) * a.bt_stride;
  auto row_at = [&](int p) -> int64_t {
    if (p < 0) return -1;
    const int e = p / a.block_size;
    if (e >= a.max_blocks) return -1;
    const int blk = bt[e];
    return blk < 0 || blk >= a.num_blocks ? -1 : static_cast<int64_t>(blk) * a.block_size + p % a.block_size;
  };
  int64_t from[kNodeRegs], to[kNodeRegs];
#pragma unroll
  for (int i = 0; i < kNodeRegs; ++i) {
    const int r = 64 * i + lane;
    from[i] = to[i] = -1;
    if (r < len && path[i] != r && C >= 0) {
      from[i] = row_at(C + path[i]);
      to[i] = row_at(C + r);
      if (to[i] < 0) from[i] = -1;
    }
  }
  const int64_t cols = a.row_bytes / 16;
  const int64_t col = static_cast<int64_t>(blockIdx.x) * kCommitThreads + threadIdx.x;
  const bool live = col < cols * a.slabs;
  const int64_t slab = live ? col / cols : 0;
  uint8_t *base = a.pool + slab * a.num_blocks * a.block_size * a.row_bytes + (live ? col % cols : 0) * 16;
  auto lane64 = [](int64_t v, int l) -> int64_t {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), l);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), l);
    return static_cast<int64_t>((static_cast<uint64_t>(hi) << 32) | lo);
  };
#pragma unroll
  for (int i = 0; i < kNodeRegs; ++i) {
    uint64_t todo = __builtin_amdgcn_ballot_w64(from[i] >= 0);
    while (todo != 0) {
      u32x4 x[kRowUnroll];
      int64_t d[kRowUnroll];
#pragma unroll
      for (int u = 0; u < kRowUnroll; ++u) {
        d[u] = -1;
        if (todo != 0) {
          const int l = static_cast<int>(__builtin_ctzll(todo));
          todo &= todo - 1;
          d[u] = lane64(to[i], l);
          if (live) x[u] = load16(base + lane64(from[i], l) * a.row_bytes);
        }
      }
#pragma unroll
      for (int u = 0; u < kRowUnroll; ++u)
        if (d[u] >= 0 && live) store16(base + d[u] * a.row_bytes, x[u]);
    }
  }
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_copy_kv_blocks(void *kv_cache, int64_t num_slabs, int64_t num_blocks, int block_size,
                                 int64_t row_bytes, const int32_t *src_blocks, const int32_t *dst_blocks,
                                 const int32_t *num_tokens, int64_t num_pairs, void *stream) {
  if (num_pairs < 0 || num_slabs < 0 || num_blocks < 0 || block_size <= 0 || row_bytes <= 0)
    return fail(NQ_EINVAL, "copy_kv_blocks: bad sizes");
  if (num_pairs == 0 || num_slabs == 0 || num_blocks == 0) return NQ_OK;
  if (!kv_cache || !src_blocks || !dst_blocks) return fail(NQ_EINVAL, "copy_kv_blocks: null pointer");
  if (row_bytes % 16 || !aligned(kv_cache, 16))
    return fail(NQ_EINVAL, "copy_kv_blocks: cache rows of %lld bytes must be 16-byte aligned", (long long)row_bytes);
  if (num_slabs > 65535) return fail(NQ_EUNSUPPORTED, "copy_kv_blocks: %lld slabs > 65535", (long long)num_slabs);
  const int64_t chunks = (block_size * row_bytes + kChunk - 1) / kChunk;
  if (chunks * num_pairs > 0x7fffffff)
    return fail(NQ_EINVAL, "copy_kv_blocks: %lld pages of %lld bytes", (long long)num_pairs,
                (long long)(block_size * row_bytes));
  copy_blocks_kernel<<<dim3(static_cast<unsigned>(chunks * num_pairs), static_cast<unsigned>(num_slabs)), kCopyThreads,
                       0, static_cast<hipStream_t>(stream)>>>(
      static_cast<uint8_t *>(kv_cache), src_blocks, dst_blocks, num_tokens, num_blocks, block_size, row_bytes,
      static_cast<int>(chunks));
  return check_launch("copy_kv_blocks");
}

extern "C" int nq_copy_kv_scales(float *kv_scales, int64_t num_slabs, int64_t num_blocks, int scales_per_block,
                                 const int32_t *src_blocks, const int32_t *dst_blocks, int64_t num_pairs, void *stream) {
  if (num_pairs < 0 || num_slabs < 0 || num_blocks < 0 || scales_per_block <= 0)
    return fail(NQ_EINVAL, "copy_kv_scales: bad sizes");
  if (num_pairs == 0 || num_slabs == 0 || num_blocks == 0) return NQ_OK;
  if (!kv_scales || !src_blocks || !dst_blocks) return fail(NQ_EINVAL, "copy_kv_scales: null pointer");
  if (num_slabs > 65535) return fail(NQ_EUNSUPPORTED, "copy_kv_scales: %lld slabs > 65535", (long long)num_slabs);
  const int64_t parts = (static_cast<int64_t>(scales_per_block) + kCopyThreads - 1) / kCopyThreads;
  if (parts * num_pairs > 0x7fffffff) return fail(NQ_EINVAL, "copy_kv_scales: %lld pages", (long long)num_pairs);
  copy_scales_kernel<<<dim3(static_cast<unsigned>(parts * num_pairs), static_cast<unsigned>(num_slabs)), kCopyThreads, 0,
                       static_cast<hipStream_t>(stream)>>>(kv_scales, src_blocks, dst_blocks, num_blocks,
                                                           scales_per_block, static_cast<int>(parts));
  return check_launch("copy_kv_scales");
}

extern "C" int nq_commit_tree(void *kv_cache, int64_t num_slabs, int64_t num_blocks, int block_size, int64_t row_bytes,
                              const int32_t *block_tables, int64_t bt_stride, int max_blocks_per_seq,
                              const int32_t *cu_seqlens_q, const int32_t *cu_seqlens_k, int num_seqs, int64_t total_q,
                              int max_seqlen_q, const int32_t *parents, const int64_t *tokens,
                              const int64_t *target_tokens, int32_t *path, int32_t *num_accepted, int64_t *next_tokens,
                              void *stream) {
  if (num_seqs < 0 || num_seqs > 65535 || num_slabs < 0 || num_blocks < 0 || block_size <= 0 || row_bytes <= 0 ||
      total_q < 0 || total_q > 0x7fffffff || max_seqlen_q < 0)
    return fail(NQ_EINVAL, "commit_tree: bad sizes");
  if (max_seqlen_q > kMaxNodes)
    return fail(NQ_EUNSUPPORTED, "commit_tree: trees of %d nodes (at most %d)", max_seqlen_q, kMaxNodes);
  if (num_seqs == 0) return NQ_OK;
  if (!block_tables || !cu_seqlens_q || !cu_seqlens_k || (max_seqlen_q > 0 && !path) || !num_accepted ||
      (num_slabs > 0 && num_blocks > 0 && !kv_cache))
    return fail(NQ_EINVAL, "commit_tree: null pointer");
  if (next_tokens ? total_q > 0 && (!parents || !tokens || !target_tokens) : parents || tokens || target_tokens)
    return fail(NQ_EINVAL, "commit_tree: null parents, tokens, target_tokens or next_tokens");
  if (max_blocks_per_seq < 0 || bt_stride < max_blocks_per_seq) return fail(NQ_EINVAL, "commit_tree: block table width");
  if (row_bytes % 16 || !aligned(kv_cache, 16))
    return fail(NQ_EINVAL, "commit_tree: cache rows of %lld bytes must be 16-byte aligned", (long long)row_bytes);
  CommitArgs a{};
  a.pool = static_cast<uint8_t *>(kv_cache);
  a.num_blocks = num_blocks;
  a.row_bytes = row_bytes;
  a.block_size = block_size;
  a.slabs = num_blocks > 0 ? static_cast<int>(std::min<int64_t>(num_slabs, 0x7fffffff)) : 0;
  a.block_tables = block_tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks_per_seq;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.total_q = static_cast<int>(total_q);
  a.max_q = max_seqlen_q;
  a.parents = parents;
  a.tokens = tokens;
  a.targets = target_tokens;
  a.path = path;
  a.count = num_accepted;
  a.next = next_tokens;
  a.given = next_tokens == nullptr;
  const int64_t units = std::max<int64_t>(1, (row_bytes / 16 * a.slabs + kCommitThreads - 1) / kCommitThreads);
  if (units > 0x7fffffff) return fail(NQ_EINVAL, "commit_tree: %lld columns", (long long)units);
  commit_tree_kernel<<<dim3(static_cast<unsigned>(units), num_seqs), kCommitThreads, 0,
                       static_cast<hipStream_t>(stream)>>>(a);
  return check_launch("commit_tree");
}
