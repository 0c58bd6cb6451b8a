// Moves inside the paged KV pools: whole blocks (forks, defragmentation) and
// the slots of an accepted draft path.
//
// A pool of one layer is [num_blocks, 2, n_kv, bs, hd] bf16, so a block is one
// contiguous run of 2*n_kv*bs*hd elements and a token's K or V of one head a
// run of hd elements.  Every call covers all layers in one launch: the layers'
// base pointers travel as a kernel parameter (POOL_LAYERS at a time), so
// nothing has to live on the device and a captured call keeps its own copy.
//
// Both kernels only move bytes: the floor is every moved byte read once and
// written once.  Measured on a B200 (CUDA graph, inputs rotated through more than
// the L2): 200 blocks of 64 KiB in 48 layers 147 us (629 MB written, 0.27 GB of
// distinct sources read: 6.1 TB/s, 0.94 of the copy bandwidth); the accepted paths of
// 64 sequences, 162 tokens in 48 layers, 15.9 us: 65 MB in runs of 256 bytes, all that
// a pool keeps contiguous of a token and head, 4.1 TB/s.  Paths that are in place (chains)
// return before the pools after 6.8 us: the start of 3072 CTAs, each with its loads of
// lengths, path and block ids that wait for one another.  So much of the 15.9 us passes
// without a move, and the moves take what the floor allows them (9.7 us); DRAM is a
// quarter busy.  More loads in flight a thread, one wave of CTAs over several layers each,
// or fewer dependent loads before the moves did not change the total.  Leaving out the
// nodes in front of a path that moves costs the others more (a loop from a start of
// their own: 20.7 instead of 16.0 us) than it saves.
#include "common.cuh"
#include "host.h"

namespace tb {

constexpr int POOL_LAYERS = 128;
struct PoolTable {
  void* p[POOL_LAYERS];
};

// ------------------------------------------------------------- block copies

constexpr int COPY_THREADS = 256;
constexpr int COPY_UNROLL = 4;   // 16-byte pieces in flight a thread
constexpr int COPY_CHUNK = COPY_THREADS * COPY_UNROLL;   // pieces a CTA moves (16 KiB)

// CTA (pair, layer, chunk of the block).  A pair is refused (status
// BAD_INDEX, nothing written) when an id is out of range or its destination
// also is another pair's source or destination: copies run in no order.
// Every CTA of a pair reads the whole list, so all decide alike; the data
// loads are issued before the list is scanned.
__global__ void __launch_bounds__(COPY_THREADS)
    copy_blocks_kernel(const __grid_constant__ PoolTable pools, const int2* pairs, int n,
                       int num_blocks, int pieces) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const int i = blockIdx.x;
  const int2 pr = pairs[i];
  const bool range = pr.x >= 0 && pr.x < num_blocks && pr.y >= 0 && pr.y < num_blocks;
  if (range && pr.x == pr.y) {
    // onto itself: nothing to move, but a second writer of the block is refused there
    return;
  }
  if (!range) {
    if (threadIdx.x == 0) set_status(ERR_BAD_INDEX);
    return;
  }
  uint4* base = static_cast<uint4*>(pools.p[blockIdx.y]);
  const uint4* src = base + (size_t)pr.x * pieces;
  uint4* dst = base + (size_t)pr.y * pieces;
  const int c0 = blockIdx.z * COPY_CHUNK + threadIdx.x;
  uint4 v[COPY_UNROLL];
#pragma unroll
  for (int k = 0; k < COPY_UNROLL; ++k)
    if (c0 + k * COPY_THREADS < pieces) v[k] = __ldcs(src + c0 + k * COPY_THREADS);
  int clash = 0;
  for (int j = threadIdx.x; j < n; j += COPY_THREADS) {
    const int2 o = pairs[j];
    clash |= j != i && (o.x == pr.y || o.y == pr.y);
  }
  if (__syncthreads_or(clash)) {
    if (threadIdx.x == 0) set_status(ERR_BAD_INDEX);
    return;
  }
#pragma unroll
  for (int k = 0; k < COPY_UNROLL; ++k)
    if (c0 + k * COPY_THREADS < pieces) __stcs(dst + c0 + k * COPY_THREADS, v[k]);
}

// ------------------------------------------------------- accepted-path moves

constexpr int KEEP_THREADS = 256;
constexpr int KEEP_MAX = 256;     // nodes of a sequence's draft tree
constexpr int KEEP_BATCH = 8;     // moves whose loads are in flight together

struct KeepArgs {
  const int* block_tables;
  int bt_ld, bt_w;   // pitch and columns of a row
  const int *q_len, *ctx_len, *path, *n_accepted;
  int path_ld, path_w;
  int n_kv_heads, block_size, head_dim, num_blocks;
};

// CTA (sequence, layer, group of columns).  A column is one 16-byte piece of
// a token's K or V; a thread owns a column and makes the sequence's moves in
// path order, KEEP_BATCH loads before their stores.  path is strictly
// increasing with path[j] >= j, so a batch's destinations are read by no
// later move, and earlier moves of the batch have read them already.
__global__ void __launch_bounds__(KEEP_THREADS)
    keep_path_kernel(const __grid_constant__ PoolTable pools, const KeepArgs a) {
  __shared__ long long s_src[KEEP_MAX], s_dst[KEEP_MAX];   // element offsets of slot (block, token)
  __shared__ bool s_still;   // the last node stays, so (the path increases) all do
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const int seq = blockIdx.x;
  const int acc = a.n_accepted[seq], ql = a.q_len[seq], ctx = a.ctx_len[seq];
  if (acc == 0) return;
  const int* path = a.path + (size_t)seq * a.path_ld;
  const int* table = a.block_tables + (size_t)seq * a.bt_ld;
  const int base = ctx - ql;   // (used only where ctx >= ql: elsewhere it may wrap)
  int bad = acc < 0 || acc >= a.path_w || acc >= ql || ql > KEEP_MAX || ctx < ql ||
            (int)(((long long)ctx + a.block_size - 1) / a.block_size) > a.bt_w;
  if (!bad) {
    const size_t token = a.head_dim;
    const size_t block = (size_t)2 * a.n_kv_heads * a.block_size * token;
    for (int j = 1 + threadIdx.x; j <= acc; j += blockDim.x) {
      const int node = path[j];
      if (node <= (j > 1 ? path[j - 1] : 0) || node >= ql) {
        bad = 1;
        break;
      }
      const int ps = base + node, pd = base + j;
      const int bs = table[ps / a.block_size], bd = table[pd / a.block_size];
      if (bs < 0 || bs >= a.num_blocks || bd < 0 || bd >= a.num_blocks) {
        bad = 1;
        break;
      }
      if (j == acc) s_still = node == j;
      s_src[j] = (long long)(bs * block + (ps % a.block_size) * token);
      s_dst[j] = (long long)(bd * block + (pd % a.block_size) * token);
    }
  }
  if (__syncthreads_or(bad)) {   // one status, nothing moved
    if (threadIdx.x == 0) set_status(ERR_BAD_INDEX);
    return;
  }
  const int per_head = a.head_dim / 8;
  const int col = blockIdx.z * KEEP_THREADS + threadIdx.x;   // one group below KEEP_THREADS columns
  if (col >= 2 * a.n_kv_heads * per_head) return;
  __nv_bfloat16* pool = static_cast<__nv_bfloat16*>(pools.p[blockIdx.y]) +
                        (size_t)(col / per_head) * a.block_size * a.head_dim + (col % per_head) * 8;
  if (s_still) return;
  for (int j0 = 1; j0 <= acc; j0 += KEEP_BATCH) {
    uint4 v[KEEP_BATCH];
#pragma unroll
    for (int k = 0; k < KEEP_BATCH; ++k)
      if (j0 + k <= acc) v[k] = *reinterpret_cast<const uint4*>(pool + s_src[j0 + k]);
#pragma unroll
    for (int k = 0; k < KEEP_BATCH; ++k)
      if (j0 + k <= acc) *reinterpret_cast<uint4*>(pool + s_dst[j0 + k]) = v[k];
  }
}

static int check_pools(const void* const* pools, int n_layers, int num_blocks, int n_kv_heads,
                       int block_size, int head_dim) {
  if (n_layers < 0 || num_blocks <= 0 || n_kv_heads <= 0 || block_size <= 0 || head_dim <= 0 ||
      head_dim % 8)
    return arg_err("pool shape: head_dim must be a multiple of 8, the other sizes positive");
  if (n_layers > 0 && pools == nullptr) return arg_err("pools_h is NULL");
  for (int l = 0; l < n_layers; ++l)
    if (pools[l] == nullptr || reinterpret_cast<uintptr_t>(pools[l]) % 16)
      return arg_err("every layer's pool must be a 16-byte aligned pointer");
  return TB_OK;
}

static PoolTable pool_table(const void* const* pools, int n) {
  PoolTable t{};
  for (int l = 0; l < n; ++l) t.p[l] = const_cast<void*>(pools[l]);
  return t;
}

int copy_blocks_launch(const void* const* pools, int n_layers, int num_blocks, int n_kv_heads,
                       int block_size, int head_dim, const int* pairs, int n, cudaStream_t st) {
  if (int rc = check_pools(pools, n_layers, num_blocks, n_kv_heads, block_size, head_dim)) return rc;
  if (n < 0) return arg_err("n_pairs");
  if (n == 0 || n_layers == 0) return TB_OK;
  if (pairs == nullptr || reinterpret_cast<uintptr_t>(pairs) % 8)
    return arg_err("pairs must be an 8-byte aligned pointer");
  const size_t pieces = (size_t)2 * n_kv_heads * block_size * (head_dim / 8);
  const size_t chunks = (pieces + COPY_CHUNK - 1) / COPY_CHUNK;
  if (chunks > 65535) return arg_err("a block of 1 GiB or more");
  for (int l0 = 0; l0 < n_layers; l0 += POOL_LAYERS) {
    const int nl = n_layers - l0 < POOL_LAYERS ? n_layers - l0 : POOL_LAYERS;
    const int rc = launch_pdl(copy_blocks_kernel, dim3(n, nl, (unsigned)chunks), dim3(COPY_THREADS),
                              0, st, 1, "copy blocks launch", pool_table(pools + l0, nl),
                              reinterpret_cast<const int2*>(pairs), n, num_blocks, (int)pieces);
    if (rc) return rc;
  }
  return TB_OK;
}

int keep_path_launch(const void* const* pools, int n_layers, KeepArgs a, int n_seqs,
                     cudaStream_t st) {
  if (int rc = check_pools(pools, n_layers, a.num_blocks, a.n_kv_heads, a.block_size, a.head_dim))
    return rc;
  if (n_seqs < 0 || a.bt_ld < 0 || a.bt_w <= 0 || a.path_w <= 0 || a.path_ld < a.path_w)
    return arg_err("n_seqs / bt_ld / path width");
  if (n_seqs == 0 || n_layers == 0) return TB_OK;
  if (a.block_tables == nullptr || a.q_len == nullptr || a.ctx_len == nullptr ||
      a.path == nullptr || a.n_accepted == nullptr)
    return arg_err("null pointer");
  const int cols = 2 * a.n_kv_heads * (a.head_dim / 8);
  const int threads = cols < KEEP_THREADS ? (cols + 31) / 32 * 32 : KEEP_THREADS;
  const int groups = (cols + KEEP_THREADS - 1) / KEEP_THREADS;
  if (groups > 65535) return arg_err("too many kv heads");
  for (int l0 = 0; l0 < n_layers; l0 += POOL_LAYERS) {
    const int nl = n_layers - l0 < POOL_LAYERS ? n_layers - l0 : POOL_LAYERS;
    const int rc = launch_pdl(keep_path_kernel, dim3(n_seqs, nl, groups), dim3(threads), 0, st, 1,
                              "keep path launch", pool_table(pools + l0, nl), a);
    if (rc) return rc;
  }
  return TB_OK;
}

}  // namespace tb

extern "C" {

int tb_copy_kv_blocks(const void* const* pools_h, int n_layers, int num_blocks, int n_kv_heads,
                      int block_size, int head_dim, const int* pairs, int n_pairs, void* stream) {
  return tb::copy_blocks_launch(pools_h, n_layers, num_blocks, n_kv_heads, block_size, head_dim,
                                pairs, n_pairs, static_cast<cudaStream_t>(stream));
}

int tb_keep_kv_path(const void* const* pools_h, int n_layers, int num_blocks, int n_kv_heads,
                    int block_size, int head_dim, const int* block_tables, int bt_ld, int bt_w,
                    const int* q_len, const int* ctx_len, const int* path, int path_ld, int path_w,
                    const int* n_accepted, int n_seqs, void* stream) {
  tb::KeepArgs a{};
  a.block_tables = block_tables;
  a.bt_ld = bt_ld;
  a.bt_w = bt_w;
  a.q_len = q_len;
  a.ctx_len = ctx_len;
  a.path = path;
  a.n_accepted = n_accepted;
  a.path_ld = path_ld;
  a.path_w = path_w;
  a.n_kv_heads = n_kv_heads;
  a.block_size = block_size;
  a.head_dim = head_dim;
  a.num_blocks = num_blocks;
  return tb::keep_path_launch(pools_h, n_layers, a, n_seqs, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
