// Paged GQA attention for trees of drafted tokens.
//
// Sequence s has q_len nodes (rows q_start .. q_start+q_len-1 of q and out);
// node i's key and value lie at position ctx - q_len + i of the sequence.  A
// node sees every key before the drafts (positions 0 .. ctx-q_len-1) and the
// nodes j whose bit is set in its row of tree_mask.  For one (sequence, kv
// head) the query rows are r = i*G + g as in attention.cu.  A row that sees
// nothing gets zeros; a key or value a row does not see never reaches it,
// whatever bits it holds.
#include "attention.cuh"
#include "common.cuh"
#include "host.h"

namespace tb {

constexpr int TREE_WORDS = 4;             // 64-bit mask words a row: at most 256 nodes
constexpr int TREE_NODES = 64 * TREE_WORDS;

struct TreeAttnArgs {
  AttnArgs a;
  const unsigned long long* mask;         // [n_rows, mask_ld], mask_w words used
  int mask_ld, mask_w;
  int n_rows;                             // rows of q, out and mask
  int max_q;                              // the grid covers max_q nodes a sequence
  int bt_w;                               // columns of a block-table row (a.bt_ld: its pitch)
};

// Sequence metadata, checked: rows inside the batch, nodes covered by the
// mask and the grid, a context the block-table row can hold.
struct TreeSeq {
  int q0, ql, ctx, base;
};
__device__ __forceinline__ bool tree_seq(const TreeAttnArgs& t, int seq, TreeSeq& s) {
  s.q0 = t.a.q_start[seq];
  s.ql = t.a.q_len[seq];
  s.ctx = t.a.ctx_len[seq];
  s.base = s.ctx - s.ql;
  return s.ql >= 0 && s.ql <= t.max_q && s.ql <= 64 * t.mask_w && s.base >= 0 && s.q0 >= 0 &&
         s.q0 <= t.n_rows - s.ql &&
         (int)(((long long)s.ctx + t.a.block_size - 1) / t.a.block_size) <= t.bt_w;
}

// ------------------------------------------------------------ any shape
//
// One warp a query row: lanes over keys for the scores (32 at a time, the row
// of q broadcast from shared memory), over the head's columns for P V, both in
// fp32 FMA, online softmax in base 2.  Serves the shapes the tensor-core kernel
// below does not (head_dim 16, blocks that are no multiple of 16 tokens).
constexpr int TS_WARPS = 4;

template <int HD>
__global__ void __launch_bounds__(TS_WARPS * 32) tree_attn_simple_kernel(const TreeAttnArgs t) {
  constexpr int CPL = (HD + 31) / 32;   // columns a lane
  __shared__ float s_q[TS_WARPS][HD];
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const AttnArgs& a = t.a;
  const int seq = blockIdx.z, kvh = blockIdx.y;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  TreeSeq s;
  if (!tree_seq(t, seq, s)) {
    if (threadIdx.x == 0) set_status(ERR_BAD_INDEX);
    return;
  }
  const int G = a.n_q_heads / a.n_kv_heads;
  const int r = blockIdx.x * TS_WARPS + warp;
  if (r >= s.ql * G) return;
  const size_t row = (size_t)s.q0 + r / G;
  const size_t col = (size_t)(kvh * G + r % G) * HD;
  for (int c = lane; c < HD; c += 32)
    s_q[warp][c] = __bfloat162float(a.q[row * a.ld_q + col + c]);
  __syncwarp();
  const int* table = a.block_tables + (size_t)seq * a.bt_ld;
  const unsigned long long* mask = t.mask + row * t.mask_ld;
  const size_t head = (size_t)a.block_size * HD;
  float o[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) o[k] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int p0 = 0; p0 < s.ctx; p0 += 32) {
    const int p = p0 + lane;
    bool seen = p < s.ctx;
    if (p >= s.base && seen) seen = (mask[(p - s.base) >> 6] >> ((p - s.base) & 63)) & 1;
    size_t off = 0;
    if (seen) {
      const int blk = table[p / a.block_size];
      if (blk < 0 || blk >= a.num_blocks) {
        set_status(ERR_BAD_INDEX);
        seen = false;
      } else {
        off = ((size_t)blk * 2 * a.n_kv_heads + kvh) * head + (size_t)(p % a.block_size) * HD;
      }
    }
    float x = -INFINITY;
    if (seen) {
      float acc = 0.f;
#pragma unroll
      for (int c = 0; c < HD; c += 8) {
        float k8[8];
        load_bf16x8(a.pool + off + c, k8);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc = fmaf(s_q[warp][c + e], k8[e], acc);
      }
      x = acc * a.scale_log2;
    }
    float mx = x;
#pragma unroll
    for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float mn = fmaxf(m, mx);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - mu);
    m = mn;
    const float pr = seen ? exp2f(x - mu) : 0.f;
    l = l * alpha + pr;
#pragma unroll
    for (int k = 0; k < CPL; ++k) o[k] *= alpha;
    unsigned todo = __ballot_sync(0xffffffffu, seen);
    while (todo) {
      const int i = __ffs(todo) - 1;
      todo &= todo - 1;
      const float pi = __shfl_sync(0xffffffffu, pr, i);
      const size_t vo = __shfl_sync(0xffffffffu, (unsigned long long)off, i) +
                        (size_t)a.n_kv_heads * head;
#pragma unroll
      for (int k = 0; k < CPL; ++k)
        if (lane + 32 * k < HD) o[k] = fmaf(pi, __bfloat162float(a.pool[vo + lane + 32 * k]), o[k]);
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < CPL; ++k)
    if (lane + 32 * k < HD)
      a.out[row * a.ld_out + col + lane + 32 * k] = __float2bfloat16_rn(o[k] * inv);
}

template <int HD>
static int tree_simple_launch(const TreeAttnArgs& t, cudaStream_t st) {
  const int rows = t.max_q * (t.a.n_q_heads / t.a.n_kv_heads);
  return launch_pdl(tree_attn_simple_kernel<HD>,
                    dim3((rows + TS_WARPS - 1) / TS_WARPS, t.a.n_kv_heads, t.a.n_seqs),
                    dim3(TS_WARPS * 32), 0, st, 1, "tree attention launch", t);
}

int tree_attention(TreeAttnArgs t, int head_dim, int max_ctx, long long ctx_total,
                   cudaStream_t st) {
  AttnArgs& a = t.a;
  if (a.n_kv_heads <= 0 || a.n_q_heads <= 0 || a.n_q_heads % a.n_kv_heads)
    return arg_err("heads: Hq % Hkv != 0");
  if (a.n_q_heads / a.n_kv_heads > 128) return arg_err("GQA group larger than 128");
  if (a.block_size <= 0 || a.num_blocks <= 0 || t.bt_w <= 0 || a.bt_ld < 0)
    return arg_err("block_size / num_blocks / block table shape");
  if (head_dim != 16 && head_dim != 64 && head_dim != 128)
    return arg_err("head_dim must be 16, 64 or 128");
  if (a.ld_q % 8 || a.ld_out % 8 || a.ld_q < a.n_q_heads * head_dim ||
      a.ld_out < a.n_q_heads * head_dim)
    return arg_err("ld_q / ld_out must be multiples of 8 and hold every head");
  if (a.n_seqs < 0 || t.n_rows < 0 || t.max_q < 0) return arg_err("n_seqs / n_rows / max_q");
  if (t.mask_w < 1 || t.mask_w > TREE_WORDS || t.mask_ld < t.mask_w)
    return arg_err("tree_mask must have 1 to 4 words a row");
  if (t.max_q > 64 * t.mask_w) return arg_err("max_q above the nodes tree_mask can name");
  if (a.n_seqs > 65535 || a.n_kv_heads > 65535) return arg_err("more than 65535 sequences or heads");
  if (a.n_seqs == 0 || t.max_q == 0 || t.n_rows == 0) return TB_OK;
  if (a.q == nullptr || a.out == nullptr || a.pool == nullptr || a.block_tables == nullptr ||
      a.q_start == nullptr || a.q_len == nullptr || a.ctx_len == nullptr || t.mask == nullptr)
    return arg_err("null pointer");
  for (const void* p : {(const void*)a.q, (const void*)a.out, (const void*)a.pool})
    if (reinterpret_cast<uintptr_t>(p) % 16) return arg_err("q / out / kv_pool must be 16-byte aligned");
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  switch (head_dim) {
    case 16: return tree_simple_launch<16>(t, st);
    case 64: return tree_simple_launch<64>(t, st);
    default: return tree_simple_launch<128>(t, st);
  }
}

}  // namespace tb

extern "C" int tb_paged_attention_tree(const void* q, int ld_q, void* out, int ld_out, int n_rows,
                                       const void* kv_pool, int num_blocks, int n_q_heads,
                                       int n_kv_heads, int head_dim, int block_size,
                                       const int* block_tables, int bt_ld, int bt_w, const int* q_start,
                                       const int* q_len, const int* ctx_len, int n_seqs,
                                       const void* tree_mask, int mask_ld, int mask_words,
                                       int max_q, int max_ctx, long long ctx_total, void* stream) {
  using namespace tb;
  TreeAttnArgs t{};
  t.a.q = static_cast<const __nv_bfloat16*>(q);
  t.a.ld_q = ld_q;
  t.a.out = static_cast<__nv_bfloat16*>(out);
  t.a.ld_out = ld_out;
  t.a.pool = static_cast<const __nv_bfloat16*>(kv_pool);
  t.a.num_blocks = num_blocks;
  t.a.n_q_heads = n_q_heads;
  t.a.n_kv_heads = n_kv_heads;
  t.a.block_size = block_size;
  t.a.block_tables = block_tables;
  t.a.bt_ld = bt_ld;
  t.bt_w = bt_w;
  t.a.q_start = q_start;
  t.a.q_len = q_len;
  t.a.ctx_len = ctx_len;
  t.a.n_seqs = n_seqs;
  t.mask = static_cast<const unsigned long long*>(tree_mask);
  t.mask_ld = mask_ld;
  t.mask_w = mask_words;
  t.n_rows = n_rows;
  t.max_q = max_q;
  return tree_attention(t, head_dim, max_ctx, ctx_total, static_cast<cudaStream_t>(stream));
}
