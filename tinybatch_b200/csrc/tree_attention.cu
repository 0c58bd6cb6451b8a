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
  bool by_length;                         // blockIdx.z-th longest sequence instead of number blockIdx.z
  int group;                              // G = n_q_heads / n_kv_heads
  unsigned group_magic;                   // ceil(2^32 / G): r / G = umulhi(r, magic) for r < 2^16, G > 1
  int log_splits;                         // log2 C
  int bt_w;                               // columns of a block-table row (a.bt_ld: its pitch)
};

// Sequence metadata, checked: rows inside the batch, nodes covered by the
// mask and the grid, a context the block-table row can hold.
struct TreeSeq {
  int q0, ql, ctx, base;
};
__device__ __forceinline__ int div_group(const TreeAttnArgs& t, int r) {
  return t.group == 1 ? r : (int)__umulhi((unsigned)r, t.group_magic);
}
__device__ __forceinline__ bool tree_seq(const TreeAttnArgs& t, int seq, TreeSeq& s) {
  s.q0 = t.a.q_start[seq];
  s.ql = t.a.q_len[seq];
  s.ctx = t.a.ctx_len[seq];
  s.base = s.ctx - s.ql;
  // (the lengths compared, not their difference: it may wrap)
  if (s.ql == 0) return true;      // takes part in nothing: the rest may be anything
  return s.ql > 0 && s.ql <= t.max_q && s.ql <= 64 * t.mask_w && s.ctx >= s.ql && s.q0 >= 0 &&
         s.q0 <= t.n_rows - s.ql &&
         s.ctx <= (long long)t.bt_w * t.a.block_size && s.ctx <= (1 << 30);
}

// ------------------------------------------------------------ short heads
//
// One warp a query row: lanes over keys for the scores (32 at a time, the row
// of q broadcast from shared memory), over the head's columns for P V, both in
// fp32 FMA, online softmax in base 2.  Serves head_dim 16, whose rows are too
// short for the tensor-core kernel below.
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
  bool lost = false;      // a block id out of range: the sequence is left out
  for (int p0 = 0; p0 < s.ctx; p0 += 32) {
    const int p = p0 + lane;
    bool seen = p < s.ctx;
    if (p >= s.base && seen) seen = (mask[(p - s.base) >> 6] >> ((p - s.base) & 63)) & 1;
    size_t off = 0;
    if (p < s.ctx) {
      const int blk = table[p / a.block_size];
      if (blk < 0 || blk >= a.num_blocks) {
        lost = true;
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
  if (__any_sync(0xffffffffu, lost)) {
    if (lane == 0) set_status(ERR_BAD_INDEX);
    return;
  }
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

// -------------------------------------------------------------- tensor cores
//
// One CTA per (row tile of 128 query rows, kv head, sequence) and split of its
// context; the splits of a row tile form a cluster of C CTAs (1 to 8).  S = Q K^T
// and O += P V run on tcgen05 (M = 128 rows, tiles of 64 keys) with S, P and O in
// TMEM:
//   warps 0-3  softmax: one query row a thread (TMEM lane = row); warps whose
//              rows do not exist stay out
//   warp 4     loads.  Block sizes that are multiples of 16: every 16 tokens of K,
//              and of V, are one TMA box {64 columns, 8 tokens, halves, 2} of a 4-d
//              view of the pool (4 KiB at hd 128, all that a block keeps
//              contiguous), landing as [8-token group][half][8][128 B] with the
//              128-byte swizzle: K is a K-major operand and V an MN-major one.  Four
//              lanes issue a tile's boxes.  Other block sizes: 16-byte cp.async
//              pieces into the same layout, every key looking up its block (1.25 to 2
//              times as long: blocks of 8 take 10 / 89 / 69 / 322 us where blocks of
//              16 take 8 / 59 / 48 / 158 on the cases below, the lone one first).  K
//              and V have rings of their own: a K stage is free once its S is done,
//              before the V that came with it
//   warp 5     MMA issue.  P (bf16) has two buffers of its own in TMEM, so S of the
//              next tile follows as soon as the softmax has S in registers and is
//              there when it has written P
// P is rounded to bf16 because the MMA takes bf16 for both operands, as in the decode
// and prefill kernels; its sum is taken of the unrounded weights, in fp32.  The output's
// error against 64 bits is 0.0021-0.0025 relative where rounding the output alone
// gives 0.0017; a second MMA with P's rest would half again lengthen the MMA work.
// O is accumulated in TMEM; a row's exponent reference moves only when its
// maximum has grown by more than TT_RESCALE (log2 units), as in the prefill kernel.
// Two CTAs an SM: one's chain S -> softmax -> P V, its start and its end hide
// behind the other's loads.
//
// Measured on a B200 (CUDA graph, inputs rotated through more than the L2): 32
// chains of 6 drafts over 500-4000 tokens (40/8 heads of 128) 58.7 us, 5.2 TB/s or
// 0.80 of the measured copy bandwidth; 16 trees of 25 over 300-6000 tokens 48.4 us,
// 0.61 of it (what is missing: ~2.5 us before a CTA's first tile, 4-5 us of merge over
// the cluster with the wait for its members, the tail of the ragged batch); 4 trees of
// 64 over 12-20 thousand tokens, 512 rows a kv head, 155-158 us in a burst, 873-857
// TFLOP/s or 0.53-0.52 of the measured bf16 peak (182 us, 744 TFLOP/s or 0.55 of the
// sustained peak, where seconds of it bring the power cap and 1.66 GHz): there the softmax's chain of
// dependent instructions bounds it (tensor pipe 52% busy, exponentials 49%).  A lone
// short request takes 7.5-7.9 us: launch, lengths, block ids, K, S, softmax, P V and
// the store one after another.  At the 128 registers a thread 10 words spill at
// head_dim 128 (7 at 64); with more registers a CTA waits for an empty SM.
// Tried and dropped: 16-byte cp.async for all loads (one warp issues 9 B a cycle: 94
// instead of 64 us for the trees), two threads a row (the exchange of maxima costs what
// the shorter softmax saves), K and V boxes issued together (K waits for V's stage).
//
// Tiles that hold drafts (or places past the context) apply the mask to S and
// clean V in shared memory before P V: rows past the context become zero (a
// block's rest may hold anything, and 0 * NaN is NaN), and so do non-finite
// elements of draft nodes, which the epilogue adds back to the rows that see
// them.
//
// With C > 1 the CTAs of a cluster exchange (reference, sum, O) through their
// shared memory and each merges 1/C of the rows, in split order: no workspace, no
// counters, nothing shared between calls.
constexpr int TT_ROWS = 128;
constexpr int TT_KEYS = 64;
constexpr int TT_THREADS = 192;
constexpr float TT_RESCALE = 8.f;
constexpr int TT_MAX_SPLITS = 8;
// What a CTA found; the members of a cluster merge theirs.
constexpr int TT_NONFINITE = 1;   // a draft's V has non-finite elements
constexpr int TT_LOST = 2;        // a block id is out of range: the sequence is left out

// Shared memory of a CTA: Q (only the warps' rows that exist: the MMA reads 128
// rows whatever they hold, the others' results are never looked at), then as many
// stages of K and of V as fit half an SM.
template <int HD>
struct TreeTcLayout {
  static constexpr int HALVES = HD / 64;
  static constexpr int GROUP = HALVES * 1024;          // 8 tokens of K (or V)
  static constexpr int BOX = 2 * GROUP;                // 16 tokens
  static constexpr int STAGE = TT_KEYS / 8 * GROUP;
  static constexpr int MAX_STAGES = HD == 128 ? 3 : 6; // of K, of V
  static constexpr int DATA = 112 * 1024;              // Q and the rings; then the merge:
  static constexpr int OFF_ML = DATA - 4096;           // (reference, sum) of the splits' rows
  static constexpr int OFF_OUT = DATA - 2048;          // rows' places in out
  static constexpr int OFF_BAR = DATA;
  static constexpr int N_BARS = 4 * MAX_STAGES + 7;
  static constexpr int SMEM = OFF_BAR + 512 + 512;     // barriers; alignment slack
  static constexpr uint32_t COL_P = TT_KEYS;           // two buffers of TT_KEYS / 2 columns
  static constexpr uint32_t COL_O = 2 * TT_KEYS;
  static constexpr uint32_t TMEM_COLS = 256;
  __device__ static constexpr int q_half(int act) { return act * 4096; }   // 32 rows a warp
  __device__ static constexpr int stages(int act) { return (DATA - HALVES * q_half(act)) / STAGE; }
  __device__ static constexpr int v_stages(int act) {
    return stages(act) / 2 < MAX_STAGES ? stages(act) / 2 : MAX_STAGES;
  }
  __device__ static constexpr int k_stages(int act) {
    return stages(act) - v_stages(act) < MAX_STAGES ? stages(act) - v_stages(act) : MAX_STAGES;
  }
  static_assert((TT_ROWS + 2 * TT_MAX_SPLITS) * HD * 4 <= OFF_ML, "merged rows over Q and the rings");
  static_assert((TT_ROWS + TT_MAX_SPLITS) * 8 <= OFF_OUT - OFF_ML && TT_ROWS * 8 <= DATA - OFF_OUT,
                "merge tables");
  static_assert(N_BARS * 8 + 12 <= 512, "barrier area");
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two CTAs an SM");
  static_assert(2 * TT_KEYS + HD <= 256, "TMEM: S, two P buffers and O in half of it");
};

// Position in a ring of n stages; `phase` flips with every lap.
struct RingPos {
  int st = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++st == n) st = 0, phase ^= 1;
  }
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int x3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %3, %3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(x3)
      : "memory");
}

// K-major 128-byte-swizzled operand whose 8-row atoms lie sbo bytes apart.
__device__ __forceinline__ uint64_t sw128_k_desc(uint32_t smem_addr, uint32_t sbo) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | (uint64_t)1u << 16 | (uint64_t)(sbo >> 4) << 32 |
         (uint64_t)1u << 46 | (uint64_t)2u << 61;
}

__device__ __forceinline__ void st_cluster_f2(uint32_t addr, float x, float y) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(addr), "f"(x), "f"(y) : "memory");
}
__device__ __forceinline__ void red_cluster_or(uint32_t addr, uint32_t x) {
  asm volatile("red.relaxed.cluster.shared::cluster.or.b32 [%0], %1;" ::"r"(addr), "r"(x) : "memory");
}

// True in one lane of the (converged) warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// Bits of a word whose bf16 halves are infinite or NaN (those halves all ones).
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  return ((w & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u) |
         ((w & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u);
}

// Which of the keys k0 .. k0+63 a row sees (base: first draft's position).  m0: its
// first mask word; the others (trees of more than 64 nodes) are read when needed.
__device__ __forceinline__ unsigned long long tree_window(const unsigned long long* mask, int words,
                                                          unsigned long long m0, int k0, int base,
                                                          int ctx) {
  const int d = k0 - base;
  unsigned long long w;
  if (d <= -64) {
    w = ~0ull;
  } else if (d < 0) {
    w = ((1ull << -d) - 1) | (m0 << -d);
  } else {
    const int k = d >> 6, o = d & 63;
    const unsigned long long lo = k == 0 ? m0 : k < words ? mask[k] : 0ull;
    w = lo >> o;
    if (o && k + 1 < words) w |= mask[k + 1] << (64 - o);
  }
  const int left = ctx - k0;
  if (left < 64) w &= left > 0 ? (1ull << left) - 1 : 0ull;
  return w;
}

// Adds to a finished output row the non-finite values of the draft nodes it
// sees (their products were left out of P V).  Rare.
template <int HD>
__device__ __forceinline__ void add_nonfinite(const TreeAttnArgs& t, const int* table, int kvh,
                                              size_t row, const TreeSeq& s, __nv_bfloat16* dst) {
  const AttnArgs& a = t.a;
#pragma unroll 1
  for (int j = 0; j < s.ql; ++j) {
    if (!((t.mask[row * t.mask_ld + (j >> 6)] >> (j & 63)) & 1)) continue;
    const int p = s.base + j;
    const int blk = table[p / a.block_size];
    if (blk < 0 || blk >= a.num_blocks) continue;
    const __nv_bfloat16* src =
        a.pool + (((size_t)blk * 2 + 1) * a.n_kv_heads + kvh) * a.block_size * HD +
        (size_t)(p % a.block_size) * HD;
#pragma unroll 1
    for (int c = 0; c < HD; ++c) {
      const float x = __bfloat162float(src[c]);
      if (!isfinite(x)) dst[c] = __float2bfloat16_rn(__bfloat162float(dst[c]) + x);
    }
  }
}

// Every thread of a cluster arrives and waits; nothing is published.
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile(
      "barrier.cluster.arrive.relaxed.aligned;\n\t"
      "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The rows a CTA owns: out = sum_z w_z O_z / sum_z w_z l_z, w_z = 2^(ref_z - max ref).
template <int HD, int C>
__device__ __forceinline__ void merge_rows(const uint8_t* smem, const float2* s_ml,
                                           const size_t* s_out, __nv_bfloat16* out, int per,
                                           int pitch, int n) {
  constexpr int LPR = HD / 4;             // lanes a row, four columns each
  constexpr int RPP = TT_THREADS / LPR;   // rows a pass
  const float* so = reinterpret_cast<const float*>(smem);
  const int c4 = threadIdx.x % LPR;
#pragma unroll (8 / C)
  for (int i = threadIdx.x / LPR; i < n; i += RPP) {
    float2 ml[C];
    float4 o[C];
    float M = -INFINITY, sum = 0.f;
#pragma unroll
    for (int z = 0; z < C; ++z) {
      ml[z] = s_ml[z * per + i];
      o[z] = *reinterpret_cast<const float4*>(so + ((z * LPR + c4) * pitch + i) * 4);
      M = fmaxf(M, ml[z].x);
    }
    const float mu = M == -INFINITY ? 0.f : M;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int z = 0; z < C; ++z) {
      const float w = ex2_approx(ml[z].x - mu);   // 0 for a split that saw nothing
      sum += w * ml[z].y;
      acc.x += w * o[z].x, acc.y += w * o[z].y, acc.z += w * o[z].z, acc.w += w * o[z].w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 v;
    v.x = pack_bf16x2(acc.x * inv, acc.y * inv);
    v.y = pack_bf16x2(acc.z * inv, acc.w * inv);
    *reinterpret_cast<uint2*>(out + s_out[i] + c4 * 4) = v;
  }
}

// (at most 128 registers: four warps of each scheduler's, so that a CTA can follow
// another as soon as it ends.  Six warps of 168 fitted twice, but with the four that
// TMEM ties to their schedulers a new CTA then waited for an empty SM)
template <int HD, bool TMA>
__global__ void __launch_bounds__(256, 2)
    tree_attn_tc_kernel(const __grid_constant__ CUtensorMap map, const TreeAttnArgs t,
                        const int row_tiles) {
  using L = TreeTcLayout<HD>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = align_smem_1024(smem_raw);
  float2* s_ml = reinterpret_cast<float2*>(smem + L::OFF_ML);
  size_t* s_out = reinterpret_cast<size_t*>(smem + L::OFF_OUT);
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_empty = k_full + L::MAX_STAGES;
  uint64_t* v_full = k_empty + L::MAX_STAGES;
  uint64_t* v_empty = v_full + L::MAX_STAGES;
  uint64_t* s_full = v_empty + L::MAX_STAGES;
  uint64_t* s_free = s_full + 1;                                    // S is in registers
  uint64_t* p_full = s_full + 2;                                    // [2]
  uint64_t* pv_done = p_full + 2;                                   // [2]
  uint64_t* q_full = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
  int* s_bad = reinterpret_cast<int*>(tmem_slot + 1);   // TT_NONFINITE, TT_LOST
  int* s_seq = s_bad + 1;

  if (smem - smem_raw > 512) {   // (dynamic shared memory starts 1 KiB aligned)
    pdl_wait();
    set_status(ERR_BAD_INDEX);
    return;
  }
  const AttnArgs& a = t.a;
  const int C = gridDim.x, rank = blockIdx.x;     // cluster = (C, 1, 1)
  const int kvh = blockIdx.y / row_tiles, rt = blockIdx.y % row_tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sbase = smem_u32(smem);
  if (warp == 5) {
    tmem_alloc(tmem_slot, L::TMEM_COLS);
    tmem_relinquish();
  } else if (warp == 4) {
    // full and empty barriers of K, then of V, then the S and P V ones
    if (lane < 4 * L::MAX_STAGES)
      mbar_init(&k_full[lane], !TMA && (lane / L::MAX_STAGES) % 2 == 0 ? 32 : 1);
    if (lane < 2) mbar_init(&pv_done[lane], 1);
    if (lane == 0) mbar_init(s_full, 1);
    fence_mbar_init();
    if (TMA && lane == 0) prefetch_tmap(&map);
    __syncwarp();
  }
  pdl_wait();
  int seq = blockIdx.z;
  if (t.by_length) {       // (at most 64 sequences) this one is the blockIdx.z-th longest
    if (warp == 5) {
      const int n = a.n_seqs;
      const int c0 = lane < n ? a.ctx_len[lane] : 0, c1 = lane + 32 < n ? a.ctx_len[lane + 32] : 0;
      int k0 = 0, k1 = 0;
      for (int j = 0; j < n; ++j) {
        const int v = __shfl_sync(0xffffffffu, j < 32 ? c0 : c1, j & 31);
        k0 += v > c0 || (v == c0 && j < lane);
        k1 += v > c1 || (v == c1 && j < lane + 32);
      }
      if (lane < n && k0 == seq) *s_seq = lane;
      if (lane + 32 < n && k1 == seq) *s_seq = lane + 32;
    }
    __syncthreads();
    seq = *s_seq;
  }
  const int* table = a.block_tables + (size_t)seq * a.bt_ld;
  // the first split starts at token 0: its block ids need not wait for the metadata
  int early = 0;
  if (TMA && warp == 4 && rank == 0 && lane * 16 / a.block_size < t.bt_w)
    early = table[lane * 16 / a.block_size];
  TreeSeq s;
  const bool ok = tree_seq(t, seq, s);
  const int G = t.group;
  const int rows = s.ql * G - rt * TT_ROWS;        // of this tile on
  if (!ok || rows <= 0) {                          // uniform over the cluster
    if (!ok && rt == 0 && threadIdx.x == 0) set_status(ERR_BAD_INDEX);
    __syncthreads();
    if (warp == 5) tmem_dealloc(*tmem_slot, L::TMEM_COLS);
    return;
  }
  const int nrows = min(rows, TT_ROWS);
  const int act = (nrows + 31) / 32;               // softmax warps with rows
  const unsigned tiles = (unsigned)(s.ctx + TT_KEYS - 1) / TT_KEYS;   // (below 2^26: times C fits)
  const int t0 = (int)(tiles * rank >> t.log_splits);
  const int nt = (int)(tiles * (rank + 1) >> t.log_splits) - t0;
  const int q_half = L::q_half(act), KS = L::k_stages(act), VS = L::v_stages(act);
  const int off_k = L::HALVES * q_half, off_v = off_k + KS * L::STAGE;

  // (rare; the fence because the barrier before the epilogue orders nothing)
  auto found = [&](int what) {
    if (what == TT_LOST) set_status(ERR_BAD_INDEX);
    atomicOr(s_bad, what);
    __threadfence_block();
  };

  // ---- loader state (warp 4)
  // TMA: lane i holds the 8-token group of K of chunk i (16 tokens) of eight tiles
  int kid = 0, vid = 0, next = 0;
  auto chunks = [&](int j, bool have) -> int {
    const int c = t0 * (TT_KEYS / 16) + j * (TT_KEYS / 16) + lane;
    if (c * 16 >= s.ctx) return 0;
    int blk = have ? early : table[c * 16 / a.block_size];
    if (blk < 0 || blk >= a.num_blocks) {
      found(TT_LOST);
      blk = 0;             // load something valid; nothing of it is stored
    }
    return (blk * 2 * a.n_kv_heads + kvh) * (a.block_size / 8) + c * 16 % a.block_size / 8;
  };
  const int v_off = a.n_kv_heads * (a.block_size / 8);   // from K's group to V's
  auto issue = [&](int j, bool is_v, int st) {
    const int g = __shfl_sync(0xffffffffu, is_v ? vid : kid, ((j & 7) * 4 + lane) & 31);
    const int left = (s.ctx - (t0 + j) * TT_KEYS + 15) / 16;   // boxes of the tile
    uint64_t* full = (is_v ? v_full : k_full) + st;
    if (lane == 0) mbar_arrive_expect_tx(full, min(left, TT_KEYS / 16) * L::BOX);
    __syncwarp();
    if (lane < min(left, TT_KEYS / 16))
      tma_load_4d(smem + (is_v ? off_v : off_k) + st * L::STAGE + lane * L::BOX, &map, full,
                  is_v ? g + v_off : g);
  };
  // cp.async: pool rows (of hd elements) of keys lane and lane + 32 of a tile
  unsigned krow[2], vrow[2], nrow[2] = {0, 0};
  auto find = [&](int j, unsigned* row) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int p = (t0 + j) * TT_KEYS + 32 * h + lane;
      row[h] = ~0u;        // past the context: zeros
      if (p < s.ctx) {
        const int blk = table[p / a.block_size];
        if (blk >= 0 && blk < a.num_blocks)
          row[h] = ((unsigned)blk * 2 * a.n_kv_heads + kvh) * a.block_size + p % a.block_size;
        else
          found(TT_LOST);
      }
    }
  };
  auto copy = [&](const unsigned* row, bool is_v, int at) {
    constexpr int PPR = HD / 8, RPI = 32 / PPR;    // lanes a row, rows an instruction
    const uint32_t st = sbase + (is_v ? off_v : off_k) + at * L::STAGE;
    const int c = lane % PPR;
    const __nv_bfloat16* src =
        a.pool + c * 8 + (is_v ? (size_t)a.n_kv_heads * a.block_size * HD : 0);
#pragma unroll
    for (int i = 0; i < TT_KEYS / RPI; ++i) {
      const int key = i * RPI + lane / PPR;
      const unsigned r = __shfl_sync(0xffffffffu, row[i * RPI / 32], key & 31);
      cp_async16(st + (key >> 3) * L::GROUP + (c >> 3) * 1024 + sw128_off(key & 7, c & 7),
                 src + (r != ~0u ? (size_t)r * HD : 0), r != ~0u);
    }
    cp_arrive_noinc((is_v ? v_full : k_full) + at);
  };
  if (warp == 4 && lane == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(&p_full[i], 32 * act);
    mbar_init(s_free, 32 * act);
    mbar_init(q_full, 32 * act);
    *s_bad = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // only now: a dependent kernel that takes tensor memory must not get in before this CTA's
  if (threadIdx.x == 0) pdl_trigger();
  const int r = threadIdx.x;                       // row of a softmax thread
  const bool valid = r < nrows;
  const int R = rt * TT_ROWS + (valid ? r : 0), node = div_group(t, R);
  const size_t row = (size_t)s.q0 + node;
  const int col = (kvh * G + R - node * G) * HD;   // the row's place in q and out
  const uint32_t tmem = *tmem_slot;
  float ref = -INFINITY, l = 0.f;                  // a row's exponent reference (log2) and sum

  if (warp == 4) {
    // ---------------- loader: K of tile j + 1, then V of tile j (the order in which
    // their stages come free); block ids are read a window or a tile ahead
    RingPos kp, vp;
    auto room = [&](uint64_t* empty, const RingPos& p) {   // the stage's last user is done
      return __all_sync(0xffffffffu, mbar_wait(&empty[p.st], p.phase ^ 1)) != 0;
    };
    if (TMA) {
      if (nt > 0) {
        kid = chunks(0, rank == 0);
        issue(0, false, 0);
        kp.next(KS);
      }
      next = chunks(8, false);
      for (int j = 0; j < nt; ++j) {
        vid = kid;
        if (((j + 1) & 7) == 0) {
          kid = next;
          next = chunks(j + 9, false);
        }
        if (j + 1 < nt) {
          if (!room(k_empty, kp)) break;
          issue(j + 1, false, kp.st);
          kp.next(KS);
        }
        if (!room(v_empty, vp)) break;
        issue(j, true, vp.st);
        vp.next(VS);
      }
    } else {
      if (nt > 0) {
        find(0, krow);
        copy(krow, false, 0);
        kp.next(KS);
      }
      if (nt > 1) find(1, nrow);
      for (int j = 0; j < nt; ++j) {
        vrow[0] = krow[0], vrow[1] = krow[1];
        if (j + 1 < nt) {
          krow[0] = nrow[0], krow[1] = nrow[1];
          if (j + 2 < nt) find(j + 2, nrow);
          if (!room(k_empty, kp)) break;
          copy(krow, false, kp.st);
          kp.next(KS);
        }
        if (!room(v_empty, vp)) break;
        copy(vrow, true, vp.st);
        vp.next(VS);
      }
      cp_wait<0>();   // nothing in flight at exit
    }
  } else if (warp == 5) {
    // ---------------- MMA issue: the whole warp walks the loop, one elected lane issues.
    // Control flow and descriptors stay warp-uniform that way (in uniform registers);
    // with a single lane in the loop an MMA took ~110 cycles to issue and the issue
    // bounded the kernel
    if (nt > 0) {
      constexpr uint32_t idesc_s = idesc_bf16_m128(TT_KEYS);
      constexpr uint32_t idesc_o = idesc_bf16_m128(HD) | (1u << 16);   // V: MN-major
      const bool lead = elect_one();
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0;
      };
      RingPos kp, vp;
      auto issue_s = [&](int j) -> bool {
        if (!wait(&k_full[kp.st], kp.phase)) return false;
        tc_fence_after();
        if (!TMA) fence_proxy_async_smem();   // K arrived through the generic proxy
        const uint32_t kb = sbase + off_k + kp.st * L::STAGE;
        if (lead) {
#pragma unroll
          for (int h = 0; h < L::HALVES; ++h)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc_mma_bf16(tm, sw128_desc(sbase + h * q_half + kk * 32),
                          sw128_k_desc(kb + h * 1024 + kk * 32, L::GROUP), idesc_s,
                          (h | kk) ? 1u : 0u);
          tc_commit(s_full);
          tc_commit(&k_empty[kp.st]);
        }
        __syncwarp();
        kp.next(KS);
        return true;
      };
      bool good = wait(q_full, 0);
      if (good) good = issue_s(0);
      for (int j = 0; j < nt && good; ++j) {
        if (j + 1 < nt) {
          good = wait(s_free, j & 1);
          if (good) good = issue_s(j + 1);
          if (!good) break;
        }
        if (!wait(&v_full[vp.st], vp.phase)) break;
        if (!wait(&p_full[j & 1], (j >> 1) & 1)) break;
        tc_fence_after();
        if (!TMA) fence_proxy_async_smem();   // V too
        const uint32_t vb = sbase + off_v + vp.st * L::STAGE;
        if (lead) {
#pragma unroll
          for (int ks = 0; ks < TT_KEYS / 16; ++ks)
            tc_mma_bf16_ts(tm + L::COL_O, tm + L::COL_P + (j & 1) * (TT_KEYS / 2) + ks * 8,
                           sw128_mn_desc(vb + ks * 2 * L::GROUP, 1024, L::GROUP), idesc_o,
                           (j | ks) ? 1u : 0u);
          tc_commit(&v_empty[vp.st]);
          tc_commit(&pv_done[j & 1]);
        }
        __syncwarp();
        vp.next(VS);
      }
    }
    __syncwarp();
  } else if (warp < act) {
    // ---------------- softmax: one row a thread
    {
      // the warp's 32 rows, HD/8 lanes a row, straight into shared memory; missing rows are zero
      constexpr int PPR = HD / 8, RPI = 32 / PPR;
      const unsigned long long mine = row * a.ld_q + col;
      const int c = lane % PPR;
#pragma unroll
      for (int i = 0; i < 32 / RPI; ++i) {
        const int rr = i * RPI + lane / PPR;
        const unsigned long long off = __shfl_sync(0xffffffffu, mine, rr);
        cp_async16(sbase + (c >> 3) * q_half + sw128_off(warp * 32 + rr, c & 7),
                   a.q + off + c * 8, warp * 32 + rr < nrows);
      }
      cp_commit();
    }
    const unsigned long long* mask = t.mask + row * t.mask_ld;   // (a missing row masks as row 0)
    const unsigned long long m0 = mask[0];
    cp_wait<0>();
    fence_proxy_async_smem();
    mbar_arrive(q_full);
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint32_t to = tmem + L::COL_O + lane_off;
    const float sc = a.scale_log2;
    int done = 0;
    for (int j = 0; j < nt; ++j) {
      const int k0 = (t0 + j) * TT_KEYS;
      const uint32_t ts = tmem + lane_off;
      const uint32_t tp = tmem + L::COL_P + (j & 1) * (TT_KEYS / 2) + lane_off;
      if (!__all_sync(0xffffffffu, mbar_wait(s_full, j & 1))) break;
      tc_fence_after();
      constexpr int KH = TT_KEYS / 2;
      float x[TT_KEYS];
      tmem_ld64(ts, x);
      tc_fence_before();
      mbar_arrive(s_free);                         // S of the next tile may overwrite it
      const bool edge = k0 + TT_KEYS > s.base;     // drafts, or places past the context
      if (edge) {
        const unsigned long long win = tree_window(mask, t.mask_w, m0, k0, s.base, s.ctx);
        const uint32_t wl = (uint32_t)win, wh = (uint32_t)(win >> 32);
#pragma unroll
        for (int e = 0; e < KH; ++e) {
          if (!(wl & (1u << e))) x[e] = -INFINITY;
          if (!(wh & (1u << e))) x[KH + e] = -INFINITY;
        }
      }
      float mx = fmax3(x[0], x[1], x[2]), mx2 = fmax3(x[3], x[4], x[5]);
#pragma unroll
      for (int e = 6; e + 3 < TT_KEYS; e += 4) {   // two chains
        mx = fmax3(mx, x[e], x[e + 1]);
        mx2 = fmax3(mx2, x[e + 2], x[e + 3]);
      }
      mx = fmaxf(fmax3(mx, x[TT_KEYS - 2], x[TT_KEYS - 1]), mx2);
      if (edge) {
        const int lap = j / VS, st = j - lap * VS;
        if (!__all_sync(0xffffffffu, mbar_wait(&v_full[st], lap & 1))) break;
        uint8_t* vb = smem + off_v + st * L::STAGE;
        const int first = max(s.base - k0, 0);
        for (int i = first * (HD / 8) + r; i < TT_KEYS * (HD / 8); i += 32 * act) {
          const int key = i / (HD / 8), c = i % (HD / 8);
          uint4* p = reinterpret_cast<uint4*>(vb + (key >> 3) * L::GROUP + (c >> 3) * 1024 +
                                              sw128_off(key & 7, c & 7));
          if (k0 + key >= s.ctx) {
            *p = make_uint4(0u, 0u, 0u, 0u);
            continue;
          }
          uint4 q = *p;
          const uint4 n = make_uint4(nonfinite2(q.x), nonfinite2(q.y), nonfinite2(q.z), nonfinite2(q.w));
          if (n.x | n.y | n.z | n.w) {
            q.x &= ~n.x, q.y &= ~n.y, q.z &= ~n.z, q.w &= ~n.w;
            *p = q;
            found(TT_NONFINITE);
          }
        }
        fence_proxy_async_smem();
      }
      mx *= sc;
      const bool move = mx > ref + TT_RESCALE;     // any finite max when ref is -inf
      const bool rescale = move && ref != -INFINITY;
      const float alpha = rescale ? ex2_approx(ref - mx) : 1.f;
      if (__any_sync(0xffffffffu, rescale)) {
        // O holds the tiles before this one: once the last of them is in, scale it
        if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1))) break;
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < HD; c0 += 16) {
          float v[16];
          tmem_ld16(to + c0, v);
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(v[e] * alpha);
          tmem_st16(to + c0, u);
        }
      }
      if (move) ref = mx;
      l *= alpha;
      const float mu = ref == -INFINITY ? 0.f : ref;
      const float2 sc2 = make_float2(sc, sc), nmu2 = make_float2(-mu, -mu);
      float2 sum2 = make_float2(0.f, 0.f), sum3 = sum2;
      // P V of two tiles before has read this P buffer
      if (j >= 2 && !__all_sync(0xffffffffu, mbar_wait(&pv_done[j & 1], ((j - 2) >> 1) & 1))) break;
#pragma unroll
      for (int c0 = 0; c0 < TT_KEYS; c0 += KH) {
        uint32_t w[KH / 2];
#pragma unroll
        for (int e = 0; e < KH; e += 4) {
          const float2 xa = fma2(make_float2(x[c0 + e], x[c0 + e + 1]), sc2, nmu2);
          const float2 xb = fma2(make_float2(x[c0 + e + 2], x[c0 + e + 3]), sc2, nmu2);
          const float2 pa = make_float2(ex2_approx(xa.x), ex2_approx(xa.y));
          const float2 pb = make_float2(ex2_approx(xb.x), ex2_approx(xb.y));
          sum2 = add2(sum2, pa);
          sum3 = add2(sum3, pb);
          w[e >> 1] = pack_bf16x2(pa.x, pa.y);
          w[(e >> 1) + 1] = pack_bf16x2(pb.x, pb.y);
        }
        tmem_st16(tp + (c0 >> 1), w);
      }
      tmem_wait_st();
      l += (sum2.x + sum2.y) + (sum3.x + sum3.y);
      tc_fence_before();
      mbar_arrive(&p_full[j & 1]);
      done = j + 1;
    }
    if (nt > 0 && done == nt) {
      __all_sync(0xffffffffu, mbar_wait(&pv_done[(nt - 1) & 1], ((nt - 1) >> 1) & 1));
      tc_fence_after();
    }
  }

  // ---------------- epilogue.  Past the barrier every load of the CTA (with C > 1: of
  // every member) has landed and every MMA is complete
  if (C == 1) __syncthreads();
  else cluster_sync_relaxed();
  const uint32_t to = tmem + L::COL_O + ((uint32_t)((warp & 3) * 32) << 16);
  if (C == 1) {
    const int bad = *s_bad;
    if (warp < act && !(bad & TT_LOST)) {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      __nv_bfloat16* dst = a.out + row * a.ld_out + col;
#pragma unroll
      for (int c0 = 0; c0 < HD; c0 += 32) {
        float v[32];
        tmem_ld32(to + c0, v);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = l == 0.f ? 0.f : v[e] * inv;
        if (valid)
#pragma unroll
          for (int e = 0; e < 32; e += 8) store_bf16x8(dst + c0 + e, v + e);
      }
      if (bad && valid) add_nonfinite<HD>(t, table, kvh, row, s, dst);
    }
    tc_fence_before();
    __syncthreads();
  } else {
    // CTA z owns rows z * per .. of the tile: every CTA stores its O of them, and
    // (reference, sum), into the owner's shared memory as [split][4 columns][row]
    // (up to 512 contiguous bytes a warp instruction); the owner adds the splits up
    // in order
    const int per = (nrows + C - 1) / C, pitch = per | 1;
    if (warp < act) {
      s_out[r] = row * a.ld_out + col;
      const int owner = valid ? r / per : 0, at = r - owner * per;
      const uint32_t dst =
          cluster_map(sbase, owner) + (uint32_t)(rank * (HD / 4) * pitch + at) * 16;
      if (valid) st_cluster_f2(cluster_map(sbase + L::OFF_ML + (rank * per + at) * 8, owner), ref, l);
#pragma unroll
      for (int c0 = 0; c0 < HD; c0 += 32) {
        float v[32];
        if (nt > 0) {
          tmem_ld32(to + c0, v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        }
        if (valid)
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            st_cluster_v4(dst + (c0 + e) / 4 * pitch * 16, v[e], v[e + 1], v[e + 2], v[e + 3]);
      }
    }
    const int mine = *s_bad;
    if (mine && threadIdx.x < C) red_cluster_or(cluster_map(smem_u32(s_bad), threadIdx.x), mine);
    tc_fence_before();
    cluster_sync_all();          // everything has arrived; nobody touches this CTA's memory after
    const int bad = *s_bad;
    const int r0 = rank * per, n = bad & TT_LOST ? 0 : min(per, nrows - r0);
    if (C == 2) merge_rows<HD, 2>(smem, s_ml, s_out + r0, a.out, per, pitch, n);
    else if (C == 4) merge_rows<HD, 4>(smem, s_ml, s_out + r0, a.out, per, pitch, n);
    else merge_rows<HD, 8>(smem, s_ml, s_out + r0, a.out, per, pitch, n);
    if (bad) {
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += TT_THREADS) {
        const int Ri = rt * TT_ROWS + r0 + i;
        add_nonfinite<HD>(t, table, kvh, (size_t)s.q0 + div_group(t, Ri), s, a.out + s_out[r0 + i]);
      }
    }
  }
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, L::TMEM_COLS);
  }
}

// The pool as {64 columns, 8 tokens, halves, 8-token groups}: group g of (block,
// K or V, head) is number ((block * 2 + V) * n_kv + head) * bs / 8 + g.
template <int HD>
static int tree_pool_map(CUtensorMap* map, const AttnArgs& a) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    set_last_error("cuTensorMapEncodeTiled entry point unavailable");
    return TB_ERR_CUDA;
  }
  const cuuint64_t tokens = (cuuint64_t)a.num_blocks * 2 * a.n_kv_heads * a.block_size;
  const cuuint64_t dims[4] = {64, 8, HD / 64, tokens / 8};
  const cuuint64_t strides[3] = {HD * 2, 128, 8 * HD * 2};
  const cuuint32_t box[4] = {64, 8, HD / 64, 2};
  const cuuint32_t one[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<__nv_bfloat16*>(a.pool),
                        dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("cuTensorMapEncodeTiled failed (%d) for the KV pool", (int)r);
    return TB_ERR_CUDA;
  }
  return TB_OK;
}

// CTAs that share a context: the power of two, at most 8, that brings the longest
// context's share down to once to twice the average work of a resident CTA (148 SMs x 2;
// more where 8 are too few), so that one wave covers a small batch and a long context
// does not outlast the others by much, but no share below four tiles (the merge
// costs more than it saves).
static int tree_splits(int n_seqs, int n_kv, int row_tiles, int max_ctx, long long ctx_total) {
  const long long share = ctx_total * n_kv * row_tiles / (148 * 2);
  const long long least = 4 * TT_KEYS;
  const long long c = max_ctx / (share > least ? share : least);
  return c >= 8 ? 8 : c >= 4 ? 4 : c >= 2 ? 2 : 1;
}

template <int HD, bool TMA>
static int tree_tc_launch(TreeAttnArgs t, int max_ctx, long long ctx_total, cudaStream_t st) {
  using L = TreeTcLayout<HD>;
  static std::atomic<unsigned long long> attr_devs{0};
  if (int rc = smem_attr_once(tree_attn_tc_kernel<HD, TMA>, L::SMEM, attr_devs,
                              "tree attention smem attribute", true))
    return rc;
  CUtensorMap map{};
  if (TMA)
    if (int rc = tree_pool_map<HD>(&map, t.a)) return rc;
  const long long rows = (long long)t.max_q * (t.a.n_q_heads / t.a.n_kv_heads);
  const int row_tiles = (int)((rows + TT_ROWS - 1) / TT_ROWS);
  if ((long long)row_tiles * t.a.n_kv_heads > 65535) return arg_err("too many heads and nodes");
  const int C = tree_splits(t.a.n_seqs, t.a.n_kv_heads, row_tiles, max_ctx, ctx_total);
  t.log_splits = C == 8 ? 3 : C == 4 ? 2 : C - 1;
  // More CTAs than fit at once and ragged, long contexts: longest sequences first,
  // so that none starts late (ranking them costs ~0.5 us a CTA).  Device us without / with:
  // 32 chains over 500-4000 tokens 60.4 / 58.8, 16 trees over 300-6000 55.9 / 48.3, 64
  // chains over 100-4000 106 / 89; lengths within a third of one another, left in the
  // caller's order, 82.4 / 83.8
  const int n = t.a.n_seqs;
  t.by_length = n > 1 && n <= 64 && (long long)C * t.a.n_kv_heads * row_tiles * n > 148 * 2 &&
                4ll * max_ctx * n > 5 * ctx_total && max_ctx / C >= 1024;
  return launch_pdl(tree_attn_tc_kernel<HD, TMA>, dim3(C, t.a.n_kv_heads * row_tiles, t.a.n_seqs),
                    dim3(TT_THREADS), L::SMEM, st, C, "tree attention launch", map, t, row_tiles);
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
  if (reinterpret_cast<uintptr_t>(t.mask) % 8) return arg_err("tree_mask must be 8-byte aligned");
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  t.group = a.n_q_heads / a.n_kv_heads;
  t.group_magic = (unsigned)((0x100000000ull + t.group - 1) / t.group);
  const long long width = (long long)t.bt_w * a.block_size;   // tokens a table row can hold
  if (max_ctx <= 0 || max_ctx > width) max_ctx = (int)(width < 0x7fffffff ? width : 0x7fffffff);
  if (ctx_total <= 0 || ctx_total > (long long)max_ctx * a.n_seqs)
    ctx_total = (long long)max_ctx * a.n_seqs;
  // pool rows (tokens of one head) are 32-bit numbers in the kernels
  if ((long long)a.num_blocks * 2 * a.n_kv_heads * a.block_size >= 0xffffffffll)
    return arg_err("KV pool rows beyond 2^32");
  const bool tma = a.block_size % 16 == 0;      // 16-token boxes inside one block
  switch (head_dim) {
    case 16: return tree_simple_launch<16>(t, st);
    case 64:
      return tma ? tree_tc_launch<64, true>(t, max_ctx, ctx_total, st)
                 : tree_tc_launch<64, false>(t, max_ctx, ctx_total, st);
    default:
      return tma ? tree_tc_launch<128, true>(t, max_ctx, ctx_total, st)
                 : tree_tc_launch<128, false>(t, max_ctx, ctx_total, st);
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
