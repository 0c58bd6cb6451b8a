// Verification of drafted tokens.
//
// A sequence's draft tree has its nodes in the rows q_start .. q_start+q_len-1
// of the flat batch; node 0 is the root (the last accepted token), parents[row]
// < node index its parent inside the sequence.  The walk starts at the root and
// goes from node to accepted child until no child is accepted.
//
// Greedy: the accepted child is the first one whose id is the target's argmax
// at the node.
//
// Sampled: at node c with children x_1 .. x_m (node order), r_0 = probs[row c]
// and, when the children were drawn without replacement from a distribution
// d_0 = draft_probs[draft_rows[row c]]:
//   x_j is accepted if d_{j-1}(x_j) > 0 and u_j d_{j-1}(x_j) < r_{j-1}(x_j);
//   else r_j = max(r_{j-1} - d_{j-1}, 0) / Z_j, Z_j its sum (r_{j-1} kept where
//   Z_j = 0), and d_j is d_0 without x_1 .. x_j over 1 - sum of their d_0.
//   A child of draft probability 0 is rejected and changes nothing.
// Children picked outright (draft row -1): x_j is accepted if
//   r(x_j) > 0 and u_j (1 - sum of the rejected r) < r(x_j), else r(x_j) becomes 0.
// When no child is accepted the next token is the first y whose cumulative
// sum of r exceeds u_root * sum(r).  With u uniform this leaves the target's
// distribution unchanged (speculative sampling; Leviathan et al. 2023, with
// several candidates a node as in Miao et al. 2024).
//
// Everything is evaluated in 64 bits: the tests compare products of 24-bit
// numbers, and the position of a sample among ~1.5e5 cumulative sums would
// move with the summation order in 32.
//
// What bounds them (B200, CUDA graph, vocabulary 152064).  Greedy: launch and two
// dependent loads, 2.3 us for one sequence, 3.3 us for 128.  Sampled: steps that wait
// for one another.  One sequence, outright drafts 9.0 us; stamps of an instrumented
// build: loads of rows, tree and probabilities 2.1 us, walk 1.7, pass over the last
// node's rows 1.9, sums over the cluster 1.4, search 2.4.  64 chains 26.6 us, of them
// ~14 in the pass (78 MB, the floor of the call is 11.9 us).  8 trees of 40 nodes
// 23.3 us: the slowest walk takes 13, as each Z is a pass that decides the next
// sibling's test; the floor counts one pass.
#include <cooperative_groups.h>

#include "common.cuh"
#include "host.h"

namespace tb {

constexpr int VF_NODES = 256;      // nodes of a sequence's tree
constexpr int VF_MAX_WARPS = 16;
constexpr int VF_MAX_CLUSTER = 16;
constexpr int VF_BATCHES = 32;     // sums a warp keeps of its part of the vocabulary
constexpr int VF_PER_LANE = VF_MAX_CLUSTER * VF_MAX_WARPS / 32;   // segments a lane looks at

struct TreeArgs {
  const int *ids, *parents, *q_start, *q_len;
  int n_seqs, n_rows;
  int *n_accepted, *path, *next_ids;
  int path_ld, path_w;
};

struct VerifyArgs {
  TreeArgs t;
  const float* probs;
  long long ld_p;
  int vocab;
  const float* draft_probs;
  long long ld_d;
  int n_draft_rows;
  const int* draft_rows;
  const float* uniforms;
};

// The rows of a sequence lie inside the batch and its tree is not too large (without
// nodes its first row may be anything).
__device__ __forceinline__ bool tree_ok(const TreeArgs& t, int q0, int ql) {
  return ql == 0 || (ql > 0 && ql <= VF_NODES && q0 >= 0 && q0 <= t.n_rows - ql);
}

// ------------------------------------------------------------------- greedy

constexpr int VG_WARPS = 4;

// One warp a sequence: its nodes in shared memory, then one ballot round a step.
__global__ void __launch_bounds__(VG_WARPS * 32)
    verify_greedy_kernel(const TreeArgs t, const int* target_ids) {
  __shared__ int s_par[VG_WARPS][VF_NODES], s_id[VG_WARPS][VF_NODES], s_tgt[VG_WARPS][VF_NODES];
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seq = blockIdx.x * VG_WARPS + warp;
  if (seq >= t.n_seqs) return;
  const int q0 = t.q_start[seq], ql = t.q_len[seq];
  int* path = t.path + (size_t)seq * t.path_ld;
  int n = 0, next = -1;
  if (!tree_ok(t, q0, ql)) {
    if (lane == 0) set_status(ERR_BAD_INDEX);
  } else if (ql > 0) {
    for (int i = lane; i < ql; i += 32) {
      int p = t.parents[q0 + i];
      const int id = t.ids[q0 + i], tgt = target_ids[q0 + i];   // (all loads before the checks)
      if (i > 0 && (p < 0 || p >= i || id < 0)) {   // unreachable
        set_status(ERR_BAD_INDEX);
        p = -1;
      }
      s_par[warp][i] = i > 0 ? p : -1;
      s_id[warp][i] = id;
      s_tgt[warp][i] = tgt;
    }
    __syncwarp();
    int c = 0;
    if (lane == 0) path[0] = 0;
    n = 1;
    next = s_tgt[warp][0];
    while (n < t.path_w) {
      int found = -1;
      for (int i0 = c & ~31; i0 < ql && found < 0; i0 += 32) {
        const int i = i0 + lane;
        const unsigned hit = __ballot_sync(
            0xffffffffu, i < ql && s_par[warp][i] == c && s_id[warp][i] == next);
        if (hit) found = i0 + __ffs(hit) - 1;
      }
      if (found < 0) break;
      c = found;
      if (lane == 0) path[n] = c;
      ++n;
      next = s_tgt[warp][c];
    }
  }
  for (int k = n + lane; k < t.path_w; k += 32) path[k] = -1;
  if (lane == 0) {
    t.n_accepted[seq] = n > 0 ? n - 1 : 0;
    t.next_ids[seq] = next;
  }
}

// ------------------------------------------------------------------ sampled

// What has been rejected at the current node, in order.
struct Rejections {
  int n;                      // entries
  int token[VF_NODES];
  double scale[VF_NODES];     // draft distribution: 1 / (1 - sum of d_0 of earlier entries)
  double inv_z[VF_NODES];     // 1 / Z, or 0 where Z was 0 (r kept)
};

// r of one token with target probability p and draft probability d after
// every rejection of h.
__device__ __forceinline__ double residual(const Rejections& h, bool dist, int token, float p,
                                           float d) {
  double r = p, dd = d;
  for (int k = 0; k < h.n; ++k) {
    if (dist && h.inv_z[k] > 0.0) r = fmax(r - dd * h.scale[k], 0.0) * h.inv_z[k];
    if (h.token[k] == token) {
      if (dist) dd = 0.0;
      else r = 0.0;
    }
  }
  return r;
}

// Whether one of the rejected tokens lies in first .. first+count-1 (all lanes of
// the warp ask the same).
__device__ __forceinline__ bool rejected(const Rejections& h, int first, int count) {
  bool s = false;
  for (int k0 = 0; k0 < h.n; k0 += 32) {
    const int k = k0 + (threadIdx.x & 31);
    s |= k < h.n && (unsigned)(h.token[k] - first) < (unsigned)count;
  }
  return __any_sync(0xffffffffu, s);
}

// Eight bytes into a cluster member's shared memory, counted by its mbarrier.
__device__ __forceinline__ void st_async_f64(uint32_t addr, double v, uint32_t bar) {
  asm volatile(
      "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(addr),
      "l"(__double_as_longlong(v)), "r"(bar)
      : "memory");
}

__device__ __forceinline__ float4 load4(const float* row, int y, int end, bool vec) {
  if (vec && y + 4 <= end) return __ldg(reinterpret_cast<const float4*>(row + y));
  return make_float4(y < end ? __ldg(row + y) : 0.f, y + 1 < end ? __ldg(row + y + 1) : 0.f,
                     y + 2 < end ? __ldg(row + y + 2) : 0.f, y + 3 < end ? __ldg(row + y + 3) : 0.f);
}

// r of tokens y + STRIDE g .. + 3, g < GROUPS (y already the lane's, base the
// warp's; 0 from `end` on); dv: their draft probabilities, 0 for rejected tokens.
// All loads are issued before the first is used.
template <bool DIST, int GROUPS, int STRIDE>
__device__ __forceinline__ void weights(const Rejections& h, const float* p, const float* d,
                                        int base, int y, int end, bool vec, double (*w)[4],
                                        float4* dv) {
  float4 pv[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) pv[g] = load4(p, y + STRIDE * g, end, vec);
  if (DIST)
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) dv[g] = load4(d, y + STRIDE * g, end, vec);
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
    w[g][0] = pv[g].x, w[g][1] = pv[g].y, w[g][2] = pv[g].z, w[g][3] = pv[g].w;
  // the warp's stretch holds a rejected token (rare): only then are tokens compared
  const bool special = rejected(h, base, 128 * GROUPS);
  for (int k = 0; k < h.n; ++k) {
    if (DIST) {
      const double sc = h.scale[k], iz = h.inv_z[k];
      if (iz > 0.0) {
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          w[g][0] = fmax(w[g][0] - dv[g].x * sc, 0.0);
          w[g][1] = fmax(w[g][1] - dv[g].y * sc, 0.0);
          w[g][2] = fmax(w[g][2] - dv[g].z * sc, 0.0);
          w[g][3] = fmax(w[g][3] - dv[g].w * sc, 0.0);
        }
        if (iz != 1.0)
#pragma unroll
          for (int g = 0; g < GROUPS; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) w[g][e] *= iz;
      }
    }
    if (special) {
      const int x = h.token[k] - y;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {
        if (DIST) {
          if (x == STRIDE * g) dv[g].x = 0.f;
          if (x == STRIDE * g + 1) dv[g].y = 0.f;
          if (x == STRIDE * g + 2) dv[g].z = 0.f;
          if (x == STRIDE * g + 3) dv[g].w = 0.f;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (x == STRIDE * g + e) w[g][e] = 0.0;
        }
      }
    }
  }
}

// Where in the sequence of all lanes' N values (lane after lane) the running sum
// passes a target: the last positive value whose exclusive prefix does not exceed
// it.  Some value qualifies whenever one is positive, and every warp that asks about
// the same values picks the same one, however the prefixes are rounded.  at: the
// target, with `fraction` as a fraction of the sum; afterwards relative to the value.
// total: the sum.  -1: nothing is positive.
template <int N>
__device__ __forceinline__ int locate(const double* v, bool fraction, double& at, double& total) {
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < N; ++k) sum += v[k];
  double inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  total = __shfl_sync(0xffffffffu, inc, 31);
  if (fraction) at = fmax(at * total, 0.0);   // a NaN aims at 0
  double ex = __shfl_up_sync(0xffffffffu, inc, 1);
  if (lane == 0) ex = 0.0;
  const unsigned some = __ballot_sync(0xffffffffu, sum > 0.0 && ex <= at);
  if (some == 0) return -1;
  const int from = 31 - __clz(some);
  int mine = 0;
  double run = ex, before = ex;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (v[k] > 0.0 && run <= at) mine = k, before = run;
    run += v[k];
  }
  at -= __shfl_sync(0xffffffffu, before, from);
  return from * N + __shfl_sync(0xffffffffu, mine, from);
}

// One cluster a sequence, the vocabulary cut into one segment a warp and a
// segment into at most VF_BATCHES batches.  Every CTA walks the tree alike (same
// loads, same arithmetic), so the cluster only meets for sums over the
// vocabulary: one for each rejection whose Z a later sibling's test needs, one
// for the sample.
// GROUPS: 128-token groups whose loads a warp has in flight.
// KEEP: a warp keeps its segment's r between the passes at a node where one step covers it.
template <int THREADS, int MIN_CTAS, int GROUPS, bool KEEP>
__global__ void __launch_bounds__(THREADS, MIN_CTAS) verify_kernel(const VerifyArgs a) {
  namespace cg = cooperative_groups;
  constexpr int WARPS = THREADS / 32;
  static_assert(WARPS <= VF_MAX_WARPS, "sum slots");
  __shared__ int s_id[VF_NODES], s_par[VF_NODES], s_drow[VF_NODES];
  __shared__ float s_p[VF_NODES], s_d[VF_NODES], s_u[VF_NODES];
  __shared__ Rejections s_h;
  __shared__ int s_node, s_sum_wanted;
  __shared__ double s_sum[2][VF_MAX_CLUSTER * WARPS + 32];   // padded: see `pad`
  __shared__ uint64_t s_arrived[2];
  __shared__ double s_batch[WARPS][VF_BATCHES];
  cg::cluster_group cluster = cg::this_cluster();
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const TreeArgs& t = a.t;
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int seq = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int q0 = t.q_start[seq], ql = t.q_len[seq];
  int* path = t.path + (size_t)seq * t.path_ld;
  const bool ok = tree_ok(t, q0, ql);
  if (!ok || ql == 0) {   // uniform over the cluster
    if (rank == 0) {
      if (!ok && tid == 0) set_status(ERR_BAD_INDEX);
      for (int k = tid; k < t.path_w; k += THREADS) path[k] = -1;
      if (tid == 0) {
        t.n_accepted[seq] = 0;
        t.next_ids[seq] = -1;
      }
    }
    return;
  }
  if (tid == 0) {
    mbar_init(&s_arrived[0], 1);
    mbar_init(&s_arrived[1], 1);
    fence_mbar_init();
  }
  __syncthreads();
  auto started = cluster.barrier_arrive();   // waited for before the first remote store

  // ---- the tree and, for every node, the probabilities its test compares
  for (int i = tid; i < ql; i += THREADS) {
    int p = t.parents[q0 + i];
    const int id = t.ids[q0 + i];
    int dr = a.draft_rows != nullptr ? a.draft_rows[q0 + i] : -1;
    if (dr >= a.n_draft_rows || dr < -1) {
      set_status(ERR_BAD_INDEX);
      dr = -1;
    }
    if (i == 0) {
      p = -1;
    } else if (p < 0 || p >= i || id < 0 || id >= a.vocab) {   // unreachable
      set_status(ERR_BAD_INDEX);
      p = -1;
    }
    s_par[i] = p;
    s_id[i] = id;
    s_u[i] = a.uniforms[q0 + i];
    s_drow[i] = dr;
  }
  if (tid == 0) s_h.n = 0;
  __syncthreads();
  for (int i = tid; i < ql; i += THREADS) {
    const int p = s_par[i];
    const int dr = p >= 0 ? s_drow[p] : -1;
    s_p[i] = p >= 0 ? a.probs[(size_t)(q0 + p) * a.ld_p + s_id[i]] : 0.f;
    s_d[i] = dr >= 0 ? a.draft_probs[(size_t)dr * a.ld_d + s_id[i]] : 0.f;
  }
  __syncthreads();
  cluster.barrier_wait(std::move(started));

  // this warp's segment of the vocabulary, in batches
  const int step = 128 * GROUPS;
  const int n_seg = C * WARPS;
  const int batch = ((a.vocab + n_seg * VF_BATCHES - 1) / (n_seg * VF_BATCHES) + step - 1) / step * step;
  const int n_batch = ((a.vocab + n_seg - 1) / n_seg + batch - 1) / batch;
  const int seg = rank * WARPS + warp;
  const long long y_begin = (long long)seg * n_batch * batch;
  const int y0 = (int)min(y_begin, (long long)a.vocab);
  const int y1 = (int)min(y_begin + (long long)n_batch * batch, (long long)a.vocab);
  const bool vec_p = a.ld_p % 4 == 0 && reinterpret_cast<uintptr_t>(a.probs) % 16 == 0;
  const bool vec_d = a.ld_d % 4 == 0 && reinterpret_cast<uintptr_t>(a.draft_probs) % 16 == 0;
  const int log_per = n_seg > 32 ? 31 - __clz(n_seg / 32) : 0;   // (n_seg is a power of two)
  auto pad = [&](int i) { return i + (i >> log_per); };   // a lane's run of sums has no bank to share
  int pass = 0;
  bool lost = false;                 // a wait ran out (the status says so): no further waits
  const double* sums = s_sum[0];
  double w[GROUPS][4];               // r of a step, and d where it is not rejected
  float4 dv[GROUPS];
  int held = -1, applied = 0;        // KEEP: the node and rejections they stand for

  // Sums over the vocabulary of r with the rejections of s_h applied, at node c:
  // `sums` gets every segment's, s_batch those of this CTA's batches.  All threads of
  // the cluster call it; no warp of the CTA reads s_h from the moment all sums have
  // arrived.  Every sum travels as an asynchronous store counted by the receiver's
  // barrier (a cluster barrier costs twice as much); two buffers take turns: a CTA is
  // at most one pass ahead, since a pass needs every CTA's sums.
  auto vocab_sums = [&](int c, bool dist) {
    const float* p = a.probs + (size_t)(q0 + c) * a.ld_p;
    const float* d = dist ? a.draft_probs + (size_t)s_drow[c] * a.ld_d : nullptr;
    double acc = 0.0;
    const bool vec = vec_p && (!dist || vec_d);
    bool have = KEEP && dist && held == c;
    if (have) {
      // fold in the last rejection's Z, apply the new one
      for (; applied < s_h.n; ++applied) {
        const double iz = applied > 0 ? s_h.inv_z[applied - 1] : 1.0, sc = s_h.scale[applied];
        if (iz == 0.0) break;        // a rejection that was taken back: start over
        const int x = s_h.token[applied] - y0 - 4 * lane;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          w[g][0] = fmax(w[g][0] * iz - dv[g].x * sc, 0.0);
          w[g][1] = fmax(w[g][1] * iz - dv[g].y * sc, 0.0);
          w[g][2] = fmax(w[g][2] * iz - dv[g].z * sc, 0.0);
          w[g][3] = fmax(w[g][3] * iz - dv[g].w * sc, 0.0);
          if (x == 128 * g) dv[g].x = 0.f;
          if (x == 128 * g + 1) dv[g].y = 0.f;
          if (x == 128 * g + 2) dv[g].z = 0.f;
          if (x == 128 * g + 3) dv[g].w = 0.f;
        }
      }
      have = applied == s_h.n && (s_h.n == 0 || s_h.inv_z[s_h.n - 1] != 0.0);
    }
    for (int b = 0; b < n_batch; ++b) {
      const int end = min(y0 + (b + 1) * batch, y1);
      double one = 0.0;
      for (int y = y0 + b * batch; y < end; y += step) {
        if (!have) {
          if (dist) weights<true, GROUPS, 128>(s_h, p, d, y, y + 4 * lane, y1, vec, w, dv);
          else weights<false, GROUPS, 128>(s_h, p, d, y, y + 4 * lane, y1, vec, w, dv);
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) one += (w[g][0] + w[g][1]) + (w[g][2] + w[g][3]);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) one += __shfl_xor_sync(0xffffffffu, one, o);
      if (lane == 0) s_batch[warp][b] = one;
      acc += one;
    }
    if (KEEP && !have) {
      // held from now on where one step is the whole segment (the last entry's
      // inv_z, still 1, has not been folded in)
      held = dist && n_batch * batch == step && s_h.n > 0 && s_h.inv_z[s_h.n - 1] == 1.0 ? c : -1;
      applied = s_h.n;
    }
    const int buf = pass & 1;
    sums = s_sum[buf];
    if (C > 1) {
      if (tid == 0) mbar_arrive_expect_tx(&s_arrived[buf], n_seg * 8);
      if (lane < C)
        st_async_f64(cluster_map(smem_u32(&s_sum[buf][pad(seg)]), lane), acc,
                     cluster_map(smem_u32(&s_arrived[buf]), lane));
      if (!lost) lost = !mbar_wait(&s_arrived[buf], (pass >> 1) & 1);
    } else if (lane == 0) {   // (asynchronous stores are for clusters: without one they are refused)
      s_sum[buf][pad(seg)] = acc;
    }
    ++pass;
    __syncthreads();
  };
  const int per = (n_seg + 31) / 32;   // segment sums a lane looks at
  auto lane_sums = [&](double* v) {
#pragma unroll
    for (int k = 0; k < VF_PER_LANE; ++k)
      v[k] = k < per && lane * per + k < n_seg ? sums[pad(lane * per + k)] : 0.0;
  };

  // ---- the walk, by the first warp of every CTA; the others join for a sum
  int c = 0, n = 1, x = 0;         // node, path length, last child looked at
  double gone = 0.0;
  bool unscaled = false;           // the last rejection's inv_z still stands for 1
  if (rank == 0 && tid == 0) path[0] = 0;
  while (true) {
    if (warp == 0) {
      bool sum = false;
      while (true) {
        // the next child in node order
        int child = -1;
        for (int i0 = (x + 1) & ~31; i0 < ql && n < t.path_w && child < 0; i0 += 32) {
          const int i = i0 + lane;
          const unsigned hit = __ballot_sync(0xffffffffu, i < ql && i > x && s_par[i] == c);
          if (hit) child = i0 + __ffs(hit) - 1;
        }
        if (child < 0) break;
        const int id = s_id[child];
        const double u = s_u[child];
        const bool again = rejected(s_h, id, 1);
        bool took;
        if (s_drow[c] >= 0) {
          const double left = 1.0 - gone;
          const double scale = left > 0.0 ? 1.0 / left : 0.0;
          const double share = again ? 0.0 : s_d[child] * scale;
          x = child;
          if (!(share > 0.0)) continue;
          if (unscaled) {          // the last rejection's Z, now that a test needs it
            x = child - 1;
            sum = true;
            break;
          }
          took = u * share < residual(s_h, true, id, s_p[child], s_d[child]);
          if (!took) {
            __syncwarp();
            if (lane == 0) {
              s_h.token[s_h.n] = id;
              s_h.scale[s_h.n] = scale;
              s_h.inv_z[s_h.n] = 1.0;
              s_h.n += 1;
            }
            __syncwarp();
            unscaled = true;
            gone += s_d[child];
          }
        } else {
          const double r = again ? 0.0 : (double)s_p[child];
          x = child;
          took = r > 0.0 && u * (1.0 - gone) < r;
          if (!took) {
            gone += r;
            __syncwarp();
            if (lane == 0) {
              s_h.token[s_h.n] = id;
              s_h.n += 1;
            }
            __syncwarp();
          }
        }
        if (took) {
          c = child;
          gone = 0.0;
          unscaled = false;
          if (rank == 0 && lane == 0) path[n] = c;
          ++n;
          __syncwarp();
          if (lane == 0) s_h.n = 0;
          __syncwarp();
        }
      }
      if (lane == 0) {
        s_node = c;
        s_sum_wanted = sum;
      }
    }
    __syncthreads();
    c = s_node;
    if (!s_sum_wanted) break;
    vocab_sums(c, true);
    if (warp == 0) {
      double z = 0.0;
      for (int k = lane; k < n_seg; k += 32) z += sums[pad(k)];
#pragma unroll
      for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
      if (lane == 0) s_h.inv_z[s_h.n - 1] = z > 0.0 ? 1.0 / z : 0.0;
      __syncwarp();
      unscaled = false;
    }
  }

  // ---- the sample (r up to its scale).  A last rejection that leaves nothing
  // (Z = 0) is taken back.
  const float* prow = a.probs + (size_t)(q0 + c) * a.ld_p;
  const bool dist = s_drow[c] >= 0;
  const float* drow = dist ? a.draft_probs + (size_t)s_drow[c] * a.ld_d : nullptr;
  vocab_sums(c, dist);
  // the segment (the same answer in every warp of the cluster), its batch, then the
  // element; a target that rounding leaves past a level's last sum takes the last
  // positive value
  double at = s_u[0], total, v[VF_PER_LANE];
  lane_sums(v);
  int found = locate<VF_PER_LANE>(v, true, at, total);
  if (found < 0 && dist && s_h.n > 0) {
    __syncthreads();
    if (tid == 0) s_h.inv_z[s_h.n - 1] = 0.0;
    __syncthreads();
    vocab_sums(c, dist);
    at = s_u[0];
    lane_sums(v);
    found = locate<VF_PER_LANE>(v, true, at, total);
  }
  if (rank == 0 && warp == 0) {
    for (int k = n + lane; k < t.path_w; k += 32) path[k] = -1;
    if (lane == 0) {
      t.n_accepted[seq] = n - 1;
      if (found < 0) t.next_ids[seq] = -1;
    }
  }
  // (a CTA that gave up waiting stays until nobody can still write to it)
  if (lost) asm volatile("barrier.cluster.arrive;\n\tbarrier.cluster.wait;" ::: "memory");
  if (found < 0 || found / VF_PER_LANE * per + found % VF_PER_LANE != seg) return;
  int b = 0;
  if (n_batch > 1) {
    const double one = lane < n_batch ? s_batch[warp][lane] : 0.0;
    b = locate<1>(&one, false, at, total);
    if (b < 0) return;     // (a positive segment has a positive batch)
  }
  // a lane's 4 * GROUPS elements are neighbours now
  const bool vec = vec_p && (!dist || vec_d);
  const int end = min(y0 + (b + 1) * batch, y1);
  int next = -1;
  for (int y = y0 + b * batch; y < end; y += step) {
    const int mine = y + lane * 4 * GROUPS;
    if (dist) weights<true, GROUPS, 4>(s_h, prow, drow, y, mine, y1, vec, w, dv);
    else weights<false, GROUPS, 4>(s_h, prow, drow, y, mine, y1, vec, w, dv);
    const double left = at;
    const int e = locate<4 * GROUPS>(&w[0][0], false, at, total);
    if (e >= 0) next = y + e;
    if (left < total) break;
    at = left - total;
  }
  if (lane == 0) t.next_ids[seq] = next;
}

static int check_tree(const TreeArgs& t, int max_q) {
  if (t.n_seqs < 0 || t.n_rows < 0 || t.path_w <= 0 || t.path_ld < t.path_w)
    return arg_err("n_seqs / n_rows / path width");
  if (max_q > VF_NODES) return arg_err("a draft tree has at most 256 nodes");
  if (t.n_seqs > 0 && (t.q_start == nullptr || t.q_len == nullptr || t.n_accepted == nullptr ||
                       t.path == nullptr || t.next_ids == nullptr))
    return arg_err("null pointer");
  // (a padded batch may have no rows at all)
  if (t.n_seqs > 0 && t.n_rows > 0 && (t.ids == nullptr || t.parents == nullptr))
    return arg_err("null pointer");
  return TB_OK;
}

int verify_greedy_launch(const TreeArgs& t, const int* target_ids, int max_q, cudaStream_t st) {
  if (int rc = check_tree(t, max_q)) return rc;
  if (t.n_seqs == 0) return TB_OK;
  if (t.n_rows > 0 && target_ids == nullptr) return arg_err("null pointer");
  return launch_pdl(verify_greedy_kernel, dim3((t.n_seqs + VG_WARPS - 1) / VG_WARPS),
                    dim3(VG_WARPS * 32), 0, st, 1, "greedy verification launch", t, target_ids);
}

int verify_launch(const VerifyArgs& a, int max_q, cudaStream_t st) {
  if (int rc = check_tree(a.t, max_q)) return rc;
  if (a.t.n_seqs == 0) return TB_OK;
  if (a.vocab <= 0 || a.vocab > (1 << 28) || a.ld_p < a.vocab ||
      (a.t.n_rows > 0 && (a.probs == nullptr || a.uniforms == nullptr)))
    return arg_err("probs / vocab / uniforms");
  if (a.t.n_rows > 0 && (a.draft_probs == nullptr) != (a.draft_rows == nullptr))
    return arg_err("draft_probs and draft_rows go together");
  if (a.draft_probs != nullptr && (a.ld_d < a.vocab || a.n_draft_rows < 0))
    return arg_err("draft_probs shape");
  // few sequences: clusters of 16 (a sequence on 16 SMs, r kept between the passes at a
  // node); many: smaller CTAs, four an SM, in one wave.  Device us of either form at a vocabulary of
  // 152064, first / second: 8 sequences: chains of 6 16.2 / 17.0, trees of 40 23.4 / 65.7,
  // outright trees of 26 15.2 / 15.8; 12: 17.4 / 17.4, 30.5 / 66.8, 16.8 / 15.2; 16:
  // 24.2 / 18.4, 34.4 / 67.4, 23.0 / 15.7; 48: 61.9 / 25.5, 104 / 91, 58.6 / 21.0.  The
  // border is where the first form's CTAs stop fitting at once, which suits chains; trees
  // with siblings to reject would gain from it up to about 32 sequences, but what a batch
  // holds is not known to the host
  const int n = a.t.n_seqs;
  if (n > 0x7fffffff / VF_MAX_CLUSTER) return arg_err("n_seqs");
  if (n * 16 <= 148) {
    static std::atomic<unsigned long long> devs{0};
    if (int rc = wide_cluster_once(verify_kernel<512, 1, 5, true>, devs, "verification cluster attribute"))
      return rc;
    return launch_pdl(verify_kernel<512, 1, 5, true>, dim3(n * 16), dim3(512), 0, st, 16,
                      "draft verification launch", a);
  }
  int cluster = 8;
  while (cluster > 1 && n * (long long)cluster > 148 * 4) cluster /= 2;
  return launch_pdl(verify_kernel<256, 4, 2, false>, dim3(n * cluster), dim3(256), 0, st, cluster,
                    "draft verification launch", a);
}

}  // namespace tb

extern "C" {

int tb_verify_drafts_greedy(const int* ids, const int* parents, const int* q_start,
                            const int* q_len, int n_seqs, int n_rows, int max_q,
                            const int* target_ids, int* n_accepted, int* path, int path_ld,
                            int path_w, int* next_ids, void* stream) {
  const tb::TreeArgs t{ids, parents, q_start, q_len, n_seqs, n_rows,
                       n_accepted, path, next_ids, path_ld, path_w};
  return tb::verify_greedy_launch(t, target_ids, max_q, static_cast<cudaStream_t>(stream));
}

int tb_verify_drafts(const int* ids, const int* parents, const int* q_start, const int* q_len,
                     int n_seqs, int n_rows, int max_q, const float* probs, long long ld_probs,
                     int vocab, const float* draft_probs, long long ld_draft, int n_draft_rows,
                     const int* draft_rows, const float* uniforms, int* n_accepted, int* path,
                     int path_ld, int path_w, int* next_ids, void* stream) {
  tb::VerifyArgs a{};
  a.t = tb::TreeArgs{ids, parents, q_start, q_len, n_seqs, n_rows,
                     n_accepted, path, next_ids, path_ld, path_w};
  a.probs = probs;
  a.ld_p = ld_probs;
  a.vocab = vocab;
  a.draft_probs = draft_probs;
  a.ld_d = ld_draft;
  a.n_draft_rows = n_draft_rows;
  a.draft_rows = draft_rows;
  a.uniforms = uniforms;
  return tb::verify_launch(a, max_q, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
