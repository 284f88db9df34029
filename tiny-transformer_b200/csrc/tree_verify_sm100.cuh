// Verification of a tree of drafted tokens against the target's probabilities for sm_100a
// (speculative sampling with given random numbers).
//
// From node 0 (the last committed token) the walk tries the children of the current node in index
// order. With p, q the target's and the draft's distribution at the current node, child c with
// token t is accepted with probability min(1, p(t) / q(t)), else p becomes max(p - q, 0)
// renormalised and the next child is tried; when none is accepted, the next token is drawn from
// what is left of p. Without draft probabilities q is 1 at the child's token and 0 elsewhere.
//
// The weights are whole numbers, so that no sum depends on its order and every split of a row
// over threads and CTAs takes the same decisions. With ONE = 2^36:
//   r_0(v) = floor(p(v) ONE), S_0 = ONE;
//   child c is accepted iff u_c q(t) < p(t) in FP32 (no child rejected here yet), or
//   u_c q(t) S_k < r_k(t) in FP64 (after k rejections);
//   r_{k+1}(v) = max(r_k(v) - floor(q(v) S_k), 0), S_{k+1} = sum of r_{k+1};
//   next token: the smallest v whose running sum of r exceeds floor(u_0 * sum of r); r is r_0
//   again where nothing is left of it.
// p, q are clamped to [0, 2] (NaN to 0), so that sums of up to 2^22 weights fit 63 bits.
//
// One thread-block cluster walks one sequence. Every CTA takes the same walk: all accept tests
// before a rejection need only p(t) and q(t) of the nodes, gathered once for the whole tree; the
// rows themselves are read only at a rejection and at the end, each CTA summing its share of the
// vocabulary in windows of 128 tokens and the cluster adding the shares through distributed
// shared memory. The rejections at a node are a short list of S_k, so r_k is folded from p and q
// as they are read (again from L2 after a second rejection) and never stored. The window sums of
// the last pass locate the next token: one window is read again.
#pragma once

#include <cstdint>

#include "sm100_ptx.cuh"

namespace tt {
namespace verify {

constexpr int MAX_NODES = 256;
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int WINDOW = 128;              // tokens per window: 4 per lane
constexpr int MAX_CLUSTER = 8;
constexpr int MAX_WINDOWS = 4096;        // per CTA
constexpr int64_t MAX_VOCAB = int64_t(1) << 22;  // = MAX_CLUSTER * MAX_WINDOWS * WINDOW
constexpr double ONE = 68719476736.0;    // 2^36

struct Params {
  const int64_t* tokens;   // [B, N]
  const int32_t* parents;  // [N] (stride 0) or [B, N]
  int64_t parents_sb;
  const float* p;          // [B, N, V], unit last stride
  int64_t p_sb, p_sn;
  const float* q;          // optional, likewise
  int64_t q_sb, q_sn;
  const float* u;          // [B, N]
  int B, N, V;
  int cluster;             // CTAs per sequence
  int windows;             // windows per CTA
  int32_t* path;           // [B, N]
  int32_t* counts;         // [B]
  int64_t* next;           // [B]
};

struct Smem {
  int32_t parent[MAX_NODES];
  int32_t token[MAX_NODES];     // -1: outside the vocabulary
  float u[MAX_NODES];
  float pt[MAX_NODES], qt[MAX_NODES];  // p and q of the node's token at its parent
  int32_t path[MAX_NODES];
  double S[MAX_NODES];          // S_k of the rejections at the current node
  int32_t rejected[MAX_NODES];  // their tokens
  unsigned long long window[MAX_WINDOWS];
  unsigned long long part[WARPS];
  unsigned long long share[2][MAX_CLUSTER];  // the cluster's sums, by pass parity
};

__device__ __forceinline__ float clamp_prob(float x) { return fminf(fmaxf(x, 0.f), 2.f); }

// floor(x * S) for 0 <= x <= 2, S a whole number below 2^53.
__device__ __forceinline__ long long scaled(float x, double S) {
  return __double2ll_rd(__dmul_rn(static_cast<double>(x), S));
}

// r_K of token v from its p and q, after the K rejections listed in s.
template <bool DENSE>
__device__ __forceinline__ long long residual(const Smem& s, int K, int v, float p, float q) {
  long long r = scaled(p, ONE);
  for (int k = 0; k < K; ++k) {
    const float qk = DENSE ? q : (v == s.rejected[k] ? 1.f : 0.f);
    const long long left = r - scaled(qk, s.S[k]);
    r = left > 0 ? left : 0;
  }
  return r;
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// One pass over the rows of node `cur`: this CTA's window sums of r_K, and the sum over all CTAs
// (whole numbers: the same in every CTA). Every thread of every CTA of the cluster calls it.
template <bool DENSE, bool VEC>
__device__ __forceinline__ unsigned long long sum_pass(Smem& s, const Params& a, int b, int cur,
                                                       int K, int rank, int pass) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* prow = a.p + b * a.p_sb + cur * a.p_sn;
  const float* qrow = DENSE ? a.q + b * a.q_sb + cur * a.q_sn : nullptr;
  const bool with_q = DENSE && K > 0;
  unsigned long long mine = 0;
  for (int w = warp; w < a.windows; w += WARPS) {
    const int64_t v0 = (static_cast<int64_t>(rank) * a.windows + w) * WINDOW;
    long long r = 0;
    if (VEC) {
      const int64_t v = v0 + lane * 4;
      if (v < a.V) {  // V % 4 == 0
        const float4 x = *reinterpret_cast<const float4*>(prow + v);
        const float4 y = with_q ? *reinterpret_cast<const float4*>(qrow + v)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
        const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          r += residual<DENSE>(s, K, static_cast<int>(v) + i, clamp_prob(xs[i]), clamp_prob(ys[i]));
      }
    } else {
      float xs[4], ys[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t v = v0 + i * 32 + lane;
        xs[i] = v < a.V ? prow[v] : 0.f;
        ys[i] = with_q && v < a.V ? qrow[v] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        r += residual<DENSE>(s, K, static_cast<int>(v0) + i * 32 + lane, clamp_prob(xs[i]),
                             clamp_prob(ys[i]));
    }
    const unsigned long long sum = warp_sum(static_cast<unsigned long long>(r));
    if (lane == 0) s.window[w] = sum;
    mine += sum;
  }
  if (lane == 0) s.part[warp] = mine;
  __syncthreads();
  unsigned long long total = 0;
  if (warp == 0) {
    total = warp_sum(lane < WARPS ? s.part[lane] : 0ull);
    if (a.cluster == 1) {
      if (lane == 0) s.share[pass & 1][0] = total;
    } else if (lane < a.cluster) {
      st_cluster_u64(map_to_rank(smem_u32(&s.share[pass & 1][rank]), lane), total);
    }
  }
  if (a.cluster == 1) __syncthreads();
  else cluster_sync();
  total = 0;
  for (int c = 0; c < a.cluster; ++c) total += s.share[pass & 1][c];
  return total;
}

template <bool DENSE, bool VEC>
__global__ void __launch_bounds__(THREADS) tree_verify_kernel(const Params a) {
  __shared__ Smem s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  const int b = static_cast<int>(blockIdx.x) / a.cluster;
  const int N = a.N;

  // The tree, the random numbers, and p(t), q(t) of every node at its parent.
  for (int n = threadIdx.x; n < N; n += THREADS) {
    const int up = __ldg(a.parents + b * a.parents_sb + n);
    const int64_t t = __ldg(reinterpret_cast<const long long*>(a.tokens) + static_cast<int64_t>(b) * N + n);
    const bool child = up >= 0 && up < n;
    const bool known = t >= 0 && t < a.V;
    s.parent[n] = child ? up : (up == -1 ? -1 : -2);
    s.token[n] = known ? static_cast<int32_t>(t) : -1;
    s.u[n] = __ldg(a.u + static_cast<int64_t>(b) * N + n);
    float pt = 0.f, qt = 0.f;
    if (child && known) {
      pt = clamp_prob(__ldg(a.p + b * a.p_sb + up * a.p_sn + t));
      qt = DENSE ? clamp_prob(__ldg(a.q + b * a.q_sb + up * a.q_sn + t)) : 1.f;
    }
    s.pt[n] = pt;
    s.qt[n] = qt;
  }
  // Also: no CTA writes another's shared memory before that CTA has started.
  if (a.cluster == 1) __syncthreads();
  else cluster_sync();

  const bool in_use = s.parent[0] == -1;
  int cur = 0, count = in_use ? 1 : 0, K = 0, passes = 0;
  unsigned long long total = 0;
  if (threadIdx.x == 0) s.path[0] = 0;
  int at = 0;  // nodes up to here have been tried
  while (in_use) {
    // The next child of `cur` in index order; every warp finds it by itself.
    int c = -1;
    for (int base = (at + 1) & ~31; base < N; base += 32) {
      const int n = base + lane;
      const unsigned hit = __ballot_sync(0xffffffffu, n > at && n < N && s.parent[n] == cur);
      if (hit != 0) {
        c = base + __ffs(hit) - 1;
        break;
      }
    }
    if (c < 0) break;
    at = c;
    const float pt = s.pt[c], qt = s.qt[c];
    bool take;
    if (K == 0) {
      take = __fmul_rn(s.u[c], qt) < pt;
    } else {
      const long long r = residual<DENSE>(s, K, s.token[c], pt, qt);
      take = __dmul_rn(__dmul_rn(static_cast<double>(s.u[c]), static_cast<double>(qt)),
                       static_cast<double>(total)) < static_cast<double>(r);
    }
    if (take) {
      cur = c;
      if (threadIdx.x == 0) s.path[count] = c;
      ++count;
      K = 0;
      continue;
    }
    __syncthreads();  // every thread has read the list of rejections
    if (threadIdx.x == 0) {
      s.S[K] = K == 0 ? ONE : static_cast<double>(total);
      s.rejected[K] = s.token[c];
    }
    __syncthreads();
    ++K;
    total = sum_pass<DENSE, VEC>(s, a, b, cur, K, rank, passes++);
  }
  if (in_use && K == 0) total = sum_pass<DENSE, VEC>(s, a, b, cur, 0, rank, passes++);
  if (in_use && K > 0 && total == 0) {
    K = 0;
    total = sum_pass<DENSE, VEC>(s, a, b, cur, 0, rank, passes++);
  }

  if (rank == 0) {
    __syncthreads();
    for (int n = threadIdx.x; n < N; n += THREADS)
      a.path[static_cast<int64_t>(b) * N + n] = n < count ? s.path[n] : -1;
    if (threadIdx.x == 0) {
      a.counts[b] = count;
      if (total == 0) a.next[b] = -1;  // not in use, or no token has any weight
    }
  }
  if (warp != 0 || total == 0) return;

  // The CTA, then the window, then the token in which the running sum passes the goal.
  unsigned long long goal = 0;
  {
    const double x = floor(__dmul_rn(static_cast<double>(s.u[0]), static_cast<double>(total)));
    goal = x > 0.0 ? (x < static_cast<double>(total) ? static_cast<unsigned long long>(x) : total - 1)
                   : 0ull;
  }
  unsigned long long before = 0;
  for (int c = 0; c < rank; ++c) before += s.share[(passes - 1) & 1][c];
  if (goal < before || goal >= before + s.share[(passes - 1) & 1][rank]) return;
  goal -= before;
  int win = -1;
  for (int base = 0; base < a.windows; base += 32) {
    const int w = base + lane;
    unsigned long long run = w < a.windows ? s.window[w] : 0ull;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run > goal);
    if (hit != 0) {
      const int first = __ffs(hit) - 1;
      const unsigned long long prev = __shfl_sync(0xffffffffu, run, first > 0 ? first - 1 : 0);
      if (first > 0) goal -= prev;
      win = base + first;
      break;
    }
    goal -= __shfl_sync(0xffffffffu, run, 31);
  }
  const float* prow = a.p + b * a.p_sb + cur * a.p_sn;
  const float* qrow = DENSE ? a.q + b * a.q_sb + cur * a.q_sn : nullptr;
  const int64_t v0 = (static_cast<int64_t>(rank) * a.windows + win) * WINDOW;
#pragma unroll 1
  for (int i = 0; i < 4; ++i) {
    const int64_t v = v0 + i * 32 + lane;
    const float x = v < a.V ? clamp_prob(prow[v]) : 0.f;
    const float y = DENSE && K > 0 && v < a.V ? clamp_prob(qrow[v]) : 0.f;
    unsigned long long run =
        static_cast<unsigned long long>(residual<DENSE>(s, K, static_cast<int>(v), x, y));
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned long long z = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += z;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run > goal);
    if (hit != 0) {
      if (lane == 0) a.next[b] = v0 + i * 32 + __ffs(hit) - 1;
      return;
    }
    goal -= __shfl_sync(0xffffffffu, run, 31);
  }
}

}  // namespace verify
}  // namespace tt
