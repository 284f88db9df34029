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
// p, q are clamped to [0, 1] (NaN to 0), so that sums of up to 2^22 weights fit 63 bits. Rounding the
// weights moves a probability by less than 2^-36. The random numbers are FP32, 2^-24 apart as generators
// draw them, which weighs more: the drawn token's probabilities move by less than 2^-24 each (V 2^-24
// together, 0.8 % at 128000 tokens), and a token below 2^-24 may never be drawn.
//
// One thread-block cluster walks one sequence, every CTA taking the same walk. All accept tests
// before a rejection need only p(t) and q(t) of the nodes, gathered once for the whole tree; the
// rows themselves are read at a rejection and at the end, each CTA summing its share of the
// vocabulary in windows of 128 tokens, one a warp. A pass is latency, not bandwidth: many warps with
// four tokens a lane (with 16 a lane the dependent whole-number steps of one warp took 10000 cycles),
// the next two windows' loads under this one's sums. The rejections at a node are a short list of S_k,
// so r_k is folded from p and q as they are read and never stored; with chosen children (no q) a
// rejection changes one weight, so the row is summed once per node. The window sums of the last pass
// locate the next token: one window is read again.
//
// Measured (B200): 5.6 us for one sequence, 8 nodes, 8192 tokens (a chain of loads: the tree, p and q of
// its tokens, the row, the window); 11.1 us for 32 sequences of 16 nodes in threes, where some reject
// three siblings (a pass each); 10.5 us for 5 x 50257 tokens, chosen children (a pass for each node at
// which one is rejected, on 40 CTAs, with 4-byte loads; at 64 registers this variant spills 120-136 bytes, the
// one with draft probabilities 16-28); 32 us for 32 x 128000
// (39 MB read; up to three passes of 8-10 us, the first from DRAM with 64 KiB a SM in flight, a second
// rejection's bound by its FP64 and whole-number steps).
#pragma once

#include <cstdint>

#include "sm100_ptx.cuh"

namespace tt {
namespace verify {

constexpr int MAX_NODES = 256;
constexpr int MAX_THREADS = 512;         // a warp per window, up to 16; two CTAs per SM
constexpr int LANE_TOKENS = 4;
constexpr int WINDOW = 128;              // tokens per window: a warp's
static_assert(WINDOW == 32 * LANE_TOKENS, "a window is what a warp reads at a time");
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

// (The window sums of the last pass are the dynamic shared memory, windows x 8 bytes.)
struct Smem {
  int32_t parent[MAX_NODES];
  int32_t token[MAX_NODES];     // -1: outside the vocabulary
  float u[MAX_NODES];
  float pt[MAX_NODES], qt[MAX_NODES];  // p and q of the node's token at its parent
  int32_t path[MAX_NODES];
  // Rejections at the current node, S_k and token. Every thread writes every entry itself (all the
  // same), so no barrier is needed to read them; a node's list goes to the other half than the last
  // one's, which slower threads may still read (each list has a pass and its barrier behind it).
  unsigned long long S[2][MAX_NODES];
  double Sd[2][MAX_NODES];       // the same in FP64
  long long lost[2][MAX_NODES];  // what r lost at that token (chosen children)
  int32_t rejected[2][MAX_NODES];
  unsigned long long share[2][MAX_CLUSTER];  // the cluster's sums, by pass parity
};

extern __shared__ unsigned long long window_sums[];
// Beside Smem more than the default 48 KiB (from 3569 windows a CTA on): the host opts in. Two CTAs
// per SM in any case, each with the 1 KiB that the system takes.
constexpr size_t kMaxDynamicSmem = MAX_WINDOWS * sizeof(unsigned long long);
static_assert(2 * (sizeof(Smem) + kMaxDynamicSmem + 1024) <= 228 * 1024, "two CTAs per SM");

__device__ __forceinline__ float clamp_prob(float x) { return __saturatef(x); }

// floor(x ONE) for 0 <= x <= 1 as high * 2^16 + low, each a whole number plus MAGIC's bits: 2^23 + y,
// rounded down, holds floor(y) in its low bits, and what the first sum leaves is exact. Four FP32
// operations (a conversion to 64 bits runs at 16 a clock and SM; shifting the significand into place
// took 20 operations a value, and a pass over 16384 tokens 12000 cycles).
constexpr float MAGIC = 8388608.f;  // 2^23
struct Fixed {
  uint32_t high, low;
};
__device__ __forceinline__ Fixed fixed_point(float x) {
  const float h = __fmaf_rd(x, 1048576.f, MAGIC);
  const float rest = __fmaf_rn(x, 1048576.f, -__fadd_rn(h, -MAGIC));
  return Fixed{__float_as_uint(h), __float_as_uint(__fmaf_rd(rest, 65536.f, MAGIC))};
}
__device__ __forceinline__ long long weight(float x) {
  const Fixed f = fixed_point(x);
  const uint32_t magic = __float_as_uint(MAGIC);
  return (static_cast<long long>(f.high - magic) << 16) + static_cast<long long>(f.low - magic);
}

// floor(fl(x S)) for a whole number S, fl the FP64 rounding.
__device__ __forceinline__ long long scaled(float x, unsigned long long S) {
  return __double2ll_rd(__dmul_rn(static_cast<double>(x), static_cast<double>(S)));
}

// x 2^E for 0 <= x <= 1 by moving x's bits into an FP64 (a zero or subnormal x becomes some number
// far below 1): conversion instructions run at 16 a clock and SM.
template <int E>
__device__ __forceinline__ double to_double(float x) {
  const uint32_t bits = __float_as_uint(x);
  return __hiloint2double(static_cast<int>((bits >> 3) + ((896u + E) << 20)),
                          static_cast<int>(bits << 29));
}

// max(r_0 - floor(q S_0) - ... - floor(q S_(K-1)), 0), which is r_K (what is taken off is never
// negative), exact in FP64 below S = 2^51: 2^52 + y, rounded down, is 2^52 + floor(y).
__device__ __forceinline__ double residual_fp64(float p, float q, int K, double S1,
                                                const double* S) {
  constexpr double M = 4503599627370496.0;  // 2^52
  double r = __dadd_rn(__dadd_rd(to_double<36>(p), M), -__dadd_rd(to_double<36>(q), M));
  const double d = to_double<0>(q);
  r = __dadd_rn(r, __dadd_rn(M, -__dadd_rd(__dmul_rn(d, S1), M)));
  for (int k = 2; k < K; ++k)
    r = __dadd_rn(r, __dadd_rn(M, -__dadd_rd(__dmul_rn(d, S[k]), M)));
  const int sign = ~(__double2hiint(r) >> 31);  // negative: zero
  return __hiloint2double(__double2hiint(r) & sign, __double2loint(r) & sign);
}

// r_K of token v from its p and q, after the K rejections in list `half`.
template <bool DENSE>
__device__ __forceinline__ long long residual(const Smem& s, int half, int K, int v, float p, float q) {
  long long r = weight(p);
  if (K == 0) return r;
  if (DENSE) {
    r = max(r - weight(q), 0ll);  // S_0 = ONE
    for (int k = 1; k < K; ++k) r = max(r - scaled(q, s.S[half][k]), 0ll);
  } else {
    for (int k = 0; k < K; ++k)
      if (v == s.rejected[half][k])
        r = max(r - static_cast<long long>(s.S[half][k]), 0ll);
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

// p and (after a rejection) q of one lane's 4 tokens of the window at v0, zero past the vocabulary.
// VEC (rows on 16-byte boundaries, V % 4 == 0): value j is token 4 lane + j of the window, else token
// 32 j + lane; both keep every load of a warp contiguous.
template <bool VEC>
__device__ __forceinline__ int token_of(int lane, int j) {
  return VEC ? lane * 4 + j : j * 32 + lane;
}
template <bool VEC>
__device__ __forceinline__ void load_lane(const float* row, int v0, int lane, int V,
                                          float (&x)[LANE_TOKENS]) {
  if (VEC) {
    const int v = v0 + lane * 4;
    const float4 y = v < V ? *reinterpret_cast<const float4*>(row + v)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
    x[0] = y.x;
    x[1] = y.y;
    x[2] = y.z;
    x[3] = y.w;
  } else {
#pragma unroll
    for (int j = 0; j < LANE_TOKENS; ++j) {
      const int v = v0 + j * 32 + lane;
      x[j] = v < V ? row[v] : 0.f;
    }
  }
}

// One pass over the rows of node `cur`: this CTA's window sums of r_K, and the sum over all CTAs
// (whole numbers: the same in every CTA). Every thread of every CTA of the cluster calls it.
template <bool DENSE, bool VEC>
__device__ __forceinline__ unsigned long long sum_pass(Smem& s, const Params& a, int b, int cur,
                                                       int half, int K, int rank, int pass) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, par = pass & 1;
  const float* prow = a.p + b * a.p_sb + cur * a.p_sn;
  const float* qrow = DENSE ? a.q + b * a.q_sb + cur * a.q_sn : nullptr;
  const int step = static_cast<int>(blockDim.x >> 5);
  const bool with_q = DENSE && K > 0;
  // Products of this size of S keep the FP64 form exact (a row of probabilities has S <= 2^36).
  const bool fp64_exact = !with_q || K == 1 || s.S[half][1] < (1ull << 51);
  const double S1 = with_q && K > 1 ? s.Sd[half][1] : 0.0;
  // Sum of r_K over one lane's tokens of the window at v0.
  auto lane_sum = [&](const float (&ps)[LANE_TOKENS], const float (&qs)[LANE_TOKENS], int v0) {
    long long sum = 0;
    if (with_q && K == 1) {
      // max(w(p) - w(q), 0) is the difference where p > q (w does not decrease), else zero.
      int high = 0, low = 0;
#pragma unroll
      for (int j = 0; j < LANE_TOKENS; ++j) {
        const float pj = clamp_prob(ps[j]), qj = clamp_prob(qs[j]);
        const Fixed fp = fixed_point(pj), fq = fixed_point(qj);
        high += pj > qj ? static_cast<int>(fp.high - fq.high) : 0;
        low += pj > qj ? static_cast<int>(fp.low - fq.low) : 0;
      }
      sum = static_cast<long long>(high) * 65536 + low;
    } else if (with_q && fp64_exact) {
      double total = 0.0;
#pragma unroll
      for (int j = 0; j < LANE_TOKENS; ++j)
        total = __dadd_rn(total, residual_fp64(clamp_prob(ps[j]), clamp_prob(qs[j]), K, S1, s.Sd[half]));
      sum = __double2ll_rn(total);
    } else if (with_q) {
#pragma unroll 1
      for (int j = 0; j < LANE_TOKENS; ++j) {
        const float pj = j == 0 ? ps[0] : j == 1 ? ps[1] : j == 2 ? ps[2] : ps[3];
        const float qj = j == 0 ? qs[0] : j == 1 ? qs[1] : j == 2 ? qs[2] : qs[3];
        sum += residual<DENSE>(s, half, K, 0, clamp_prob(pj), clamp_prob(qj));
      }
    } else {
      uint32_t high = 0, low = 0;
#pragma unroll
      for (int j = 0; j < LANE_TOKENS; ++j) {
        const Fixed f = fixed_point(clamp_prob(ps[j]));
        high += f.high - __float_as_uint(MAGIC);
        low += f.low - __float_as_uint(MAGIC);
      }
      sum = (static_cast<long long>(high) << 16) + low;
      if (!DENSE) {
        for (int k = 0; k < K; ++k) {
          // The rejected token's weight, where this lane has it: S_k taken off, down to zero.
          const int at = s.rejected[half][k] - v0;
#pragma unroll
          for (int j = 0; j < LANE_TOKENS; ++j)
            if (at == token_of<VEC>(lane, j)) {
              const float pj = clamp_prob(ps[j]);
              sum += residual<DENSE>(s, half, k + 1, v0 + at, pj, 0.f) -
                     residual<DENSE>(s, half, k, v0 + at, pj, 0.f);
            }
        }
      }
    }
    return sum;
  };
  // Two windows at a time, the next two's loads under their sums.
  float ps[2][LANE_TOKENS], qs[2][LANE_TOKENS], pn[2][LANE_TOKENS], qn[2][LANE_TOKENS];
  auto request = [&](int w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // A window past this CTA's share is past the row for these loads.
      const int v0 = w + i * step < a.windows ? (rank * a.windows + w + i * step) * WINDOW : a.V;
      load_lane<VEC>(prow, v0, lane, a.V, pn[i]);
      if (with_q) load_lane<VEC>(qrow, v0, lane, a.V, qn[i]);
    }
  };
  request(warp);
  for (int w = warp; w < a.windows; w += 2 * step) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < LANE_TOKENS; ++j) {
        ps[i][j] = pn[i][j];
        qs[i][j] = qn[i][j];
      }
    if (w + 2 * step < a.windows) request(w + 2 * step);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = w + i * step;
      if (at >= a.windows) break;
      const unsigned long long all = warp_sum(static_cast<unsigned long long>(
          lane_sum(ps[i], qs[i], (rank * a.windows + at) * WINDOW)));
      if (lane == 0) window_sums[at] = all;
    }
  }
  __syncthreads();
  unsigned long long total = 0;
  if (warp == 0) {
    for (int w = lane; w < a.windows; w += 32) total += window_sums[w];
    total = warp_sum(total);
    if (a.cluster == 1) {
      if (lane == 0) s.share[par][0] = total;
    } else if (lane < a.cluster) {
      st_cluster_u64(map_to_rank(smem_u32(&s.share[par][rank]), lane), total);
    }
  }
  __syncwarp();  // cluster barriers take whole warps
  if (a.cluster == 1) __syncthreads();
  else cluster_sync();
  total = 0;
  for (int c = 0; c < a.cluster; ++c) total += s.share[par][c];
  return total;
}

template <bool DENSE, bool VEC>
__global__ void __launch_bounds__(MAX_THREADS, 2) tree_verify_kernel(const Params a) {
  __shared__ Smem s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = static_cast<int>(cluster_ctarank());
  const int b = static_cast<int>(blockIdx.x) / a.cluster;
  const int N = a.N;

  wait_for_previous_kernel();
  // The tree, the random numbers, and p(t), q(t) of every node at its parent.
  for (int n = threadIdx.x; n < N; n += blockDim.x) {
    const int up = a.parents[b * a.parents_sb + n];
    const int64_t t = a.tokens[static_cast<int64_t>(b) * N + n];
    const bool child = up >= 0 && up < n;
    const bool known = t >= 0 && t < a.V;
    s.parent[n] = child ? up : (up == -1 ? -1 : -2);
    s.token[n] = known ? static_cast<int32_t>(t) : -1;
    s.u[n] = a.u[static_cast<int64_t>(b) * N + n];
    float pt = 0.f, qt = 0.f;
    if (child && known) {
      pt = clamp_prob(a.p[b * a.p_sb + up * a.p_sn + t]);
      qt = DENSE ? clamp_prob(a.q[b * a.q_sb + up * a.q_sn + t]) : 1.f;
    } else if (!DENSE) {
      qt = 1.f;
    }
    s.pt[n] = pt;
    s.qt[n] = qt;
  }
  // Also: no CTA writes another's shared memory before that CTA has started.
  __syncwarp();
  if (a.cluster == 1) __syncthreads();
  else cluster_sync();

  const bool in_use = s.parent[0] == -1;
  int cur = 0, count = in_use ? 1 : 0, passes = 0;
  int K = 0, half = 0;       // rejections at this node, and where their list is
  bool summed = false;       // `total` is the sum of r_K
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
    const int token = s.token[c];
    long long r = 0;  // r_K of the child's token
    bool take;
    if (K == 0) {
      take = __fmul_rn(s.u[c], qt) < pt;
      r = weight(pt);
    } else {
      r = residual<DENSE>(s, half, K, token, pt, qt);
      take = __dmul_rn(__dmul_rn(static_cast<double>(s.u[c]), static_cast<double>(qt)),
                       static_cast<double>(total)) < static_cast<double>(r);
    }
    if (take) {
      cur = c;
      if (threadIdx.x == 0) s.path[count] = c;
      ++count;
      K = 0;
      summed = false;
      continue;
    }
    if (K == 0) half ^= 1;
    const unsigned long long S = K == 0 ? static_cast<unsigned long long>(ONE) : total;
    s.S[half][K] = S;
    s.Sd[half][K] = static_cast<double>(S);
    s.rejected[half][K] = token;
    __syncwarp();
    ++K;
    if (DENSE || !summed) {
      total = sum_pass<DENSE, VEC>(s, a, b, cur, half, K, rank, passes++);
      summed = true;
    } else {
      // One weight has changed, and the sum by as much (the last pass's windows: at the end).
      const long long lost = r - max(r - static_cast<long long>(S), 0ll);
      s.lost[half][K - 1] = lost;
      total -= static_cast<unsigned long long>(lost);
    }
  }
  if (in_use && K == 0) total = sum_pass<DENSE, VEC>(s, a, b, cur, half, 0, rank, passes++);
  if (in_use && K > 0 && total == 0) {
    K = 0;
    total = sum_pass<DENSE, VEC>(s, a, b, cur, half, 0, rank, passes++);
  }

  if (rank == 0) {
    __syncthreads();
    for (int n = threadIdx.x; n < N; n += blockDim.x)
      a.path[static_cast<int64_t>(b) * N + n] = n < count ? s.path[n] : -1;
    if (threadIdx.x == 0) {
      a.counts[b] = count;
      if (total == 0) a.next[b] = -1;  // not in use, or no token has any weight
    }
  }
  if (warp != 0 || total == 0) return;

  // The CTA, then the window, then the token in which the running sum passes the goal.
  const int par = (passes - 1) & 1;
  unsigned long long goal = 0;
  {
    const double x = floor(__dmul_rn(static_cast<double>(s.u[0]), static_cast<double>(total)));
    goal = x > 0.0 ? (x < static_cast<double>(total) ? static_cast<unsigned long long>(x) : total - 1)
                   : 0ull;
  }
  // Chosen children rejected after the pass at this node: what the sums of their windows lost since.
  const int later = DENSE ? 0 : K;
  auto lost_in = [&](int from, int to) {  // windows [from, to) of the row
    unsigned long long x = 0;
    for (int k = 1; k < later; ++k) {
      const int t = s.rejected[half][k];
      if (t >= from * WINDOW && t < to * WINDOW) x += static_cast<unsigned long long>(s.lost[half][k]);
    }
    return x;
  };
  __syncwarp();
  unsigned long long before = 0;
  for (int c = 0; c < rank; ++c) before += s.share[par][c];
  before -= lost_in(0, rank * a.windows);
  const unsigned long long own =
      s.share[par][rank] - lost_in(rank * a.windows, (rank + 1) * a.windows);
  if (goal < before || goal >= before + own) return;
  goal -= before;
  auto scan = [&](unsigned long long x) {  // running sum over the lanes
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, x, off);
      if (lane >= off) x += y;
    }
    return x;
  };
  int win = 0;
  for (int base = 0; base < a.windows; base += 32) {
    const int w = base + lane;
    const int at_row = rank * a.windows + w;
    const unsigned long long x =
        w < a.windows ? window_sums[w] - lost_in(at_row, at_row + 1) : 0ull;
    const unsigned long long run = scan(x);
    const unsigned hit = __ballot_sync(0xffffffffu, run > goal);
    if (hit != 0) {
      const int first = __ffs(hit) - 1;
      goal -= __shfl_sync(0xffffffffu, run - x, first);
      win = base + first;
      break;
    }
    goal -= __shfl_sync(0xffffffffu, run, 31);
  }
  const float* prow = a.p + b * a.p_sb + cur * a.p_sn;
  const float* qrow = DENSE ? a.q + b * a.q_sb + cur * a.q_sn : nullptr;
  const int v0 = (rank * a.windows + win) * WINDOW;
  float ps[LANE_TOKENS], qs[LANE_TOKENS];
  load_lane<VEC>(prow, v0, lane, a.V, ps);
  if (DENSE && K > 0) {
    load_lane<VEC>(qrow, v0, lane, a.V, qs);
  } else {
#pragma unroll
    for (int j = 0; j < LANE_TOKENS; ++j) qs[j] = 0.f;
  }
  constexpr int GROUP = VEC ? LANE_TOKENS : 1;  // adjacent tokens of a lane
#pragma unroll
  for (int i = 0; i < LANE_TOKENS; i += GROUP) {
    unsigned long long r[GROUP], x = 0;
#pragma unroll
    for (int j = 0; j < GROUP; ++j) {
      r[j] = static_cast<unsigned long long>(
          residual<DENSE>(s, half, K, v0 + token_of<VEC>(lane, i + j), clamp_prob(ps[i + j]),
                          clamp_prob(qs[i + j])));
      x += r[j];
    }
    const unsigned long long run = scan(x);
    const unsigned hit = __ballot_sync(0xffffffffu, run > goal);
    if (hit != 0) {
      if (lane == __ffs(hit) - 1) {
        unsigned long long left = goal - (run - x);
        int j = 0;
#pragma unroll
        for (int k = 0; k + 1 < GROUP; ++k)
          if (j == k && left >= r[k]) {
            left -= r[k];
            ++j;
          }
        a.next[b] = v0 + token_of<VEC>(lane, i + j);
      }
      return;
    }
    goal -= __shfl_sync(0xffffffffu, run, 31);
  }
}

}  // namespace verify
}  // namespace tt
