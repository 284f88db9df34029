// Append of the accepted path of a verified token tree to the KV caches of all layers, sm_100a.
//
// Row i < counts[b] of sequence b's path: cache[layer][b, h, lens[b] + i] = tree[layer][b, h,
// path[b, i]], keys and values, every layer in one launch; new_lens[b] = lens[b] + counts[b].
// A path entry outside [0, N), or a row outside [0, capacity), is skipped and sets the range bit
// of the device status, as the other appends do. new_lens counts the rows before the first one
// that does not fit the capacity; the row of a skipped path entry is among them and holds what it held.
//
// 2 * 128 bytes a row: a few hundred kilobytes at most, so latency decides. One block takes one
// (layer, keys or values, sequence) and copies its heads x rows with 8 threads of 16 bytes a row;
// the lengths, counts and path are one dependent load in front of the copies. Measured (B200): 1.9 us
// for 8 layers of one sequence (196 KB read and written), 3.1 us for 8 layers of 32 (7 MB); the call
// from the host takes 9 us, of which four tensors a layer are about four.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace tt {
namespace commit {

constexpr int MAX_LAYERS = 64;   // per launch (pointers travel as kernel parameters)
constexpr int THREADS = 256;

struct Params {
  __nv_bfloat16* cache[2][MAX_LAYERS];       // keys, values: [B, H, C, 64]
  const __nv_bfloat16* tree[2][MAX_LAYERS];  // [B, H, N, 64]
  int64_t c_sb[2], c_sh[2], c_st[2];
  int64_t t_sb[2], t_sh[2], t_st[2];
  const int32_t* path;     // [B, P]
  const int32_t* counts;   // [B]
  const int32_t* lens;     // [B]
  int32_t* new_lens;       // [B], written by the first launch only (else NULL)
  int B, H, N, C, P;
  int layers;
};

__global__ void __launch_bounds__(THREADS) tree_commit_kernel(const __grid_constant__ Params p) {
  const int b = static_cast<int>(blockIdx.x) % p.B;
  const int lk = static_cast<int>(blockIdx.x) / p.B;   // layer * 2 + (keys or values)
  const int kv = lk & 1, layer = lk >> 1;
  wait_for_previous_kernel();
  const int len = p.lens[b];
  const int count = min(max(p.counts[b], 0), p.P);
  // Rows that fit: all of them unless the length is negative or the cache is full.
  const int room = (len < 0 || len > p.C) ? 0 : p.C - len;
  const int rows = min(count, room);
  if (lk == 0 && threadIdx.x == 0) {
    if (p.new_lens != nullptr) p.new_lens[b] = len + rows;
    if (rows < count) atomicOr(&g_tt_status, TT_ERR_RANGE);
  }
  const __nv_bfloat16* src = p.tree[kv][layer] + b * p.t_sb[kv];
  __nv_bfloat16* dst = p.cache[kv][layer] + b * p.c_sb[kv];
  const int piece = threadIdx.x & 7;
  for (int i = threadIdx.x >> 3; i < rows * p.H; i += THREADS / 8) {
    const int h = i / rows, r = i - h * rows;
    const int n = p.path[static_cast<int64_t>(b) * p.P + r];
    if (n < 0 || n >= p.N) {
      atomicOr(&g_tt_status, TT_ERR_RANGE);
      continue;
    }
    const uint4 x = *(reinterpret_cast<const uint4*>(src + h * p.t_sh[kv] + n * p.t_st[kv]) + piece);
    *(reinterpret_cast<uint4*>(dst + h * p.c_sh[kv] + (static_cast<int64_t>(len) + r) * p.c_st[kv]) +
      piece) = x;
  }
}

}  // namespace commit
}  // namespace tt
