// pack.hip — the tables of a packed pass over prompts of different lengths,
// built on the GPU from the request lengths.
//
// With new[b] tokens of sequence b behind cached[b] cached ones:
//   starts[b] = sum of new[0..b)               (first packed token; starts[B] = all)
//   seq[i]    = the b with starts[b] <= i < starts[b + 1]
//   pos[i]    = cached[b] + i - starts[b]      (cache row and rotary position)
//   tiles     = blocks of up to `bt` consecutive tokens of one sequence, the one
//               with most keys first: (first packed token, tokens, b, cached + offset)
// Every workgroup scans the lengths itself (at most 4096, in LDS) and then writes
// its own tokens, so one launch does it all; the last workgroup writes the tiles.
// Memory would need 12 bytes per token; what a call takes is its launch and the
// scan's latency.
#include "common.h"

#include <algorithm>

namespace lap {
namespace {

constexpr int kMaxSeqs = 4096;
constexpr int kPackThreads = 1024;
constexpr int kPackTokens = 4;  // tokens per thread and pass
constexpr int kBuckets = 1024;

struct PackArgs {
  const int32_t* lens;
  const int32_t* cached;  // or null: nothing cached
  int B, total, bt, n_tiles;
  int32_t* starts;
  int32_t* seq;
  int64_t* pos;
  int4* tiles;  // or null
};

// Inclusive scan over the workgroup's 1024 values.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t u = __shfl_up((long long)v, d, 64);
    if (lane >= d) v += u;
  }
  __syncthreads();  // s_wave may still be read by an earlier scan
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += s_wave[w];
  return v;
}

// The last b in [0, B) with at[b] <= i (at ascending, at[0] = 0).
__device__ __forceinline__ int find(const int* at, int B, int i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kPackThreads) void pack_kernel(PackArgs a) {
  __shared__ int s_at[kMaxSeqs + 1], s_tile[kMaxSeqs + 1], s_hist[kBuckets];
  __shared__ int64_t s_wave[kPackThreads / 64];
  __shared__ int s_top;
  const int tid = threadIdx.x;
  const bool tiles = a.tiles && blockIdx.x == gridDim.x - 1;
  if (tid == 0) s_top = 0;
  __syncthreads();
  int sum = 0, tsum = 0;
  for (int b0 = 0; b0 < a.B; b0 += kPackThreads) {
    const int b = b0 + tid;
    // a length below zero counts as zero, and what passes `total` is cut off, so
    // that no table can address past its end
    const int n = b < a.B ? max(a.lens[b], 0) : 0;
    const int64_t end = sum + block_scan(min(n, a.total), s_wave);
    const int hi = (int)min(end, (int64_t)a.total);
    const int lo = (int)min(end - min(n, a.total), (int64_t)a.total);
    if (b < a.B) s_at[b] = lo;
    if (b == a.B - 1) s_at[a.B] = hi;
    if (tiles) {
      const int t = (hi - lo + a.bt - 1) / a.bt, tend = tsum + (int)block_scan(t, s_wave);
      if (b < a.B) {
        s_tile[b] = tend - t;
        if (hi > lo) atomicMax(&s_top, (a.cached ? max(a.cached[b], 0) : 0) + hi - lo);
      }
      if (b == a.B - 1) s_tile[a.B] = tend;
      __syncthreads();
      if (tid == kPackThreads - 1) s_wave[0] = tend;
      __syncthreads();
      tsum = (int)s_wave[0];
    }
    __syncthreads();
    if (tid == kPackThreads - 1) s_wave[0] = hi;
    __syncthreads();
    sum = (int)s_wave[0];
  }
  if (tiles) {
    const int n = min(s_tile[a.B], a.n_tiles);
    const int64_t top = s_top;
    for (int i = tid; i < kBuckets; i += kPackThreads) s_hist[i] = 0;
    __syncthreads();
    // counting sort by the keys of a tile, most first; tiles of one bucket may
    // come in any order, they do not depend on each other
    auto tile = [&](int t, int& bucket) {
      const int b = find(s_tile, a.B, t);
      const int off = (t - s_tile[b]) * a.bt;
      const int have = a.cached ? max(a.cached[b], 0) : 0;
      const int cnt = min(a.bt, s_at[b + 1] - s_at[b] - off);
      bucket = kBuckets - 1 - (int)((int64_t)(have + off + cnt) * (kBuckets - 1) / max(top, (int64_t)1));
      bucket = min(max(bucket, 0), kBuckets - 1);
      return make_int4(s_at[b] + off, cnt, b, have + off);
    };
    int bk;
    for (int t = tid; t < n; t += kPackThreads) {
      tile(t, bk);
      atomicAdd(&s_hist[bk], 1);
    }
    __syncthreads();
    const int c = s_hist[tid];
    const int at = (int)block_scan(c, s_wave) - c;
    __syncthreads();
    s_hist[tid] = at;
    __syncthreads();
    for (int t = tid; t < n; t += kPackThreads) {
      const int4 v = tile(t, bk);
      a.tiles[atomicAdd(&s_hist[bk], 1)] = v;
    }
    for (int t = n + tid; t < a.n_tiles; t += kPackThreads) a.tiles[t] = make_int4(0, 0, 0, 0);
    return;
  }
  if (blockIdx.x == 0)
    for (int b = tid; b <= a.B; b += kPackThreads) a.starts[b] = s_at[b];
  const int i0 = (blockIdx.x * kPackThreads + tid) * kPackTokens;
  if (i0 >= a.total) return;
  int b = find(s_at, a.B, i0);
#pragma unroll
  for (int e = 0; e < kPackTokens; ++e) {
    const int i = i0 + e;
    if (i >= a.total) break;
    while (b < a.B - 1 && s_at[b + 1] <= i) ++b;
    const bool in = i < s_at[a.B];  // behind the last sequence: no sequence
    a.seq[i] = in ? b : -1;
    a.pos[i] = in ? (int64_t)(a.cached ? max(a.cached[b], 0) : 0) + i - s_at[b] : 0;
  }
}

}  // namespace
}  // namespace lap

using namespace lap;

extern "C" int lap_pack_prompts(const int32_t* new_lens, const int32_t* cached_lens, int B,
                                int total, int tokens_per_tile, int n_tiles, int32_t* starts,
                                int32_t* seq, int64_t* pos, int32_t* tiles, lap_stream_t stream) {
  clear_error();
  LAP_CHECK(new_lens && starts && (total == 0 || (seq && pos)), "lap_pack_prompts: null pointer");
  LAP_CHECK(B > 0 && total >= 0 && total <= (1 << 30), "lap_pack_prompts: bad sizes");
  LAP_CHECK_CODE(B <= kMaxSeqs, LAP_ERR_UNSUPPORTED, "lap_pack_prompts: %d sequences, at most %d",
                 B, kMaxSeqs);
  LAP_CHECK(!tiles || (tokens_per_tile > 0 && n_tiles >= 0 &&
                       (int64_t)n_tiles >= (int64_t)total / tokens_per_tile + std::min(B, total)),
            "lap_pack_prompts: n_tiles must be at least total / tokens_per_tile + min(B, total)");
  LAP_CHECK((reinterpret_cast<uintptr_t>(tiles) & 15) == 0, "lap_pack_prompts: tiles 16-byte aligned");
  PackArgs a{new_lens, cached_lens, B, total, tokens_per_tile, n_tiles, starts, seq, pos,
             reinterpret_cast<int4*>(tiles)};
  const int per = kPackThreads * kPackTokens;
  const int blocks = std::max(1, (total + per - 1) / per) + (tiles ? 1 : 0);
  hipLaunchKernelGGL(pack_kernel, dim3(blocks), dim3(kPackThreads), 0, as_stream(stream), a);
  LAP_LAUNCH_CHECK("pack_kernel");
  return LAP_OK;
}
