// prompt.hip — attention of many query rows over a K/V cache: causal attention of
// packed prompts (grouped heads, sequences of different lengths, tokens cached
// before them), and a decode step over a cache whose first tokens are the same in
// every sequence.
//
// Both are, per KV head, a block of rows (a row is one query head of one token) over
// a range of keys:
//   o[r] = sum_{t < lim[r]} 2^(c (q[r].k[t]) - m[r]) v[t] / sum of the same weights,
// c = scale * log2(e), m close to the row's running maximum (one pass over the keys, fp32;
// kSlack and kUp say how close).
//
// Products are 32x32x16 MFMAs with the scores transposed, S^T = K Q^T: a lane then
// holds 16 keys of one query (column lane % 32, keys 8 i + 4 (lane / 32) + e), so a
// row's maximum and sum are lane-local but for one exchange with lane + 32, and the
// weights are, in place, the B operand of o^T = V^T P^T (the reduction's order of
// keys is free as long as V^T's operand uses the same).  V^T comes from the row-major
// V tile through the transposing LDS read.
//
// All query heads of a KV head lie in one block (row = token * G + head): K and V are
// read once for the group, and 32 rows span few tokens, so little of a causal block
// is masked.  A wave skips a tile of keys that none of its rows sees.
//
// K and V tiles are copied straight into LDS, one tile ahead; 252 registers and 64 KB let
// two workgroups share a CU, whose products and exponentials overlap.  One prompt of
// 16384 tokens, 32 query heads on 8, D = 128: 2.03 ms, 1085 TFLOP/s, where a large library
// product reaches 1280 to 1330 on the same card.  The matrix pipe is busy 58 % of the
// cycles and the card runs at 1.79 GHz under this load: saved cycles come back as a lower
// clock (20 % fewer cycles than an earlier form gave 9 % in time).  LDS reads have no bank
// conflicts.  Short prompts wait: a tile takes one workgroup 1.2 us, its start, masked
// tile and end together about 15 us of a 2048-token prompt's 55.
#include "common.h"
#include "attn_core.h"

#include <algorithm>

namespace lap {
namespace {

// Rows of a workgroup: four waves of 32.  (Two waves, or eight, were slower or the same
// at every size: one prompt of 16384 tokens, 32 query heads on 8, D = 128, 3146 and 2065
// us against 2051; of 2048 68 and 67 against 57; of 512 18.3 and 22.8 against 17.8.)
constexpr int NW = 4, kThreads = 64 * NW, kRows = 32 * NW;
constexpr int kGran = 64;  // parts of the keys are multiples of this
// Keys per tile.  At D = 256 a row's o^T takes 128 registers and its query 64: scores and
// weights of 32 keys leave room for operands (64 keys spill: 5922 us against then 3492 for
// a prompt of 16384 tokens with 16 heads).
template <int D>
constexpr int bn() {
  return D == 256 ? 32 : 64;
}
// A lane's byte offset within a tile is 32 bits.
constexpr int kMaxRowStride = 1 << 24;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

#define LAP_LDS __attribute__((address_space(3)))

template <int DT>
__device__ __forceinline__ f32x16 mfma32(i16x8 a, i16x8 b, f32x16 c) {
  if constexpr (DT == LAP_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two weights in the data type, round to nearest even.  The weights enter the second
// product in 16 bits (off by up to half a step, 2^-8 or 2^-11 of each; fp16 below its
// normal range, see kUp); their sum stays fp32.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == LAP_DTYPE_F16) {
    const f16x2 r = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, r);
  } else {
    const bf16x2 r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
  }
}

// Swizzle of a tile row: the row's 16-byte chunks are stored at chunk ^ swz(row).
// 16 rows of one chunk (a K read) then fall in 16 different slots of 256 bytes, and
// 4 rows of 64 contiguous bytes (a V read) in four different quarters.
template <int D>
__device__ __forceinline__ int swz(int row) {
  if constexpr (D == 64) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
  return (row & 3) << 2 | ((row >> 2) & 3);
}

struct FlashArgs {
  const uint16_t* q;
  int64_t q_sb, q_st, q_sh;  // per sequence (uniform form), token, head
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_sb, k_sh, k_st, v_sb, v_sh, v_st;
  int B, Hq, Hkv, G;
  int Tq, Tk;        // query tokens (of a sequence, or packed), cache rows
  const int4* tiles; // packed form
  int bt;            // tokens per tile
  int n_tiles;
  int tps;           // uniform form: tiles per sequence
  int nsplit, per_split;
  float c;           // scale * log2(e)
  uint16_t* out;
  int64_t o_sb, o_st, o_sh;
  float* part_o;     // [rows][nsplit][D]
  float* part_ml;    // [rows][nsplit][2]
  // decode over a shared prefix
  int prefix;             // keys that every sequence shares, read from sequence 0
  int psplit, pblocks;    // splits of the prefix, row blocks of it
  const int32_t* plans;   // lap_row_plan[B] (t_total), or null: Tk keys each
};

// What a workgroup works on.
struct FlashTile {
  const uint16_t* q;   // token 0 of the tile, query head 0 of the KV head
  uint16_t* out;
  int64_t q_st, o_st;  // per token
  int64_t row0;        // row of part_* of token 0, head 0 of the KV head
  const uint16_t* k;   // row 0 of the sequence's keys
  const uint16_t* v;
  int n;               // tokens
  int key0;            // token j sees keys [0, key0 + j + 1), or
  const int32_t* lens; // [0, min(hi, lens[8 j])) where not null
  int lo, hi;          // keys of this workgroup
  int split, parts;    // this part of the keys, and how many hold any (1: no merge)
};

// Copies of key tiles straight into LDS, 16 bytes per lane: a wave writes 1 KB of
// consecutive slots, and the lane's global address undoes the swizzle.  A lane's offset
// within a tile does not change, so a copy costs a base in scalar registers and m0.
template <int D>
struct TileCopy {
  static constexpr int kBN = bn<D>(), C = D / 8, PER = kBN * C / (64 * NW);
  // (at D = 256 the registers are worth more: every copy computes its offset anew, 2374 us
  // against 2430 for a prompt of 16384 tokens with 16 heads)
  static constexpr bool kKeep = D < 256;
  uint32_t off[kKeep ? PER : 1];
  uint32_t st;

  __device__ __forceinline__ void init(int64_t stride, int tid) {
    st = (uint32_t)stride;
    if constexpr (kKeep)
#pragma unroll
      for (int i = 0; i < PER; ++i) off[i] = offset(i, tid, kBN - 1);
  }
  __device__ __forceinline__ uint32_t offset(int i, int tid, int last) const {
    const int slot = (i * NW + (tid >> 6)) * 64 + (tid & 63);
    const int row = slot / C, chunk = (slot % C) ^ swz<D>(row);
    return (min(row, last) * st + chunk * 8) * 2;
  }
  // The tile whose first row is at base; rows past `last` repeat row `last`.
  __device__ __forceinline__ void issue(const char* s_dst, const uint16_t* base, int last,
                                        int tid) const {
    const uint32_t lds = (uint32_t)(uintptr_t)(LAP_LDS const char*)s_dst + (tid >> 6) * 1024;
    if (kKeep && last >= kBN - 1) {
#pragma unroll
      for (int i = 0; i < PER; ++i) copy(lds + i * NW * 1024, base, off[kKeep ? i : 0]);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) copy(lds + i * NW * 1024, base, offset(i, tid, last));
    }
  }
  static __device__ __forceinline__ void copy(uint32_t lds, const uint16_t* base, uint32_t o) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(o), "s"(base), "s"(__builtin_amdgcn_readfirstlane(lds))
                 : "memory", "m0");
  }
};

// The running state of a wave's 32 rows.
template <int DT, int D>
struct Rows {
  i16x8 qf[D / 16];   // Q^T operand
  f32x16 o[D / 32];   // o^T: rows d = 32 dc + (i & 3) + 8 (i >> 2) + 4 (lane / 32)
  float m, l;         // exponent of the weights (log2; equal in the lane pair), this lane's sum
};

// Where a wave has 512 registers (D = 256), products accumulate in the upper 256, which
// vector instructions do not reach.  o^T stays there: after the few places that do compute
// with it, it goes back, instead of all of it moving to and fro with every tile (a prompt
// of 16384 tokens with 16 heads 3006 -> 2416 us).
template <int DT, int D>
__device__ __forceinline__ void in_acc(Rows<DT, D>& w) {
  if constexpr (D == 256)
#pragma unroll
    for (int dc = 0; dc < D / 32; ++dc) asm volatile("" : "+a"(w.o[dc]));
}

// A row's maximum is raised only when a tile exceeds it by more than this, so weights
// go up to 2^8 before the division by their sum and the o^T registers are rescaled in
// few tiles (one prompt of 16384 tokens, 32 heads on 8, D = 128, 2026 us, with exact
// maxima 2102; 16 heads at D = 256 2423 and 3290).  The price: with an exact maximum the
// largest weight is 1 and not rounded, so the outputs' error against 64 bits (256 to 8192
// tokens, scores of deviation 1.5) is 1.15 to 1.19 times that of their own rounding, and
// 1.19 to 1.32 so.
constexpr float kSlack = 8.f;
// The exponent m that a row's weights are relative to lies this far below its maximum.  fp16
// has no relative steps below 2^-14 and nothing below 2^-25: with weights of up to 2^15 (and the
// slack in it) those of 2^-21 and more of the largest keep half a step, and what lies below
// 2^-32 of it is lost, where 65000 keys of 2^-25 each would still be 0.2 % of the row (same time:
// one prompt of 16384 tokens 2130 and 2142 us in fp16).  The sum and o^T carry the factor too.
template <int DT>
constexpr float kUp = DT == LAP_DTYPE_F16 ? 7.f : 0.f;

// LDS addresses of a lane's operands in the first buffer.  The others are a constant
// away, or, within a row, a constant XORed to the chunk's bits: rows of 128 bytes or
// more, aligned to their size, and a swizzle that is an XOR.
template <int D>
struct LaneAddr {
  uint32_t k, v[2];
  __device__ __forceinline__ void init(const char* s_k, const char* s_v, int lane) {
    constexpr int C = D / 8;
    const int col = lane & 31, hl = lane >> 5, g16 = (lane >> 4) & 1, i16 = lane & 15;
    k = (uint32_t)(uintptr_t)(LAP_LDS const char*)s_k + (col * C + (hl ^ swz<D>(col))) * 16;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      const int r = 8 * jj + 4 * hl + (i16 >> 2), chunk = 2 * g16 + ((i16 & 3) >> 1);
      v[jj] = (uint32_t)(uintptr_t)(LAP_LDS const char*)s_v +
              (r * C + (chunk ^ swz<D>(r))) * 16 + (i16 & 1) * 8;
    }
  }
};

// An address as one register, so that what is added to it later is an instruction's
// offset and not another register.
__device__ __forceinline__ uint32_t pinned(uint32_t at) {
  asm("" : "+v"(at));
  return at;
}

// The three parts of a tile's work.  Buffers are named by their byte offset from the
// first one.

// Scores of the keys of the K buffer at kb: their operands, and the products.
template <int D>
using KeyOps = i16x8[bn<D>() / 32][D / 16];
template <int D>
using Scores = f32x16[bn<D>() / 32];
template <int D>
using Weights = uint32_t[bn<D>() / 4];
template <int D>
__device__ __forceinline__ void load_keys(const LaneAddr<D>& la, uint32_t kb, KeyOps<D>& kf) {
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const uint32_t at = pinned((la.k + kb) ^ (ks << 5));
#pragma unroll
    for (int h = 0; h < bn<D>() / 32; ++h)
      kf[h][ks] = *(LAP_LDS const i16x8*)(uintptr_t)(at + h * 32 * D * 2);
  }
}
template <int DT, int D>
__device__ __forceinline__ void scores(const Rows<DT, D>& w, const KeyOps<D>& kf, Scores<D>& s) {
#pragma unroll
  for (int h = 0; h < bn<D>() / 32; ++h)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[h][i] = 0.f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
    for (int h = 0; h < bn<D>() / 32; ++h) s[h] = mfma32<DT>(kf[h][ks], w.qf[ks], s[h]);
}

// Scores -> weights pk (two to a register) and the rows' running state.  MASK: key
// kt + r counts for a row only below its `end`.
template <int DT, int D, bool MASK>
__device__ __forceinline__ void weights(Rows<DT, D>& w, Scores<D>& s, Weights<D>& pk, float c,
                                        int kt, int end, int lane) {
  constexpr int DC = D / 32;
  if constexpr (MASK) {
    const int left = end - kt - 4 * (lane >> 5);
#pragma unroll
    for (int h = 0; h < bn<D>() / 32; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[h][i] = h * 32 + (i & 3) + 8 * (i >> 2) < left ? s[h][i] : -INFINITY;
  }
  float mx = s[0][0];
#pragma unroll
  for (int h = 0; h < bn<D>() / 32; ++h)
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[h][i]);
  {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mx),
                                                    __builtin_bit_cast(uint32_t, mx), false, false);
    // (a bit cast of a vector's element itself reads the vector's first one)
    const uint32_t lower = r[0], upper = r[1];
    mx = fmaxf(__builtin_bit_cast(float, lower), __builtin_bit_cast(float, upper)) * c;
  }
  const float top = mx - kUp<DT>;
  if (__ballot(top > w.m + kSlack)) {  // also where m is -inf and a score is not
    const float m_new = top > w.m + kSlack ? top : w.m;
    const float alpha = m_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w.m - m_new);
    w.m = m_new;
    w.l *= alpha;
    in_acc<DT, D>(w);
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) w.o[dc] *= alpha;
    in_acc<DT, D>(w);
  }
  const float base = w.m == -INFINITY ? 0.f : w.m;
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int h = 0; h < bn<D>() / 32; ++h)
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i], c, -base));
      const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[h][i + 1], c, -base));
      sum[0] += p0;
      sum[1] += p1;
      pk[8 * h + i / 2] = pack2<DT>(p0, p1);
    }
  w.l += sum[0] + sum[1];
}

// o^T += V^T P^T of the rows of the V buffer at vb.
template <int DT, int D>
__device__ __forceinline__ void values(Rows<DT, D>& w, const LaneAddr<D>& la, uint32_t vb,
                                       const Weights<D>& pk) {
  uint32_t at[D / 32][2];
#pragma unroll
  for (int dc = 0; dc < D / 32; ++dc)
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) at[dc][jj] = pinned((la.v[jj] + vb) ^ (dc << 6));
#pragma unroll
  for (int ks = 0; ks < bn<D>() / 16; ++ks) {
    const uint4 pw = make_uint4(pk[4 * ks], pk[4 * ks + 1], pk[4 * ks + 2], pk[4 * ks + 3]);
#pragma unroll
    for (int dc = 0; dc < D / 32; ++dc) {
      i16x4 vt[2];
#pragma unroll
      for (int jj = 0; jj < 2; ++jj)
        vt[jj] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (LAP_LDS i16x4*)(uintptr_t)(at[dc][jj] + ks * 16 * D * 2));
      const i16x8 vf = {vt[0][0], vt[0][1], vt[0][2], vt[0][3],
                        vt[1][0], vt[1][1], vt[1][2], vt[1][3]};
      w.o[dc] = mfma32<DT>(vf, __builtin_bit_cast(i16x8, pw), w.o[dc]);
    }
  }
}

// The same of a tile that not every row of the wave sees in whole.  A value that is not
// finite in a row that some of these queries do not see must not reach them as 0 * inf:
// a tile that holds one is summed key by key instead.
template <int DT, int D>
__device__ __forceinline__ void values_masked(Rows<DT, D>& w, const LaneAddr<D>& la,
                                              const char* s_v, uint32_t vb,
                                              const Weights<D>& pk, int kt, int end, int hi,
                                              int lane) {
  constexpr int DC = D / 32, C = D / 8, kBN = bn<D>();
  const int col = lane & 31, hl = lane >> 5;
  u16x2 top = {0, 0};
#pragma unroll
  for (int i0 = 0; i0 < kBN * C / 64; i0 += 4) {  // four reads in flight
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = *reinterpret_cast<const uint4*>(s_v + vb + ((i0 + i) * 64 + lane) * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, u[e] & 0x7fff7fffu));
    }
  }
  constexpr unsigned short kInf = DT == LAP_DTYPE_F16 ? 0x7c00 : 0x7f80;
  if (!__ballot(top[0] >= kInf || top[1] >= kInf)) {
    values<DT, D>(w, la, vb, pk);
    return;
  }
  in_acc<DT, D>(w);
#pragma unroll 1
  for (int r = 0; r < kBN && kt + r < hi; ++r) {
    // the weight of key r: register 4 * (r / 8) + r % 4 of half r / 32, in the lane of
    // the pair with hl = r / 4 % 2
    const int want = (r >> 5) * 8 + ((r >> 3) & 3) * 2 + ((r & 3) >> 1);
    uint32_t u = 0;
#pragma unroll
    for (int i = 0; i < kBN / 4; ++i) u = i == want ? pk[i] : u;
    u = __shfl(u, col + 32 * ((r >> 2) & 1), 64);
    const float p = ld16<DT>((uint16_t)(r & 1 ? u >> 16 : u));
    const bool sees = kt + r < end;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int d = 32 * dc + (i & 3) + 8 * (i >> 2) + 4 * hl;
        const float x = ld16<DT>(*reinterpret_cast<const uint16_t*>(
            s_v + vb + (r * C + ((d >> 3) ^ swz<D>(r))) * 16 + (d & 7) * 2));
        w.o[dc][i] = sees ? __builtin_fmaf(p, x, w.o[dc][i]) : w.o[dc][i];
      }
  }
  in_acc<DT, D>(w);
}

template <int DT, int D, bool SHARED>
__device__ __forceinline__ void flash(const FlashArgs& a, const FlashTile& t,
                                      const char* s_k0, const char* s_v0) {
  constexpr int kBN = bn<D>(), KS = D / 16, DC = D / 32, TILE = kBN * D * 2;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int col = lane & 31, hl = lane >> 5;
  const int row = wave * 32 + col, j = row / a.G, head = row - j * a.G;
  const bool live = j < t.n;

  TileCopy<D> ck, cv;
  ck.init(a.k_st, tid);
  cv.init(a.v_st, tid);
  const auto fetch = [&](int kt, uint32_t buf) {
    ck.issue(s_k0 + buf, t.k + (int64_t)kt * a.k_st, t.hi - 1 - kt, tid);
    cv.issue(s_v0 + buf, t.v + (int64_t)kt * a.v_st, t.hi - 1 - kt, tid);
  };
  if (t.lo < t.hi) fetch(t.lo, 0);

  int lim, w_max, w_min;  // keys that this row, some row and every row of the wave sees
  if (SHARED && t.lens) {
    lim = live ? t.lens[j * kPlanInts + 1] : 0;
    w_max = lim;
    w_min = live ? lim : INT32_MAX;
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) {
      w_max = max(w_max, __shfl_xor(w_max, d, 64));
      w_min = min(w_min, __shfl_xor(w_min, d, 64));
    }
  } else {
    lim = live ? t.key0 + j + 1 : 0;
    const int j_lo = wave * 32 / a.G, j_hi = min((wave * 32 + 31) / a.G, t.n - 1);
    w_max = j_lo < t.n ? t.key0 + (SHARED ? 0 : j_hi) + 1 : 0;
    w_min = t.key0 + (SHARED ? 0 : j_lo) + 1;
    if (SHARED) lim = live ? t.key0 + 1 : 0;  // a step's tokens do not see each other
  }
  w_max = __builtin_amdgcn_readfirstlane(w_max);
  w_min = __builtin_amdgcn_readfirstlane(w_min);

  Rows<DT, D> w;
  LaneAddr<D> la;
  la.init(s_k0, s_v0, lane);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    w.qf[ks] = i16x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (live)
      w.qf[ks] =
          *reinterpret_cast<const i16x8*>(t.q + j * t.q_st + head * a.q_sh + ks * 16 + hl * 8);
  }
#pragma unroll
  for (int dc = 0; dc < DC; ++dc)
#pragma unroll
    for (int i = 0; i < 16; ++i) w.o[dc][i] = 0.f;
  in_acc<DT, D>(w);
  w.m = -INFINITY;
  w.l = 0.f;

  const int end = min(lim, t.hi);
  const int whole = w_max > 0 ? min(w_min, t.hi) : t.lo;  // keys below it are all seen
  // Two buffers: the copies of a tile are in flight while the one before it is worked on.
  Scores<D> s;
  Weights<D> pk;
  KeyOps<D> kf;
  uint32_t buf = 0;
  const auto begin = [&](int kt) {
    // this wave's copies have come and its reads are done; then everybody's
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    // The same once more, where the compiler sees it: it would otherwise take loads from
    // before the loop (the query, arguments) for pending in every round and wait for all
    // of memory, the copies of the next tile among it, at the first use of each (64
    // sequences behind 2000 shared tokens 53.3 -> 47.6 us).
    __builtin_amdgcn_s_waitcnt(0x0070);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (kt + kBN < t.hi) fetch(kt + kBN, buf ^ TILE);
  };
  int kt = t.lo;
  for (; kt + kBN <= whole; kt += kBN, buf ^= TILE) {
    begin(kt);
    load_keys<D>(la, buf, kf);
    // products before the other workgroup's weights: 2066 us against 2108 (a prompt of
    // 16384 tokens, 32 heads on 8, D = 128)
    __builtin_amdgcn_s_setprio(1);
    scores<DT, D>(w, kf, s);
    __builtin_amdgcn_s_setprio(0);
    weights<DT, D, false>(w, s, pk, a.c, kt, 0, lane);
    __builtin_amdgcn_s_setprio(1);
    values<DT, D>(w, la, buf, pk);
    __builtin_amdgcn_s_setprio(0);
  }
  for (; kt < t.hi; kt += kBN, buf ^= TILE) {  // every wave passes a barrier per tile
    begin(kt);
    if (kt >= w_max) continue;
    load_keys<D>(la, buf, kf);
    scores<DT, D>(w, kf, s);
    weights<DT, D, true>(w, s, pk, a.c, kt, end, lane);
    values_masked<DT, D>(w, la, s_v0, buf, pk, kt, end, t.hi, lane);
  }

  w.l += __shfl_xor(w.l, 32, 64);
  if (!live) return;
  if (t.parts == 1) {
    // weights that sum to zero (no key, or all scores -inf) give zeros
    const float inv = w.l == 0.f ? 0.f : 1.0f / w.l;
    uint16_t* op = t.out + j * t.o_st + head * a.o_sh;
#pragma unroll
    for (int dc = 0; dc < DC; ++dc)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint2 x;
        x.x = pack2<DT>(w.o[dc][4 * g] * inv, w.o[dc][4 * g + 1] * inv);
        x.y = pack2<DT>(w.o[dc][4 * g + 2] * inv, w.o[dc][4 * g + 3] * inv);
        *reinterpret_cast<uint2*>(op + 32 * dc + 8 * g + 4 * hl) = x;
      }
    return;
  }
  const int64_t at = (t.row0 + (int64_t)j * a.Hq + head) * a.nsplit + t.split;
  if (hl == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(w.m, w.l);
#pragma unroll
  for (int dc = 0; dc < DC; ++dc)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(a.part_o + at * D + 32 * dc + 8 * g + 4 * hl) = make_float4(
          w.o[dc][4 * g], w.o[dc][4 * g + 1], w.o[dc][4 * g + 2], w.o[dc][4 * g + 3]);
}

// Tile ti of a prompt call: its sequence, first token (of the sequence in the uniform
// form, of all in the packed one), tokens and cached keys; false: nothing to do.
struct PromptTile {
  int b, q0, n, key0;
};
__device__ __forceinline__ bool prompt_tile(const FlashArgs& a, int ti, PromptTile& p) {
  if (a.tiles) {
    const int4 w = a.tiles[ti];
    p = {w.z, w.x, min(min(w.y, a.bt), a.Tq - w.x), w.w};
    return p.n > 0 && p.q0 >= 0 && p.b >= 0 && p.b < a.B && p.key0 >= 0;
  }
  // B sequences of Tq tokens at the end of Tk keys, the last tokens first
  const int i = a.tps - 1 - ti / a.B;
  p = {ti % a.B, i * a.bt, min(a.bt, a.Tq - i * a.bt), a.Tk - a.Tq + i * a.bt};
  return true;
}
// The keys of a tile's last token, and the parts that they fill (all but the last of
// per_split keys); no key past the cache is read.
__device__ __forceinline__ int prompt_keys(const FlashArgs& a, const PromptTile& p) {
  return max(min(p.key0 + p.n, a.Tk), 0);
}
__device__ __forceinline__ int prompt_parts(const FlashArgs& a, int keys) {
  return min(max((keys - 1) / a.per_split + 1, 1), a.nsplit);
}
__device__ __forceinline__ int64_t prompt_row(const FlashArgs& a, const PromptTile& p) {
  return (a.tiles ? 0 : (int64_t)p.b * a.Tq) + p.q0;
}

// Workgroup -> (split, tile, KV head), the KV head fastest: consecutive workgroups go
// to different XCDs, so an XCD's L2 holds the keys of few heads.  Split by split: all
// first parts, which are whole, start before the last ones, which causal tiles leave short
// or empty (with a tile's splits side by side an even number of them put the same split on
// the same XCDs: one prompt of 16384 tokens, 4 heads on 1, D = 128, two splits 405 us, 312
// so).
template <int DT, int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
void prompt_kernel(FlashArgs a) {
  __shared__ __attribute__((aligned(256))) char s_k[2 * bn<D>() * D * 2],
      s_v[2 * bn<D>() * D * 2];
  const int hkv = blockIdx.x % a.Hkv;
  const int rest = blockIdx.x / a.Hkv;
  const int split = rest / a.n_tiles, tile = rest % a.n_tiles;
  PromptTile p;
  if (!prompt_tile(a, tile, p)) return;
  const int keys = prompt_keys(a, p);
  FlashTile t;
  t.parts = prompt_parts(a, keys);
  if (split >= t.parts) return;
  const int64_t qb = a.tiles ? 0 : p.b;
  t.n = p.n;
  t.key0 = p.key0;
  t.lens = nullptr;
  t.row0 = prompt_row(a, p) * a.Hq + hkv * a.G;
  t.q = a.q + qb * a.q_sb + (int64_t)p.q0 * a.q_st + (int64_t)hkv * a.G * a.q_sh;
  t.out = a.out + qb * a.o_sb + (int64_t)p.q0 * a.o_st + (int64_t)hkv * a.G * a.o_sh;
  t.q_st = a.q_st;
  t.o_st = a.o_st;
  t.k = a.k + (int64_t)p.b * a.k_sb + (int64_t)hkv * a.k_sh;
  t.v = a.v + (int64_t)p.b * a.v_sb + (int64_t)hkv * a.v_sh;
  t.split = split;
  t.lo = split * a.per_split;
  t.hi = split == t.parts - 1 ? keys : t.lo + a.per_split;
  flash<DT, D, false>(a, t, s_k, s_v);
}

// One query token per sequence over keys of which the first `prefix` are the same in
// every sequence.  Items: for the prefix, blocks of as many sequences as fill the
// workgroup's rows, by splits of the keys of sequence 0; behind it, each sequence by
// splits of its own keys.
template <int DT, int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
void shared_kernel(FlashArgs a) {
  __shared__ __attribute__((aligned(256))) char s_k[2 * bn<D>() * D * 2],
      s_v[2 * bn<D>() * D * 2];
  const int hkv = blockIdx.x % a.Hkv;
  const int it = blockIdx.x / a.Hkv, n_pre = a.psplit * a.pblocks;
  FlashTile t;
  t.parts = a.nsplit;
  int b, kb = 0;
  if (it < n_pre) {
    b = it / a.psplit * a.bt;
    t.split = it % a.psplit;
    t.n = min(a.bt, a.B - b);
    t.key0 = a.Tk - 1;
    t.lens = a.plans ? a.plans + (int64_t)b * kPlanInts : nullptr;
    t.lo = t.split * a.per_split;
    t.hi = min(a.prefix, t.lo + a.per_split);
  } else {
    const int ss = a.nsplit - a.psplit, i = (it - n_pre) % ss;
    b = kb = (it - n_pre) / ss;
    t.split = a.psplit + i;
    t.n = 1;
    const int len = a.plans ? min(a.plans[(int64_t)b * kPlanInts + 1], a.Tk) : a.Tk;
    t.key0 = len - 1;
    t.lens = nullptr;
    t.lo = (int)min((int64_t)a.prefix + (int64_t)i * a.per_split, (int64_t)a.Tk);
    t.hi = min(len, t.lo + a.per_split);
  }
  t.row0 = (int64_t)b * a.Hq + hkv * a.G;
  t.q = a.q + (int64_t)b * a.q_sb + (int64_t)hkv * a.G * a.q_sh;
  t.out = a.out + t.row0 * D;
  t.q_st = a.q_sb;
  t.o_st = (int64_t)a.Hq * D;
  t.k = a.k + (int64_t)kb * a.k_sb + (int64_t)hkv * a.k_sh;
  t.v = a.v + (int64_t)kb * a.v_sb + (int64_t)hkv * a.v_sh;
  flash<DT, D, true>(a, t, s_k, s_v);
}

// out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) of one row by WPR waves: a wave takes
// every WPR-th batch of kMergeAhead splits, and the first wave adds the waves up.  Four
// waves where there are more than kMergeFew splits (their batches come one after the
// other), one where there are few (a decode step of 8 sequences behind 30000 tokens, 8
// heads on 1: 33.2 us with one wave, 20.0 with four; a prompt of 300 tokens behind 36057, 7
// splits: 192.7 and 200.0); a wave of its own then has 16 bytes of each split to a lane
// and up to four rows (38912 rows of 6 splits, D = 128: 31.6 us with one row, 22.6 with
// two, 5.3 TB/s; 16384 of 4 splits 12.9 and 9.2).
constexpr int kMergeAhead = 8, kMergeFew = 16, kMergeThreads = 256;
// Lanes of a row: four values each where a wave has rows of its own.
template <int D, int WPR>
constexpr int merge_lanes() {
  return WPR == 1 ? D / 4 : 64;
}
template <int V>
struct Vals;
template <> struct Vals<1> { typedef float type; };
template <> struct Vals<2> { typedef float2 type; };
template <> struct Vals<4> { typedef float4 type; };

template <int DT, int D, int WPR>
__device__ __forceinline__ void merge_row(const FlashArgs& a, int64_t row, int parts, bool live,
                                          uint16_t* out) {
  constexpr int LPR = merge_lanes<D, WPR>(), V = D / LPR;
  typedef typename Vals<V>::type vals;
  const int lane = threadIdx.x % LPR, lane0 = (threadIdx.x & 63) - lane;
  const int part = (threadIdx.x >> 6) % WPR;
  float M = -INFINITY, l = 0.f, o[V] = {};
  if (live) {
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row * a.nsplit;
    const vals* po = reinterpret_cast<const vals*>(a.part_o + row * a.nsplit * D) + lane;
    // LPR splits at a time: the row's lane s holds split s's weight
    for (int s0 = 0; s0 < parts; s0 += LPR) {
      const int n = min(LPR, parts - s0);
      const float2 x = lane < n ? ml[s0 + lane] : make_float2(-INFINITY, 0.f);
      vals v[kMergeAhead];
      const auto request = [&](int s) {
#pragma unroll
        for (int i = 0; i < kMergeAhead; ++i) v[i] = po[(int64_t)(s0 + min(s + i, n - 1)) * LPR];
      };
      int s = part * kMergeAhead;
      if (s < n) request(s);
      float top = x.x;
#pragma unroll
      for (int d = LPR / 2; d >= 1; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
      top = fmaxf(top, M);
      const float base = top == -INFINITY ? 0.f : top;
      // a split without keys of this row: weight 0, and its values are 0
      const float w = x.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(x.x - base);
      const float before = __builtin_amdgcn_exp2f(M - base);
      float sum = x.y * w;
#pragma unroll
      for (int d = LPR / 2; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
      l = l * before + sum;
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] *= before;
      M = top;
      while (s < n) {
#pragma unroll
        for (int i = 0; i < kMergeAhead; ++i) {
          const float ws = s + i < n ? __shfl(w, lane0 + s + i, 64) : 0.f;
          const float* f = reinterpret_cast<const float*>(&v[i]);
#pragma unroll
          for (int e = 0; e < V; ++e) o[e] = ws == 0.f ? o[e] : __builtin_fmaf(f[e], ws, o[e]);
        }
        s += WPR * kMergeAhead;
        if (s < n) request(s);
      }
    }
  }
  if constexpr (WPR > 1) {  // every wave has the same maxima and sum
    __shared__ float s_o[WPR - 1][D];
    if (part > 0)
#pragma unroll
      for (int e = 0; e < V; ++e) s_o[part - 1][lane * V + e] = o[e];
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int p = 0; p < WPR - 1; ++p)
#pragma unroll
      for (int e = 0; e < V; ++e) o[e] += s_o[p][lane * V + e];
  }
  if (!live) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if constexpr (V == 4) {
    const uint2 x = make_uint2(pack2<DT>(o[0] * inv, o[1] * inv), pack2<DT>(o[2] * inv, o[3] * inv));
    *reinterpret_cast<uint2*>(out + lane * 4) = x;
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) out[lane * V + e] = st16<DT>(o[e] * inv);
  }
}

template <int D, int WPR>
__device__ __forceinline__ int merge_row_of() {
  constexpr int threads = merge_lanes<D, WPR>() * WPR;  // of a row
  return blockIdx.x * (kMergeThreads / threads) + threadIdx.x / threads;
}

// A row per (tile, token, head); only rows of a tile with more than one part are written.
template <int DT, int D, int WPR>
__global__ __launch_bounds__(kMergeThreads) void prompt_merge_kernel(FlashArgs a, int rows) {
  const int r = merge_row_of<D, WPR>();
  const int h = r % a.Hq, rest = r / a.Hq, j = rest % a.bt;
  PromptTile p{};
  int parts = 1;
  if (r < rows && prompt_tile(a, rest / a.bt, p) && j < p.n)
    parts = prompt_parts(a, prompt_keys(a, p));
  const bool live = parts > 1;
  uint16_t* out = a.out + (a.tiles ? 0 : p.b) * a.o_sb + (int64_t)(p.q0 + j) * a.o_st + h * a.o_sh;
  merge_row<DT, D, WPR>(a, (prompt_row(a, p) + j) * a.Hq + h, parts, live, out);
}

template <int DT, int D, int WPR>
__global__ __launch_bounds__(kMergeThreads) void shared_merge_kernel(FlashArgs a, int rows) {
  const int r = merge_row_of<D, WPR>();
  merge_row<DT, D, WPR>(a, r, a.nsplit, r < rows, a.out + (int64_t)r * D);
}

int merge_waves(int nsplit) { return nsplit > kMergeFew ? 4 : 1; }
int64_t merge_blocks(int64_t rows, int nsplit, int D) {
  const int per = merge_waves(nsplit) > 1 ? 1 : kMergeThreads / (D / 4);
  return (rows + per - 1) / per;
}

template <bool SHARED, int DT, int D, int WPR>
void launch_merge(const FlashArgs& a, int64_t rows, hipStream_t st) {
  const dim3 g((unsigned)merge_blocks(rows, a.nsplit, D)), threads(kMergeThreads);
  if constexpr (SHARED)
    hipLaunchKernelGGL((shared_merge_kernel<DT, D, WPR>), g, threads, 0, st, a, (int)rows);
  else hipLaunchKernelGGL((prompt_merge_kernel<DT, D, WPR>), g, threads, 0, st, a, (int)rows);
}

// The kernel and, with more than one split, the merge of `rows` rows.
template <bool SHARED, int DT, int D>
int launch_flash(const FlashArgs& a, int64_t grid, int64_t rows, hipStream_t st) {
  const dim3 g((unsigned)grid);
  if constexpr (SHARED) hipLaunchKernelGGL((shared_kernel<DT, D>), g, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((prompt_kernel<DT, D>), g, dim3(kThreads), 0, st, a);
  LAP_LAUNCH_CHECK("attention of many rows");
  if (a.nsplit > 1) {
    if (merge_waves(a.nsplit) == 4) launch_merge<SHARED, DT, D, 4>(a, rows, st);
    else launch_merge<SHARED, DT, D, 1>(a, rows, st);
    LAP_LAUNCH_CHECK("merge of splits");
  }
  return LAP_OK;
}

template <bool SHARED>
int launch_by_type(const FlashArgs& a, int dtype, int D, int64_t grid, int64_t rows,
                   hipStream_t st) {
#define LAP_BY_D(DT)                                                  \
  return D == 64    ? launch_flash<SHARED, DT, 64>(a, grid, rows, st)  \
         : D == 128 ? launch_flash<SHARED, DT, 128>(a, grid, rows, st) \
                    : launch_flash<SHARED, DT, 256>(a, grid, rows, st)
  if (dtype == LAP_DTYPE_F16) LAP_BY_D(LAP_DTYPE_F16);
  LAP_BY_D(LAP_DTYPE_BF16);
#undef LAP_BY_D
}

size_t part_bytes(int64_t rows, int nsplit, int D) {
  return nsplit > 1 ? (size_t)rows * nsplit * (D + 2) * sizeof(float) : 0;
}

int check_heads(const char* fn, int Hq, int Hkv, int D) {
  LAP_CHECK(Hq > 0 && Hkv > 0 && D > 0, "%s: bad sizes", fn);
  LAP_CHECK(Hq % Hkv == 0, "invalid GQA head counts: Hq=%d, Hkv=%d", Hq, Hkv);
  LAP_CHECK_CODE(Hq / Hkv <= kRows, LAP_ERR_UNSUPPORTED, "%s: group size %d unsupported (1 to %d)",
                 fn, Hq / Hkv, kRows);
  LAP_CHECK_CODE(D == 64 || D == 128 || D == 256, LAP_ERR_UNSUPPORTED,
                 "%s: head dim %d unsupported (64/128/256)", fn, D);
  return LAP_OK;
}

// Parts of the keys for `items` (tile, KV head) pairs with up to max_keys keys each, `fresh`
// of them new tokens'.  Estimated time in tiles of 64 keys of a workgroup that has its CU
// to itself (1.2 us at D = 128).  Two share a CU below D = 256: the second one slows both
// down, to 1.65 when all CUs are full, less while few are or parts end early.  A merge
// costs its launch and the partial sums.  Fitted to 53 shapes of 1 to 16 sequences, at most
// 1024 items and 256 to 65536 keys: 1.7 % behind the best count on average, where filling
// one round of workgroups with parts of at least 512 keys was 10 % (16384 tokens of 2 heads
// on 2, 3 parts 172 us, 1 301, 4 202; 1200 tokens behind 64336, 32 heads on 8, 6 parts 1278,
// 1 1651; 2048 tokens of 8 heads on 4, D = 256, 3 parts 48, 4 66, 1 80; 2048 tokens of 32
// heads on 8, 1 part 52, 2 66).  In all of them a batch's sequences had one cached length:
// every tile counts with max_keys, so one long cache among short ones gets too few parts
// (64 turns of 32 tokens, 32 heads on 8, one behind 131040 and 63 behind 200: 1 part, 2382
// us, where they take 142 and 21 in passes of their own).
int prompt_splits(int64_t items, double fresh, int max_keys, int D) {
  if (items == 0 || max_keys == 0) return 1;
  const int64_t slots = D == 256 ? 256 : 512;  // workgroups that run at a time
  const double seen = 1 - std::min(fresh, (double)max_keys) / (2.0 * max_keys);  // on average
  const double work = items * seen * max_keys / 64;
  double least = 0;
  int best = 1;
  for (int64_t n = 1; n == 1 || (n <= 32 && n * kGran <= max_keys && items * n <= 2048); ++n) {
    const int64_t per = ((max_keys + n - 1) / n + kGran - 1) / kGran,
                  ns = (max_keys + per * kGran - 1) / (per * kGran);
    const double parts = ns * seen + 1 - seen, live = items * parts;  // that hold keys
    const double fill = std::min(1.0, work / (live * per));
    double cost = per;
    if (live > slots)
      cost = D == 256 ? work / slots + per * fill : 1.65 * work / slots + per * fill * fill / 2;
    else if (live > 256)
      cost = per * (1.1 + (0.1 + 0.45 * (live - 256) / 256) * (2 * fill - 1));
    cost += 6 + (ns > 1 ? 4 + items * (2 + parts) / 80 : 0);
    if (n == 1 || cost < 0.98 * least) {
      least = cost;
      best = (int)ns;
    }
  }
  return best;
}

}  // namespace
}  // namespace lap

using namespace lap;

extern "C" int lap_prompt_shape(int total, int B, int tiles, int max_keys, int Hq, int Hkv,
                                int D, int* tokens_per_tile, int* n_tiles, int* nsplit) {
  clear_error();
  LAP_CHECK(tokens_per_tile && n_tiles && nsplit, "lap_prompt_shape: null output");
  LAP_CHECK(total >= 0 && B > 0 && max_keys >= 0, "lap_prompt_shape: bad sizes");
  int s = check_heads("lap_prompt_shape", Hq, Hkv, D);
  if (s != LAP_OK) return s;
  const int bt = kRows / (Hq / Hkv), bound = total / bt + std::min(B, total);
  const int64_t items = (int64_t)(tiles > 0 ? std::min(tiles, bound) : bound) * Hkv;
  *tokens_per_tile = bt;
  *n_tiles = bound;
  *nsplit = prompt_splits(items, (double)total / B, max_keys, D);
  return LAP_OK;
}

extern "C" int lap_prompt_attention_workspace_size(int64_t tokens, int Hq, int D, int nsplit,
                                                   size_t* bytes) {
  clear_error();
  LAP_CHECK(bytes, "lap_prompt_attention_workspace_size: null output");
  LAP_CHECK(tokens >= 0 && Hq > 0 && D > 0 && nsplit > 0, "bad sizes");
  *bytes = part_bytes(tokens * Hq, nsplit, D);
  return LAP_OK;
}

extern "C" int lap_prompt_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                    const void* keys, const void* vals, int64_t k_sb, int64_t k_sh,
                                    int64_t k_st, int64_t v_sb, int64_t v_sh, int64_t v_st,
                                    int dtype, int B, int Hq, int Hkv, int D, int Tq, int Tk,
                                    const int32_t* tiles, int n_tiles, int tokens_per_tile,
                                    int nsplit, int max_keys, float scale, void* out, int64_t o_sb,
                                    int64_t o_st, int64_t o_sh, void* workspace,
                                    size_t workspace_bytes, lap_stream_t stream) {
  clear_error();
  LAP_CHECK(q && keys && vals && out, "lap_prompt_attention: null pointer");
  LAP_CHECK(dtype == LAP_DTYPE_F16 || dtype == LAP_DTYPE_BF16,
            "lap_prompt_attention: dtype must be fp16/bf16");
  LAP_CHECK(B > 0 && Tq > 0 && Tk > 0 && Tk < (1 << 30), "lap_prompt_attention: bad sizes");
  int s = check_heads("lap_prompt_attention", Hq, Hkv, D);
  if (s != LAP_OK) return s;
  LAP_CHECK(tiles || Tq <= Tk, "lap_prompt_attention: %d queries exceed %d keys", Tq, Tk);
  LAP_CHECK(scale > 0.f && scale < INFINITY, "lap_prompt_attention: scale must be positive");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(keys) |
                         reinterpret_cast<uintptr_t>(vals) | reinterpret_cast<uintptr_t>(out) |
                         reinterpret_cast<uintptr_t>(tiles);
  LAP_CHECK(k_st >= 0 && v_st >= 0 && k_st <= kMaxRowStride && v_st <= kMaxRowStride,
            "lap_prompt_attention: K/V row strides above %d", kMaxRowStride);
  LAP_CHECK((ptrs & 15) == 0 && ((q_sb | q_st | q_sh | k_sb | k_sh | k_st | v_sb | v_sh | v_st |
                                  o_sb | o_st | o_sh) & 7) == 0,
            "lap_prompt_attention: rows must be 16-byte aligned");
  const int G = Hq / Hkv;
  LAP_CHECK(tokens_per_tile > 0 && (int64_t)tokens_per_tile * G <= kRows && nsplit > 0 &&
                n_tiles >= 0 && max_keys >= 0,
            "lap_prompt_attention: bad tile shape");
  const int tps = (Tq - 1) / tokens_per_tile + 1;
  const int64_t all_tiles = tiles ? n_tiles : (int64_t)B * tps;
  if (all_tiles == 0) return LAP_OK;
  FlashArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_sb; a.q_st = q_st; a.q_sh = q_sh;
  a.k = static_cast<const uint16_t*>(keys);
  a.v = static_cast<const uint16_t*>(vals);
  a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = G; a.Tq = Tq; a.Tk = Tk;
  a.tiles = reinterpret_cast<const int4*>(tiles);
  a.bt = tokens_per_tile;
  a.n_tiles = (int)all_tiles;
  a.tps = tps;
  a.nsplit = nsplit;
  a.per_split =
      (std::max(1, (int)(((int64_t)std::min(max_keys, Tk) + nsplit - 1) / nsplit)) + kGran - 1) /
      kGran * kGran;
  a.c = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.o_sb = o_sb; a.o_st = o_st; a.o_sh = o_sh;
  const int64_t rows = (int64_t)(tiles ? 1 : B) * Tq * Hq;
  const int64_t grid = all_tiles * nsplit * Hkv;
  LAP_CHECK(grid <= kMaxBlocks256, "lap_prompt_attention: too many rows");
  const int64_t tile_rows = all_tiles * tokens_per_tile * Hq;  // at most 128 * grid
  if (nsplit > 1) {
    LAP_CHECK(merge_blocks(tile_rows, nsplit, D) <= kMaxBlocks256,
              "lap_prompt_attention: too many rows");
    LAP_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "lap_prompt_attention: workspace must be 16-byte aligned");
    const size_t need = part_bytes(rows, nsplit, D);
    LAP_CHECK_CODE(workspace && workspace_bytes >= need, LAP_ERR_WORKSPACE,
                   "lap_prompt_attention: workspace of %zu bytes needed", need);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + rows * nsplit * D;
  }
  return launch_by_type<false>(a, dtype, D, grid, tile_rows, as_stream(stream));
}

namespace lap {
namespace {

// Rows per block, keys per split and splits of a decode step over a shared prefix.  512
// workgroups run at a time; a workgroup's start, its first copies and its part of the
// merge cost about as much as six tiles of 64 keys (64 sequences
// behind 2000 tokens with up to 2000 of their own: 54.1 us, 70.6 if counted as three).
// Every sequence counts as T keys long; where its length is on the device T is the caches'
// capacity, and room in them costs parts (16 sequences behind 16384 tokens with up to 883 of
// their own: 24.9 us at T = 17267, 40.8, 49.9 and 89.5 at two, four and eight times as many).
struct SharedShape {
  int bt, pblocks, per, psplit, nsplit;
};
SharedShape shared_shape(int B, int Hkv, int G, int T, int prefix) {
  SharedShape s{};
  s.bt = kRows / G;
  s.pblocks = (B + s.bt - 1) / s.bt;
  int64_t least = INT64_MAX;
  for (int64_t tiles = 2; tiles <= 4 || tiles * kGran < 2 * (int64_t)T; tiles += tiles / 4 + 1) {
    const int64_t per = tiles * kGran, p = (prefix + per - 1) / per,
                  n = p + (T - prefix + per - 1) / per;
    const int64_t items = (p * s.pblocks + (n - p) * B) * Hkv;
    const int64_t cost = (items + 511) / 512 * (tiles + 6);
    if (cost < least && n <= 1024) {
      least = cost;
      s.per = (int)std::min<int64_t>(per, 1 << 30);
      s.psplit = (int)p;
      s.nsplit = (int)n;
    }
  }
  return s;
}

int check_shared(int B, int Hq, int Hkv, int D, int T, int prefix) {
  LAP_CHECK(B > 0 && T > 0 && T < (1 << 30), "shared-prefix decode: bad sizes");
  int s = check_heads("shared-prefix decode", Hq, Hkv, D);
  if (s != LAP_OK) return s;
  LAP_CHECK(prefix >= 0 && prefix <= T, "shared-prefix decode: a prefix of %d of %d keys", prefix, T);
  return LAP_OK;
}

}  // namespace
}  // namespace lap

extern "C" int lap_shared_attn_decode_workspace_size(int B, int Hq, int Hkv, int D, int T,
                                                     int prefix, size_t* bytes) {
  clear_error();
  LAP_CHECK(bytes, "lap_shared_attn_decode_workspace_size: null output");
  int s = check_shared(B, Hq, Hkv, D, T, prefix);
  if (s != LAP_OK) return s;
  *bytes = part_bytes((int64_t)B * Hq, shared_shape(B, Hkv, Hq / Hkv, T, prefix).nsplit, D);
  return LAP_OK;
}

extern "C" int lap_shared_attn_decode(const void* q, int64_t q_sb, int64_t q_sh, const void* keys,
                                      const void* vals, int dtype, int B, int Hq, int Hkv, int T,
                                      int D, int64_t k_sb, int64_t k_sh, int64_t k_st,
                                      int64_t v_sb, int64_t v_sh, int64_t v_st, int prefix,
                                      const lap_row_plan* plans, float scale, void* out,
                                      void* workspace, size_t workspace_bytes,
                                      lap_stream_t stream) {
  clear_error();
  LAP_CHECK(q && keys && vals && out, "lap_shared_attn_decode: null pointer");
  LAP_CHECK(dtype == LAP_DTYPE_F16 || dtype == LAP_DTYPE_BF16,
            "lap_shared_attn_decode: dtype must be fp16/bf16");
  int s = check_shared(B, Hq, Hkv, D, T, prefix);
  if (s != LAP_OK) return s;
  LAP_CHECK(scale > 0.f && scale < INFINITY, "lap_shared_attn_decode: scale must be positive");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(keys) |
                         reinterpret_cast<uintptr_t>(vals) | reinterpret_cast<uintptr_t>(out);
  LAP_CHECK(k_st >= 0 && v_st >= 0 && k_st <= kMaxRowStride && v_st <= kMaxRowStride,
            "lap_shared_attn_decode: K/V row strides above %d", kMaxRowStride);
  LAP_CHECK((ptrs & 15) == 0 &&
                ((q_sb | q_sh | k_sb | k_sh | k_st | v_sb | v_sh | v_st) & 7) == 0,
            "lap_shared_attn_decode: rows must be 16-byte aligned");
  const SharedShape sh = shared_shape(B, Hkv, Hq / Hkv, T, prefix);
  FlashArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_sb = q_sb; a.q_sh = q_sh;
  a.k = static_cast<const uint16_t*>(keys);
  a.v = static_cast<const uint16_t*>(vals);
  a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.Tq = 1; a.Tk = T;
  a.bt = sh.bt;
  a.nsplit = sh.nsplit;
  a.per_split = sh.per;
  a.c = scale * kLog2e;
  a.out = static_cast<uint16_t*>(out);
  a.o_sh = D;
  a.prefix = prefix;
  a.psplit = sh.psplit;
  a.pblocks = sh.pblocks;
  a.plans = reinterpret_cast<const int32_t*>(plans);
  const int64_t rows = (int64_t)B * Hq;
  const int64_t grid =
      ((int64_t)sh.pblocks * sh.psplit + (int64_t)B * (sh.nsplit - sh.psplit)) * Hkv;
  LAP_CHECK(grid <= kMaxBlocks256 && merge_blocks(rows, sh.nsplit, D) <= kMaxBlocks256,
            "lap_shared_attn_decode: too many rows");
  if (sh.nsplit > 1) {
    LAP_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
              "lap_shared_attn_decode: workspace must be 16-byte aligned");
    const size_t need = part_bytes(rows, sh.nsplit, D);
    LAP_CHECK_CODE(workspace && workspace_bytes >= need, LAP_ERR_WORKSPACE,
                   "lap_shared_attn_decode: workspace of %zu bytes needed", need);
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + rows * sh.nsplit * D;
  }
  return launch_by_type<true>(a, dtype, D, grid, rows, as_stream(stream));
}
