// cache.hip — N1/N2: the decode step's writes into the device-resident cache.
//
// lap_rope_append applies the rotary embedding to the step's query and key
// (HF apply_rotary_pos_emb as aq_evaluation.py:296-305 calls it, the
// rotate_half convention) and writes the rotated key and the value of one
// token per sequence into the K/V capacity buffers at device positions
// (the cache write of _kv_cache_append, aq_evaluation.py:65-112), in one
// launch instead of about a dozen element-wise kernels per layer.
//
// Arithmetic matches torch's element-wise ops in the model dtype: each
// product and the sum are computed in fp32 and rounded to the dtype,
//     out = rnd(rnd(x * cos) + rnd(rotate_half(x) * sin)),
// rotate_half(x) = cat(-x[D/2:], x[:D/2]), so the rotated tensors are
// bit-identical to the reference's.
//
// lap_qk_rope_append does the same for any number of tokens, each with its own
// sequence and position (a prompt's packed tokens, or one token per sequence), and
// first norms the heads of q and k where the model has norms for them:
//     y = w * x * rsqrt(mean(x^2) + eps),  out = y * cos + rotate_half(y) * sin.
// With a norm everything is fp32 and rounded once at the end: the model code would
// round the normed value, each product and the sum, and every rounding is an error
// that the cache keeps.  Without one the roundings are lap_rope_append's, so a key is
// the same whether a prompt or a decode step wrote it.
#include "common.h"

namespace lap {
namespace {

template <int DT>
__device__ __forceinline__ float ld(const uint16_t* p, int64_t i) {
  return DT == LAP_DTYPE_F16 ? h2f(p[i]) : bf2f(p[i]);
}
template <int DT>
__device__ __forceinline__ uint16_t rnd(float f) {
  return DT == LAP_DTYPE_F16 ? f2h(f) : f2bf(f);
}
template <int DT>
__device__ __forceinline__ float rf(float f) {  // f rounded to the dtype, as fp32
  return DT == LAP_DTYPE_F16 ? h2f(f2h(f)) : bf2f(f2bf(f));
}

struct RopeArgs {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const uint16_t* k;
  int64_t k_sb, k_sh;
  const uint16_t* v;
  int64_t v_sb, v_sh;
  const uint16_t* cos;
  const uint16_t* sin;
  int64_t cs_sb;
  int Hq, Hkv, D;
  const int64_t* pos;
  uint16_t* ck;
  int64_t ck_sb, ck_sh, ck_st;
  uint16_t* cv;
  int64_t cv_sb, cv_sh, cv_st;
  int t_cap;
  uint16_t* q_out;
};

// Workgroup (b, r): r < Hq rotates query head r into q_out; r >= Hq rotates
// key head r - Hq into the cache and copies its value row.  Thread i owns
// the rotation pair (i, i + D/2).
template <int DT>
__global__ __launch_bounds__(128) void rope_append_kernel(RopeArgs a) {
  const int b = blockIdx.x / (a.Hq + a.Hkv), r = blockIdx.x % (a.Hq + a.Hkv);
  const int i = threadIdx.x, h2 = a.D / 2;
  if (i >= h2) return;
  const uint16_t* cs = a.cos + (int64_t)b * a.cs_sb;
  const uint16_t* sn = a.sin + (int64_t)b * a.cs_sb;
  const float c0 = ld<DT>(cs, i), c1 = ld<DT>(cs, i + h2);
  const float s0 = ld<DT>(sn, i), s1 = ld<DT>(sn, i + h2);
  const uint16_t* x;
  uint16_t* dst;
  if (r < a.Hq) {
    x = a.q + (int64_t)b * a.q_sb + (int64_t)r * a.q_sh;
    dst = a.q_out + ((int64_t)b * a.Hq + r) * a.D;
  } else {
    const int h = r - a.Hq;
    const int64_t t = a.pos[b];
    if (t < 0 || t >= a.t_cap) return;  // outside the capacity buffer: no write
    x = a.k + (int64_t)b * a.k_sb + (int64_t)h * a.k_sh;
    dst = a.ck + (int64_t)b * a.ck_sb + (int64_t)h * a.ck_sh + t * a.ck_st;
    const uint16_t* vs = a.v + (int64_t)b * a.v_sb + (int64_t)h * a.v_sh;
    uint16_t* vd = a.cv + (int64_t)b * a.cv_sb + (int64_t)h * a.cv_sh + t * a.cv_st;
    vd[i] = vs[i];
    vd[i + h2] = vs[i + h2];
  }
  const float x0 = ld<DT>(x, i), x1 = ld<DT>(x, i + h2);
  dst[i] = rnd<DT>(rf<DT>(x0 * c0) + rf<DT>(-x1 * s0));
  dst[i + h2] = rnd<DT>(rf<DT>(x1 * c1) + rf<DT>(x0 * s1));
}

struct QkRopeArgs {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* k;
  int64_t k_st, k_sh;
  const uint16_t* v;
  int64_t v_st, v_sh;
  const uint16_t* cos;
  const uint16_t* sin;
  int64_t cs_st;
  const uint16_t* q_w;  // norm weights [D], or null: no norm
  const uint16_t* k_w;
  float q_eps, k_eps;
  int64_t rows;  // tokens * (Hq + 2 Hkv)
  int Hq, Hkv, D, B;
  const int32_t* seq;  // or null: token i is sequence i
  const int64_t* pos;
  uint16_t* ck;
  int64_t ck_sb, ck_sh, ck_st;
  uint16_t* cv;
  int64_t cv_sb, cv_sh, cv_st;
  int t_cap;
  uint16_t* q_out;
};

union Vec8 {
  uint4 w;
  uint16_t e[8];
};

// LPR lanes per head row (the power of two from D / 16): a lane holds elements
// [8 c, 8 c + 8) of the row's first half and the same of its second, 16 bytes each,
// so the rotation's partners are in one lane and the norm's sum is log2(LPR)
// exchanges.
template <int DT, int LPR>
__global__ __launch_bounds__(256) void qk_rope_kernel(QkRopeArgs a) {
  const int R = a.Hq + 2 * a.Hkv;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  if (row >= a.rows) return;
  const int64_t tok = row / R;
  const int r = (int)(row - tok * R);
  const int64_t b = a.seq ? a.seq[tok] : tok;
  const int64_t pos = a.pos[tok];
  const int half = a.D / 2;
  const bool in = 8 * c < half;
  // behind the last sequence, or a key outside the capacity buffer: nothing written
  // (a whole row at a time, so the exchanges below stay among the lanes of a row)
  if (b < 0 || b >= a.B) return;
  if (r >= a.Hq && (pos < 0 || pos >= a.t_cap)) return;
  const uint16_t* x;
  uint16_t* dst;
  const uint16_t* w = nullptr;
  float eps = 0.f;
  if (r < a.Hq) {
    x = a.q + tok * a.q_st + r * a.q_sh;
    dst = a.q_out + (tok * a.Hq + r) * a.D;
    w = a.q_w;
    eps = a.q_eps;
  } else if (r < a.Hq + a.Hkv) {
    const int h = r - a.Hq;
    x = a.k + tok * a.k_st + h * a.k_sh;
    dst = a.ck + b * a.ck_sb + h * a.ck_sh + pos * a.ck_st;
    w = a.k_w;
    eps = a.k_eps;
  } else {
    const int h = r - a.Hq - a.Hkv;
    const uint16_t* vs = a.v + tok * a.v_st + h * a.v_sh;
    uint16_t* vd = a.cv + b * a.cv_sb + h * a.cv_sh + pos * a.cv_st;
    if (in) {
      const uint4 lo = *reinterpret_cast<const uint4*>(vs + 8 * c);
      const uint4 hi = *reinterpret_cast<const uint4*>(vs + half + 8 * c);
      *reinterpret_cast<uint4*>(vd + 8 * c) = lo;
      *reinterpret_cast<uint4*>(vd + half + 8 * c) = hi;
    }
    return;
  }
  auto at = [&](const uint16_t* p) { return *reinterpret_cast<const uint4*>(p + 8 * c); };
  Vec8 x0{}, x1{}, c0{}, c1{}, s0{}, s1{};
  if (in) {
    x0.w = at(x);
    x1.w = at(x + half);
    c0.w = at(a.cos + tok * a.cs_st);
    c1.w = at(a.cos + tok * a.cs_st + half);
    s0.w = at(a.sin + tok * a.cs_st);
    s1.w = at(a.sin + tok * a.cs_st + half);
  }
  Vec8 y0, y1;
  if (w) {
    Vec8 w0{}, w1{};
    if (in) {
      w0.w = at(w);
      w1.w = at(w + half);
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = ld<DT>(x0.e, e), v = ld<DT>(x1.e, e);
      sum = __builtin_fmaf(u, u, sum);
      sum = __builtin_fmaf(v, v, sum);
    }
#pragma unroll
    for (int d = LPR / 2; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
    const float inv = rsqrtf(sum / (float)a.D + eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = ld<DT>(x0.e, e) * inv * ld<DT>(w0.e, e);
      const float v = ld<DT>(x1.e, e) * inv * ld<DT>(w1.e, e);
      y0.e[e] = rnd<DT>(__builtin_fmaf(u, ld<DT>(c0.e, e), -v * ld<DT>(s0.e, e)));
      y1.e[e] = rnd<DT>(__builtin_fmaf(v, ld<DT>(c1.e, e), u * ld<DT>(s1.e, e)));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float u = ld<DT>(x0.e, e), v = ld<DT>(x1.e, e);
      y0.e[e] = rnd<DT>(rf<DT>(u * ld<DT>(c0.e, e)) + rf<DT>(-v * ld<DT>(s0.e, e)));
      y1.e[e] = rnd<DT>(rf<DT>(v * ld<DT>(c1.e, e)) + rf<DT>(u * ld<DT>(s1.e, e)));
    }
  }
  if (in) {
    *reinterpret_cast<uint4*>(dst + 8 * c) = y0.w;
    *reinterpret_cast<uint4*>(dst + half + 8 * c) = y1.w;
  }
}

}  // namespace
}  // namespace lap

using namespace lap;

extern "C" int lap_rope_append(const void* q, int64_t q_sb, int64_t q_sh, const void* k,
                               int64_t k_sb, int64_t k_sh, const void* v, int64_t v_sb,
                               int64_t v_sh, const void* cos, const void* sin, int64_t cs_sb,
                               int dtype, int B, int Hq, int Hkv, int D, const int64_t* pos,
                               void* cache_k, int64_t ck_sb, int64_t ck_sh, int64_t ck_st,
                               void* cache_v, int64_t cv_sb, int64_t cv_sh, int64_t cv_st,
                               int t_cap, void* q_out, lap_stream_t stream) {
  clear_error();
  LAP_CHECK(q && k && v && cos && sin && pos && cache_k && cache_v && q_out,
            "lap_rope_append: null pointer");
  LAP_CHECK(dtype == LAP_DTYPE_F16 || dtype == LAP_DTYPE_BF16,
            "lap_rope_append: dtype must be fp16/bf16");
  LAP_CHECK(B > 0 && Hq > 0 && Hkv > 0 && t_cap > 0, "lap_rope_append: bad sizes");
  LAP_CHECK(D > 0 && D % 2 == 0 && D <= 256, "lap_rope_append: D=%d must be even and <= 256", D);
  LAP_CHECK(q_sh >= D && k_sh >= D && v_sh >= D && cs_sb >= D && ck_st >= D && cv_st >= D,
            "lap_rope_append: strides smaller than D");
  RopeArgs a{static_cast<const uint16_t*>(q), q_sb, q_sh, static_cast<const uint16_t*>(k),
             k_sb, k_sh, static_cast<const uint16_t*>(v), v_sb, v_sh,
             static_cast<const uint16_t*>(cos), static_cast<const uint16_t*>(sin), cs_sb, Hq,
             Hkv, D, pos, static_cast<uint16_t*>(cache_k), ck_sb, ck_sh, ck_st,
             static_cast<uint16_t*>(cache_v), cv_sb, cv_sh, cv_st, t_cap,
             static_cast<uint16_t*>(q_out)};
  const dim3 grid((unsigned)(B * (Hq + Hkv)));
  hipStream_t st = as_stream(stream);
  if (dtype == LAP_DTYPE_F16)
    hipLaunchKernelGGL(rope_append_kernel<LAP_DTYPE_F16>, grid, dim3(128), 0, st, a);
  else
    hipLaunchKernelGGL(rope_append_kernel<LAP_DTYPE_BF16>, grid, dim3(128), 0, st, a);
  LAP_LAUNCH_CHECK("rope_append_kernel");
  return LAP_OK;
}

extern "C" int lap_qk_rope_append(const void* q, int64_t q_st, int64_t q_sh, const void* k,
                                  int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                                  int64_t v_sh, const void* cos, const void* sin, int64_t cs_st,
                                  const void* q_weight, float q_eps, const void* k_weight,
                                  float k_eps, int dtype, int64_t tokens, int B, int Hq, int Hkv,
                                  int D, const int32_t* seq, const int64_t* pos, void* cache_k,
                                  int64_t ck_sb, int64_t ck_sh, int64_t ck_st, void* cache_v,
                                  int64_t cv_sb, int64_t cv_sh, int64_t cv_st, int t_cap,
                                  void* q_out, lap_stream_t stream) {
  clear_error();
  LAP_CHECK(tokens >= 0 && B > 0 && Hq > 0 && Hkv > 0 && t_cap > 0,
            "lap_qk_rope_append: bad sizes");
  LAP_CHECK(seq || tokens <= B, "lap_qk_rope_append: more tokens than sequences");
  if (tokens == 0) return LAP_OK;
  LAP_CHECK(q && k && v && cos && sin && pos && cache_k && cache_v && q_out,
            "lap_qk_rope_append: null pointer");
  LAP_CHECK(dtype == LAP_DTYPE_F16 || dtype == LAP_DTYPE_BF16,
            "lap_qk_rope_append: dtype must be fp16/bf16");
  LAP_CHECK_CODE(D > 0 && D % 16 == 0 && D <= 256, LAP_ERR_UNSUPPORTED,
                 "lap_qk_rope_append: D=%d must be a multiple of 16 up to 256", D);
  LAP_CHECK(q_sh >= D && k_sh >= D && v_sh >= D && cs_st >= 0 && ck_st >= D && cv_st >= D,
            "lap_qk_rope_append: strides smaller than D");
  uintptr_t ptrs = 0;
  for (const void* p : {q, k, v, cos, sin, q_weight, k_weight, (const void*)cache_k,
                        (const void*)cache_v, (const void*)q_out})
    ptrs |= reinterpret_cast<uintptr_t>(p);
  int64_t strides = 0;
  for (int64_t x : {q_st, q_sh, k_st, k_sh, v_st, v_sh, cs_st, ck_sb, ck_sh, ck_st, cv_sb, cv_sh,
                    cv_st})
    strides |= x;
  LAP_CHECK((ptrs & 15) == 0 && (strides & 7) == 0,
            "lap_qk_rope_append: rows must be 16-byte aligned");
  QkRopeArgs a{static_cast<const uint16_t*>(q), q_st, q_sh, static_cast<const uint16_t*>(k), k_st,
               k_sh, static_cast<const uint16_t*>(v), v_st, v_sh,
               static_cast<const uint16_t*>(cos), static_cast<const uint16_t*>(sin), cs_st,
               static_cast<const uint16_t*>(q_weight), static_cast<const uint16_t*>(k_weight),
               q_eps, k_eps, tokens * (Hq + 2 * (int64_t)Hkv), Hq, Hkv, D, B, seq, pos,
               static_cast<uint16_t*>(cache_k), ck_sb, ck_sh, ck_st,
               static_cast<uint16_t*>(cache_v), cv_sb, cv_sh, cv_st, t_cap,
               static_cast<uint16_t*>(q_out)};
  const int lpr = D <= 16 ? 1 : D <= 32 ? 2 : D <= 64 ? 4 : D <= 128 ? 8 : 16;
  const int64_t blocks = (a.rows + 256 / lpr - 1) / (256 / lpr);
  LAP_CHECK(blocks <= kMaxBlocks256, "lap_qk_rope_append: too many rows");
  const dim3 grid((unsigned)blocks);
  hipStream_t st = as_stream(stream);
#define LAP_QK_ROPE(DT)                                                                      \
  do {                                                                                       \
    if (lpr == 1) hipLaunchKernelGGL((qk_rope_kernel<DT, 1>), grid, dim3(256), 0, st, a);      \
    else if (lpr == 2) hipLaunchKernelGGL((qk_rope_kernel<DT, 2>), grid, dim3(256), 0, st, a); \
    else if (lpr == 4) hipLaunchKernelGGL((qk_rope_kernel<DT, 4>), grid, dim3(256), 0, st, a); \
    else if (lpr == 8) hipLaunchKernelGGL((qk_rope_kernel<DT, 8>), grid, dim3(256), 0, st, a); \
    else hipLaunchKernelGGL((qk_rope_kernel<DT, 16>), grid, dim3(256), 0, st, a);             \
  } while (0)
  if (dtype == LAP_DTYPE_F16) LAP_QK_ROPE(LAP_DTYPE_F16);
  else LAP_QK_ROPE(LAP_DTYPE_BF16);
#undef LAP_QK_ROPE
  LAP_LAUNCH_CHECK("qk_rope_kernel");
  return LAP_OK;
}
