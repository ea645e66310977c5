// Kernels of the distribution operators around their tensor-core GEMMs: the row statistics
// (log-normaliser and entropy) with the given tokens' log-probabilities, the merge over
// vocabulary shards, the backward's row constants and target entries, and the selection of
// the most likely tokens with the top-k / top-p draw.
//
// Notation, per row: z = softcap(h . W_v), m = max z, S = sum e^(z-m), A = sum e^(z-m) (z-m),
//   lse = m + log S,   log p_v = z_v - lse,   entropy = -sum p log p = log S - A / S.
// A's terms are all <= 0 and log S >= 0, so the entropy has no cancellation.
#pragma once

#include "lp_ptx.cuh"

namespace lpk {

struct DistAcc {
  float m, s, a;  // base 2: max, sum 2^(z-m), sum 2^(z-m) (z-m)
};

__device__ __forceinline__ float dist_lse(const DistAcc& x) { return x.m * kLn2 + logf(x.s); }
__device__ __forceinline__ float dist_entropy(const DistAcc& x) { return logf(x.s) - kLn2 * (x.a / x.s); }

// A log-probability is never above 0; the roundings of z and lse can leave it there by an ulp
// (a NaN stays a NaN).
__device__ __forceinline__ float dist_logp(float z, float lse) {
  const float lp = z - lse;
  return lp > 0.f ? 0.f : lp;
}

__device__ __forceinline__ float dist_logp(double z, double lse) {
  const float lp = (float)(z - lse);
  return lp > 0.f ? 0.f : lp;
}

__device__ __forceinline__ float softcap_exact(float x, float cap) { return cap > 0.f ? cap * tanhf(x / cap) : x; }
__device__ __forceinline__ double softcap_f64(double x, float cap) {
  return cap > 0.f ? (double)cap * tanh(x / (double)cap) : x;
}

// Raw dot product h . w over one warp (every lane returns it): 16-byte loads, products of two
// bf16 numbers are exact in f32.
__device__ __forceinline__ float warp_dot(const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ w,
                                          long long d, int lane) {
  float acc0 = 0.f, acc1 = 0.f;
  const int n = (int)(d / 8);
#pragma unroll 4
  for (int i = lane; i < n; i += 32) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(h) + i);
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(w) + i);
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc0 = fmaf(__uint_as_float(av[j] << 16), __uint_as_float(bv[j] << 16), acc0);
      acc1 = fmaf(__uint_as_float(av[j] & 0xffff0000u), __uint_as_float(bv[j] & 0xffff0000u), acc1);
    }
  }
  float acc = acc0 + acc1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  return acc;
}

// Sum of f32 terms held as s + e, exact but for the rounding of e (about 2^-48 of the terms): each
// addition's rounding error is itself an f32 number, which e collects (Knuth's two-sum).
struct TwoSum {
  float s = 0.f, e = 0.f;
  __device__ __forceinline__ void add(float p) {
    const float t = s + p;
    const float b = t - s;
    e += (s - (t - b)) + (p - b);
    s = t;
  }
  __device__ __forceinline__ void add(const TwoSum& o) {
    add(o.s);
    e += o.e;
  }
};

// Two such sums side by side; a - b is an FMA with -1, rounded once as a subtraction is.
struct TwoSum2 {
  f32x2 s = 0, e = 0;
  __device__ __forceinline__ void add(f32x2 p, f32x2 minus_one) {
    const f32x2 t = add_f32x2(s, p);
    const f32x2 b = fma_f32x2(s, minus_one, t);
    const f32x2 c = fma_f32x2(b, minus_one, t);
    e = add_f32x2(e, add_f32x2(fma_f32x2(c, minus_one, s), fma_f32x2(b, minus_one, p)));
    s = t;
  }
};

// h . w over one warp (complete in lane 0), to about 2^-48 of sum |h w|: products of two bf16 numbers
// are exact in f32. f64 would convert every product, which took three times as long.
__device__ __forceinline__ double warp_dot_exact(const __nv_bfloat16* __restrict__ h,
                                                 const __nv_bfloat16* __restrict__ w, long long d, int lane) {
  TwoSum2 both;  // of the even and of the odd columns
  const f32x2 minus_one = pack_f32x2(-1.f, -1.f);
  const int n = (int)(d / 8);
#pragma unroll 1
  for (int i0 = 0; i0 < n; i0 += 128) {
    uint4 w4[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + 32 * u + lane;
      w4[u] = i < n ? __ldg(reinterpret_cast<const uint4*>(w) + i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i0 + 32 * u >= n) break;
      // a row of h is in L1; beyond its end w is 0
      const uint4 h4 = __ldg(reinterpret_cast<const uint4*>(h) + min(i0 + 32 * u + lane, n - 1));
      const uint32_t hv[4] = {h4.x, h4.y, h4.z, h4.w}, wv[4] = {w4[u].x, w4[u].y, w4[u].z, w4[u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        both.add(mul_f32x2(pack_f32x2(__uint_as_float(hv[j] << 16), __uint_as_float(hv[j] & 0xffff0000u)),
                           pack_f32x2(__uint_as_float(wv[j] << 16), __uint_as_float(wv[j] & 0xffff0000u))),
                 minus_one);
    }
  }
  TwoSum a, b;
  unpack_f32x2(both.s, a.s, b.s);
  unpack_f32x2(both.e, a.e, b.e);
  a.add(b);
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) {
    TwoSum x;
    x.s = __shfl_down_sync(0xffffffffu, a.s, o);
    x.e = __shfl_down_sync(0xffffffffu, a.e, o);
    a.add(x);
  }
  return (double)a.s + (double)a.e;
}

// The same; two-sums of infinities are NaN, for which the f32 sum stands in (an infinity, or NaN).
__device__ __forceinline__ double warp_score(const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ w,
                                             long long d, int lane) {
  double z = warp_dot_exact(h, w, d, lane);
  if (__any_sync(0xffffffffu, lane == 0 && z != z)) z = warp_dot(h, w, d, lane);
  return z;
}

// Merges the GEMM's partials of R consecutive rows per block and computes the given tokens'
// logits, one warp per (row, token) pair.
//   stats (optional, [3, T]): m, S, A of this shard in natural units, for dist_combine_kernel
//   zt [T, K]: softcapped logit of tokens owned by this shard, else 0
//   lse, entropy, logp (optional): valid where the shard is the whole vocabulary; a token
//   outside [0, Vs) has logp 0
constexpr int kDistThreads = 256;

template <int R>
__global__ void __launch_bounds__(kDistThreads, 4)
    dist_finalize_kernel(const float2* __restrict__ part, const float* __restrict__ part_a, int n_parts, int T,
                         const __nv_bfloat16* __restrict__ H, long long ldh, const __nv_bfloat16* __restrict__ W,
                         long long d, long long Vs, long long v_off, const int32_t* __restrict__ y, int K, float cap,
                         float* __restrict__ stats, float* __restrict__ zt, float* __restrict__ lse,
                         float* __restrict__ entropy, float* __restrict__ logp) {
  constexpr int kWarps = kDistThreads / 32;
  __shared__ float m_s[kWarps][R], s_s[kWarps][R], a_s[kWarps][R];
  __shared__ float lse_s[R];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.x * R;
  const int r = threadIdx.x % R;
  const int t = min(t0 + r, T - 1);
  const int rows = min(R, T - t0);
  // the row's maximum, then the sums at it: no chain of rescaled pairs, so the loads pass together
  float m = -INFINITY;
#pragma unroll 8
  for (int g = threadIdx.x / R; g < n_parts; g += kDistThreads / R) m = fmaxf(m, part[(size_t)g * T + t].x);
#pragma unroll
  for (int o = R; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane < R) m_s[warp][lane] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, m_s[w][r]);
  float s = 0.f, a = 0.f;
#pragma unroll 8
  for (int g = threadIdx.x / R; g < n_parts; g += kDistThreads / R) {
    const float2 p = part[(size_t)g * T + t];
    const float pa = part_a[(size_t)g * T + t];
    if (p.y != 0.f) {  // 0: a partial that saw padding only
      const float dm = p.x - m, e = exp2f(dm);
      s = fmaf(p.y, e, s);
      a = fmaf(fmaf(p.y, dm, pa), e, a);
    }
  }
#pragma unroll
  for (int o = R; o < 32; o <<= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  if (lane < R) {
    s_s[warp][lane] = s;
    a_s[warp][lane] = a;
  }
  __syncthreads();
  if (threadIdx.x < rows) {
    DistAcc acc{m, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      acc.s += s_s[w][r];
      acc.a += a_s[w][r];
    }
    const float l = dist_lse(acc);
    lse_s[r] = l;
    if (stats != nullptr) {
      stats[t] = acc.m * kLn2;
      stats[(size_t)T + t] = acc.s;
      stats[(size_t)2 * T + t] = acc.a * kLn2;
    }
    if (lse != nullptr) lse[t] = l;
    if (entropy != nullptr) entropy[t] = dist_entropy(acc);
  }
  __syncthreads();
  for (int i = warp; i < rows * K; i += kDistThreads / 32) {
    const int rr = i / K;
    const size_t at = (size_t)(t0 + rr) * K + i % K;
    const long long v = (long long)y[at] - v_off;
    const bool owned = v >= 0 && v < Vs;  // warp-uniform
    float z = 0.f;
    if (owned) z = softcap_exact(warp_dot(H + (size_t)(t0 + rr) * ldh, W + (size_t)v * d, d, lane), cap);
    if (lane == 0) {
      if (zt != nullptr) zt[at] = z;
      if (logp != nullptr) logp[at] = owned ? dist_logp(z, lse_s[rr]) : 0.f;
    }
  }
}

// Merges P shards: stats [P, 3, T] and owned target logits zt_in [P, T, K] (0 where another
// shard owns the token) into the global lse, entropy, logits and log-probabilities. V is the
// whole vocabulary: a token outside it has logp 0.
__global__ void dist_combine_kernel(const float* __restrict__ stats, const float* __restrict__ zt_in, int P, int T,
                                    int K, long long V, const int32_t* __restrict__ y, float* __restrict__ lse,
                                    float* __restrict__ entropy, float* __restrict__ zt, float* __restrict__ logp) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= T) return;
  float m = -INFINITY;
  for (int p = 0; p < P; ++p) m = fmaxf(m, stats[((size_t)p * 3 + 0) * T + t]);
  float s = 0.f, a = 0.f;
  for (int p = 0; p < P; ++p) {
    const float ps = stats[((size_t)p * 3 + 1) * T + t];
    const float dm = stats[((size_t)p * 3 + 0) * T + t] - m;
    const float e = expf(dm);
    s = fmaf(ps, e, s);
    a = fmaf(fmaf(ps, dm, stats[((size_t)p * 3 + 2) * T + t]), e, a);
  }
  const float l = m + logf(s);
  lse[t] = l;
  entropy[t] = logf(s) - a / s;
  for (int k = 0; k < K; ++k) {
    const size_t at = (size_t)t * K + k;
    float z = 0.f;
    for (int p = 0; p < P; ++p) z += zt_in[(size_t)p * T * K + at];
    const long long v = y[at];
    zt[at] = z;
    logp[at] = v >= 0 && v < V ? dist_logp(z, l) : 0.f;
  }
}

// Row constants of the backward. With G = sum_k g_k over the row's tokens, e the gradient of the
// entropy E, and log p = ln2 * log2 p:
//   G + e (log p + E) = a + b log2 p,   a = G + e E,   b = e ln2
// row_const = [3, T]: a, b, lse in base 2. g ([T, K]) or ge ([T]) may be null (no gradient).
__global__ void dist_row_const_kernel(const float* __restrict__ lse, const float* __restrict__ entropy,
                                      const int32_t* __restrict__ y, const float* __restrict__ g,
                                      const float* __restrict__ ge, int T, int K, long long V,
                                      float* __restrict__ row_const) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= T) return;
  float sum = 0.f;
  if (g != nullptr) {
    for (int k = 0; k < K; ++k) {
      const long long v = y[(size_t)t * K + k];
      if (v >= 0 && v < V) sum += g[(size_t)t * K + k];
    }
  }
  // a zero gradient of the entropy takes no part, whatever the entropy is
  const float e = ge != nullptr ? ge[t] : 0.f;
  row_const[t] = e != 0.f ? fmaf(e, entropy[t], sum) : sum;
  row_const[(size_t)T + t] = e * kLn2;
  row_const[(size_t)2 * T + t] = lse[t] * kLog2e;
}

// mask[t] = whether row t sends any gradient: one of its g [T, K] or its ge [T] is not zero (either
// may be null).
__global__ void dist_row_mask_kernel(const float* __restrict__ g, const float* __restrict__ ge, int T, int K,
                                     uint8_t* __restrict__ mask) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= T) return;
  bool sent = ge != nullptr && ge[t] != 0.f;
  if (g != nullptr)
    for (int k = 0; k < K; ++k) sent |= g[(size_t)t * K + k] != 0.f;
  mask[t] = sent ? 1 : 0;
}

// Everything the backward reads of the rows that do, one warp per row: the hidden state, the tokens
// with their logits and gradients, and the row's scalars.
struct DistRows {
  const __nv_bfloat16* H;
  long long ldh;
  const int32_t* y;
  const float *zt, *lse, *entropy, *g, *ge;
};
struct DistRowsOut {
  __nv_bfloat16* H;
  int32_t* y;
  float *zt, *lse, *entropy, *g, *ge;
};
__global__ void dist_gather_kernel(const int32_t* __restrict__ idx, const int* __restrict__ count, const DistRows from,
                                   const DistRowsOut to, long long d, int K) {
  const int lane = threadIdx.x & 31;
  const int n = *count;
  const int stride = (int)((gridDim.x * blockDim.x) >> 5);
  for (int i = (int)((blockIdx.x * blockDim.x + threadIdx.x) >> 5); i < n; i += stride) {
    const int t = idx[i];
    const uint4* src = reinterpret_cast<const uint4*>(from.H + (size_t)t * from.ldh);
    uint4* dst = reinterpret_cast<uint4*>(to.H + (size_t)i * d);
    for (int v = lane; v < (int)(d / 8); v += 32) dst[v] = src[v];
    for (int k = lane; k < K; k += 32) {
      const size_t a = (size_t)t * K + k, b = (size_t)i * K + k;
      to.y[b] = from.y[a];
      to.zt[b] = from.zt[a];
      if (from.g != nullptr) to.g[b] = from.g[a];
    }
    if (lane == 0) {
      to.lse[i] = from.lse[t];
      to.entropy[i] = from.entropy[t];
      if (from.ge != nullptr) to.ge[i] = from.ge[t];
    }
  }
}

// dZ of a chunk from kept logits (EPI_DIST_KEEP) instead of a recomputed product: reads 2 bytes and
// writes 2 per entry, where the recompute costs 2 d flops. The same formula as EPI_DIST_DZ's; with one
// token per row its entry is in it, too, from its f32 logit: where p is near 1, g - p G keeps nothing of
// a logit in 16 bits. A block takes a run of one row's columns, eight (16 bytes) per
// thread and step, the next step's load ahead of the arithmetic. Bound by HBM: 4 T Vs bytes. It takes
// many warps to keep HBM busy: 3686 rows of 262144 in 727 us (5.3 TB/s; a copy of the same bytes takes
// 575) with 2048 threads an SM, 911 with 1024 threads and four steps in flight each.
struct DistDzParams {
  const uint16_t* kept;   // [rows, ldk]
  const float* kept_max;  // [rows, ld_max]
  const int32_t* row_of;  // [T] row of the kept logits, or null: the row itself
  long long ldk, ld_max;
  const float* row_const;  // [3][row_ld], or null: one token per row and the pointers below
  long long row_ld;
  const int32_t* y;
  const float *zt, *g, *ge, *lse, *entropy;
  long long vocab, v_off, Vs;
  float cap;
  __nv_bfloat16* dz;
  long long ldz;
  int steps;  // per block
};
constexpr int kDzStep = 2048;  // columns of a block's step

// Eight entries of columns of which one is far (keep_far). By y, with e = 2^y and r = 1 / (1 + e):
// z = c (1 - 2 r) and softcap' = 4 e r^2, near 0 too.
__device__ __forceinline__ uint4 dist_dz_far(uint4 kept, float slot, float cap, float a, float b, float l2) {
  const uint32_t w[4] = {kept.x, kept.y, kept.z, kept.w};
  const float c2 = cap * kLog2e;
  const float top = kept_far_top(slot, c2), step = keep_range(c2) / 32767.f;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t n = (j & 1) ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
    float lp, slope;
    if (n & 0x8000u) {
      const float y = fmaf((float)(n & 0x3fffu), kKeepFarUnit, kKeepFarFrom);
      const float e = fast_ex2(n & 0x4000u ? -y : y);
      const float r = fast_rcp(1.f + e);
      lp = fmaf(-2.f * c2, r, c2 - l2);
      slope = 4.f * e * r * r;
    } else {
      const float z = fmaf((float)n, -step, top);
      const float u = z / c2;
      lp = z - l2;
      slope = fmaf(-u, u, 1.f);
    }
    v[j] = -slope * (fast_ex2(lp) * fmaf(b, lp, a));
  }
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

// The entry of a token whose slots' gradients sum to `sum`, from its f32 logit:
// softcap'(z) * (sum - p * (a + b log2 p)), softcap'(z) = 1 - (z / c)^2.
__device__ __forceinline__ float dist_dz_given(float z, float cap, float a, float b, float l2, float sum) {
  const float lp = fmaf(z, kLog2e, -l2);
  const float u = cap > 0.f ? z / cap : 0.f;
  return fmaf(-u, u, 1.f) * (sum - exp2f(lp) * fmaf(b, lp, a));
}

__global__ void __launch_bounds__(256, 8) dist_dz_kernel(const DistDzParams P) {
  const int t = blockIdx.y;
  float a, b, l2, gv = 0.f;
  long long yl = -1;
  if (P.row_const != nullptr) {
    a = P.row_const[t];
    b = P.row_const[P.row_ld + t];
    l2 = P.row_const[2 * P.row_ld + t];
  } else {
    const long long v = P.y[t];
    if (P.g != nullptr && v >= 0 && v < P.vocab) {
      gv = P.g[t];
      yl = v - P.v_off;
    }
    const float e = P.ge != nullptr ? P.ge[t] : 0.f;
    a = e != 0.f ? fmaf(e, P.entropy[t], gv) : gv;
    b = e * kLn2;
    l2 = P.lse[t] * kLog2e;
  }
  const long long from = P.row_of != nullptr ? P.row_of[t] : t;
  const uint16_t* kept = P.kept + from * P.ldk;
  const float* kept_max = P.kept_max + from * P.ld_max;
  __nv_bfloat16* dz = P.dz + (size_t)t * P.ldz;
  const float ucap = P.cap > 0.f ? kLn2 / P.cap : 0.f;  // z2 -> tanh(x / c), without softcap 0
  const int c0 = (int)blockIdx.x * P.steps * kDzStep + (int)threadIdx.x * 8;
  const int end = min((int)P.Vs, (int)(blockIdx.x + 1) * P.steps * kDzStep);
  uint4 q = make_uint4(0, 0, 0, 0);
  float mx = 0.f;
  if (c0 < end) {
    q = __ldcs(reinterpret_cast<const uint4*>(kept + c0));
    mx = __ldg(kept_max + c0 / 32);
  }
  const float step = keep_range(P.cap * kLog2e) / 65535.f;
  auto two = [](float x) { return pack_f32x2(x, x); };
  const f32x2 a2 = two(a), b2 = two(b), ml2 = two(-l2), ucap2 = two(ucap), mstep2 = two(-step), m23 = two(-8388608.f),
              mone = two(-1.f);
  bool far = false;
#pragma unroll 1
  for (int col = c0; col < end; col += kDzStep) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    const float m = mx;
    if (col + kDzStep < end) {
      q = __ldcs(reinterpret_cast<const uint4*>(kept + col + kDzStep));
      mx = __ldg(kept_max + (col + kDzStep) / 32);
    }
    far |= kept_far(m);
    const f32x2 top = two(m);
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // 2^23 + n, whose low bits are n, less 2^23
      const f32x2 n = add_f32x2(pack_f32x2(__uint_as_float(__byte_perm(w[j], 0x4b000000u, 0x7610)),
                                           __uint_as_float(__byte_perm(w[j], 0x4b000000u, 0x7632))),
                                m23);
      const f32x2 z = fma_f32x2(n, mstep2, top);
      const f32x2 lp = add_f32x2(z, ml2);
      const f32x2 u = mul_f32x2(z, ucap2);
      float l0, l1, v0, v1;
      unpack_f32x2(lp, l0, l1);
      // p (a + b log2 p) (u^2 - 1)
      const f32x2 v = mul_f32x2(mul_f32x2(pack_f32x2(fast_ex2(l0), fast_ex2(l1)), fma_f32x2(b2, lp, a2)),
                                fma_f32x2(u, u, mone));
      unpack_f32x2(v, v0, v1);
      out[j] = pack_bf16x2(v0, v1);
    }
    // rows of dZ are padded to 16 bytes
    *reinterpret_cast<uint4*>(dz + col) = make_uint4(out[0], out[1], out[2], out[3]);
  }
  // Rare: this thread's far columns, once more. Here, not above, where they would take registers that
  // the loop's loads in flight need (809 instead of 727 us).
  if (far) {
#pragma unroll 1
    for (int col = c0; col < end; col += kDzStep) {
      const float m = kept_max[col / 32];
      if (kept_far(m))
        *reinterpret_cast<uint4*>(dz + col) =
            dist_dz_far(*reinterpret_cast<const uint4*>(kept + col), m, P.cap, a, b, l2);
    }
  }
  // the row's token, where this thread has written its entry
  if (yl >= c0 && yl < end && (yl - c0) % kDzStep < 8) 
    dz[yl] = __float2bfloat16_rn(dist_dz_given(P.zt[t], P.cap, a, b, l2, gv));
}

// The given tokens' entries of a chunk's dZ, `sum` over the row's slots that hold the token. The first slot of a token writes the entry, so a token that a row
// names twice is written once, with both gradients.
__global__ void dist_dz_targets_kernel(const int32_t* __restrict__ y, const float* __restrict__ zt,
                                       const float* __restrict__ g, const float* __restrict__ row_const,
                                       long long row_ld, int T, int K, long long v_off, long long Vs, float cap,
                                       __nv_bfloat16* __restrict__ dz, long long ldz) {
  const long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  if (i >= (long long)T * K) return;
  const int t = (int)(i / K), k = (int)(i % K);
  const int32_t* yt = y + (size_t)t * K;
  const int32_t id = yt[k];
  const long long v = (long long)id - v_off;
  if (v < 0 || v >= Vs) return;
  for (int j = 0; j < k; ++j)
    if (yt[j] == id) return;
  float sum = 0.f;
  if (g != nullptr)
    for (int j = k; j < K; ++j)
      if (yt[j] == id) sum += g[(size_t)t * K + j];
  dz[(size_t)t * ldz + v] = __float2bfloat16_rn(
      dist_dz_given(zt[i], cap, row_const[t], row_const[row_ld + t], row_const[2 * row_ld + t], sum));
}

// The given tokens' entries are most of a row's gradient, and what rounding them to bf16 leaves (of each up
// to 2^-8) is most of the gradients' error where few rows enter a sum. So they do not keep that rounding:
// dH takes the rest beside the product, and the rows of dW that few rows make are summed again in f32.
// (Error of the gradients against 64 bits, over that of rounding the exact ones to bf16, of 150 random calls,
// most of fewer than a hundred rows: up to 2.1 with the entries as they are in dZ, at most 1.3 without their
// rounding.)
struct DistEntries {
  const int32_t* y;  // [T, K]
  int K;
  const float *zt, *g;     // [T, K] (g or null)
  const float* row_const;  // [3][row_ld], or null: one token per row and the pointers below
  long long row_ld;
  const float *ge, *lse, *entropy;
  long long v_off, Vs;
  float cap;
  const __nv_bfloat16* dz;
  long long ldz;
};

// Row t's entry in f32 if `id` is one of its tokens, else as it is in dZ; id is one of this shard's.
__device__ __forceinline__ float dist_entry(const DistEntries& P, int t, int32_t id, bool& given) {
  const int32_t* y = P.y + (size_t)t * P.K;
  float sum = 0.f, z = 0.f;
  given = false;
  for (int k = 0; k < P.K; ++k) {
    if (y[k] != id) continue;
    given = true;
    z = P.zt[(size_t)t * P.K + k];
    if (P.g != nullptr) sum += P.g[(size_t)t * P.K + k];
  }
  if (!given) return __bfloat162float(P.dz[(size_t)t * P.ldz + (id - P.v_off)]);
  float a, b, l2;
  if (P.row_const != nullptr) {
    a = P.row_const[t];
    b = P.row_const[P.row_ld + t];
    l2 = P.row_const[2 * P.row_ld + t];
  } else {
    const float e = P.ge != nullptr ? P.ge[t] : 0.f;
    a = e != 0.f ? fmaf(e, P.entropy[t], sum) : sum;
    b = e * kLn2;
    l2 = P.lse[t] * kLog2e;
  }
  return dist_dz_given(z, P.cap, a, b, l2, sum);
}

// Adds f times four bf16 numbers.
__device__ __forceinline__ void add_scaled(float4& acc, float f, const __nv_bfloat16* __restrict__ x) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(x));
  acc.x = fmaf(f, __uint_as_float(v.x << 16), acc.x);
  acc.y = fmaf(f, __uint_as_float(v.x & 0xffff0000u), acc.y);
  acc.z = fmaf(f, __uint_as_float(v.y << 16), acc.z);
  acc.w = fmaf(f, __uint_as_float(v.y & 0xffff0000u), acc.w);
}
__device__ __forceinline__ void store_row4(void* out, long long at, bool bf16, const float4& v) {
  if (bf16)
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(out) + at) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  else
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at) = v;
}

// dH of row t: the product's f32 partials part [S][mpad][d] and, for each of the row's tokens once, what
// rounding left of its entry times its row of W. One block per row; K at most the block's threads. Bound by
// HBM and L2 (4096 rows x 2048, two partials, one token each: 66 us, the sum of the partials alone 48).
constexpr int kDistRowThreads = 256;
__global__ void __launch_bounds__(kDistRowThreads)
    dist_dh_finish_kernel(const float* __restrict__ part, int S, long long mpad, const DistEntries P,
                          const __nv_bfloat16* __restrict__ W, long long d, void* __restrict__ out, long long ld_out,
                          bool out_bf16) {
  __shared__ float left_s[kDistRowThreads];
  __shared__ int row_s[kDistRowThreads];
  const int t = blockIdx.x, tid = threadIdx.x;
  if (tid < P.K) {
    const int32_t* y = P.y + (size_t)t * P.K;
    const long long v = (long long)y[tid] - P.v_off;
    float left = 0.f;
    if (v >= 0 && v < P.Vs) {
      bool first = true, given;
      for (int j = 0; j < tid; ++j) first &= y[j] != y[tid];
      if (first) left = dist_entry(P, t, y[tid], given) - __bfloat162float(P.dz[(size_t)t * P.ldz + v]);
    }
    left_s[tid] = left;
    row_s[tid] = left != 0.f ? (int)v : -1;
  }
  __syncthreads();
  for (long long c = tid * 4; c < d; c += kDistRowThreads * 4) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = 0; s < S; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(part + ((size_t)s * mpad + t) * d + c);
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
    }
#pragma unroll 4
    for (int k = 0; k < P.K; ++k)
      if (row_s[k] >= 0) add_scaled(acc, left_s[k], W + (size_t)row_s[k] * d + c);
    store_row4(out, t * ld_out + c, out_bf16, acc);
  }
}

// The given tokens' rows of dW over T rows, T at most the block's threads: dW[v] = sum over t of dZ[t, v] h[t],
// its given entries in f32. One block per (row, slot); the first that names a token has it. It reads T rows of
// H, so it is taken for T T K <= kDistDwRows (268 MB from L2 at d = 2048, some 30 us): with more rows the
// roundings of their entries average out.
constexpr int kDistDwRows = 65536;
__global__ void __launch_bounds__(kDistRowThreads)
    dist_dw_rows_kernel(const DistEntries P, int T, const __nv_bfloat16* __restrict__ H, long long ldh, long long d,
                        void* __restrict__ dW, bool out_bf16) {
  __shared__ float entry_s[kDistRowThreads];
  const int i = blockIdx.x, tid = threadIdx.x;
  const int32_t id = P.y[i];
  const long long v = (long long)id - P.v_off;
  if (v < 0 || v >= P.Vs) return;  // the whole block
  bool earlier = false;
  for (int j = tid; j < i; j += kDistRowThreads) earlier |= P.y[j] == id;
  if (tid < T) {
    bool given;
    entry_s[tid] = dist_entry(P, tid, id, given);
  }
  if (__syncthreads_or(earlier)) return;
  for (long long c = tid * 4; c < d; c += kDistRowThreads * 4) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int t = 0; t < T; ++t) add_scaled(acc, entry_s[t], H + (size_t)t * ldh + c);
    store_row4(dW, v * d + c, out_bf16, acc);
  }
}

// ----------------------------------------------------------------------------- selection
// The k most likely tokens of a row, in the order of the exact dot products h . W_v (softcap is
// monotone), the lowest id first among equals. The GEMM only nominates: a key is one accumulator
// (f32) or the largest of G neighbours with the second largest beside it. The largest keys, a few more
// than k, are selected. The k-th largest of the values seen there (keys and second largest) is a lower
// bound of the k-th logit: a key below it, beyond what either may be off by, is dropped, and a group
// whose second largest reaches it has all its columns scored. Candidates are scored again to 2^-48 and
// ranked by that. Where a key that was not selected could still hold one of the k (it reaches the exact
// k-th score, but for what it may be off by), all such keys follow, as many at a time as there are slots:
// equal or nearly equal tokens by the thousand, which a row in earnest does not have.
//
// What an accumulator may be off by (top_accumulator_error): one step of the tensor core adds 16
// products, aligned to the largest of them and the sum so far, without what lies below 2^-25 of that,
// and drops the new sum's bits below 2^-23. (Sums of one large and many small terms lose just this.)
// All of these are at most sum |h w|, which is at most |h| |w|: a step is off by (17/4 + 1) 2^-23 of
// the product of the lengths. The longest row of the embedding stands for all.
// A group's values lose log2(G) low bits on top, G 2^-23 of themselves.
//
// Finding the keys: each thread keeps the largest of the keys it loads; the n-th largest of those
// kTopThreads maxima is a lower bound of the n-th largest key, and few more than n keys reach it
// (about n^2 / (2 kTopThreads), the keys that share a thread). Only when more than kTopSel do, a
// bisection over all keys follows.
constexpr int kTopMax = 128;
constexpr int kTopSpare = 8;  // keys selected beyond k, with k / 16 more: they lie the closer, the larger k
constexpr int kTopThreads = 512;
constexpr int kTopSel = kTopMax + 8 * kTopSpare;  // most selected keys
constexpr int kTopBatch = 384;                    // candidates scored and ranked at a time,
constexpr int kTopCand = kTopBatch + kTopMax;     // beside the best of those before them
constexpr int kTopKeyBytes = 184 * 1024;  // most key bytes kept in shared memory, beside the static part

// Order-preserving map of f32 to u32; NaN comes last.
__device__ __forceinline__ uint32_t ordered_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// Its inverse (0, a NaN's key, becomes -inf).
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k <= 0x007fffffu) return -INFINITY;
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// A group's value without its column bits.
template <int G>
__device__ __forceinline__ float group_value(float x) {
  return __uint_as_float(__float_as_uint(x) & ~(uint32_t)(G - 1));
}

// Bound on an accumulator's error, from the squared lengths of the two rows. The sums of 64 squares in
// bf16 that w2 is made of can be an eighth too small (32 steps of 2^-8), h2 and the rest by far less, so the
// product of the lengths by a fifteenth: 1.08 makes up for it, as sqrt(d) 2^-62 does for squares below
// the range of the two types.
__device__ __forceinline__ float top_accumulator_error(float h2, float w2, long long d) {
  const float least = sqrtf((float)d) * 2.168404344971009e-19f;
  return 1.08f * 5.25f * 1.1920928955078125e-07f * (float)(d / 16 + 2) * (sqrtf(h2) + least) * (sqrtf(w2) + least);
}

struct TopParams {
  const float2* part;
  const float* part_a;
  int n_parts;
  const float* length2;  // [n_lengths] the largest is the embedding's longest row's squared length
  int n_lengths;
  int T;  // rows of this launch
  const __nv_bfloat16* H;
  long long ldh;
  const __nv_bfloat16* W;
  long long d, V;
  float cap;
  const float* logits;  // [T, ld_keys] accumulators, or
  const float* groups;  // [2, T, ld_keys] the largest and the second of every G columns
  long long ld_keys;
  int n_keys;
  int keys_in_smem;
  int k;
  const int32_t* tokens;  // [T] or null
  int32_t* ids;           // top: [T, k]
  float* logps;           // top: [T, k]; sample: [T]
  float* entropy;         // top: [T]
  float* token_logps;     // top: [T] (with tokens)
  const float* uniform;   // sample: [T] in [0, 1)
  double temperature, top_p;
  int32_t* sampled;  // sample: [T]
};

__device__ __forceinline__ int block_sum(int v, int* warp_s) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) warp_s[threadIdx.x >> 5] = v;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < kTopThreads / 32; ++w) sum += warp_s[w];
  __syncthreads();
  return sum;
}

// f64 to i64 with the same order (a NaN first, as a -inf).
__device__ __forceinline__ long long ordered_i64(double z) {
  if (z != z) z = -INFINITY;
  const long long b = __double_as_longlong(z == 0. ? 0. : z);
  return b < 0 ? b ^ 0x7fffffffffffffffll : b;
}
__device__ __forceinline__ double ordered_f64(long long b) {
  return __longlong_as_double(b < 0 ? b ^ 0x7fffffffffffffffll : b);
}

// G: columns per key (1: the keys are the accumulators).
template <bool SAMPLE, int G>
__global__ void __launch_bounds__(kTopThreads, 2) top_select_kernel(const TopParams P) {
  constexpr bool GROUPS = G > 1;
  extern __shared__ __align__(16) uint32_t keys_s[];  // where they fit
  __shared__ long long cand_z[kTopCand];
  __shared__ int cand_id[kTopCand];
  constexpr int kWarps = kTopThreads / 32;
  __shared__ __align__(16) uint32_t max_s[kTopThreads];
  __shared__ float red_s[4][kWarps];
  __shared__ uint32_t length_s[kWarps];
  __shared__ int warp_s[kWarps];
  __shared__ int n_sel_s, next_s;
  __shared__ uint32_t lo_s;
  __shared__ int sel_key[kTopSel];
  __shared__ float sel_v[2 * kTopSel];  // of the selected keys: [0, n) the keys, [n, 2 n) the second
  __shared__ float error_s, least_s;
  __shared__ long long best_i[kTopMax];
  __shared__ double best_z[kTopMax];
  __shared__ int best_id[kTopMax];
  const int t = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_keys = P.n_keys;
  const __nv_bfloat16* h = P.H + (size_t)t * P.ldh;
  const float* values = (GROUPS ? P.groups : P.logits) + (size_t)t * P.ld_keys;

  auto load_key = [&](int i) -> uint32_t {
    return ordered_key(group_value<G>(values[i]));
  };
  auto key = [&](int i) -> uint32_t { return P.keys_in_smem ? keys_s[i] : load_key(i); };

  // ---- loads: the row's partials (up to four per thread at once), hidden state and keys
  const long long token = !SAMPLE && P.tokens != nullptr ? P.tokens[t] : -1;
  constexpr int PN = 4;
  float2 pv[PN];
  float pa[PN];
#pragma unroll
  for (int j = 0; j < PN; ++j) {
    const int g = tid + j * kTopThreads;
    pv[j] = g < P.n_parts ? P.part[(size_t)g * P.T + t] : make_float2(-INFINITY, 0.f);
    pa[j] = g < P.n_parts ? P.part_a[(size_t)g * P.T + t] : 0.f;
  }
  uint32_t ww = 0u;  // the embedding's longest row, squared: as integers they have the same order, a NaN last
  for (int i = tid; i < P.n_lengths; i += kTopThreads) ww = max(ww, __float_as_uint(P.length2[i]));
  // a row of zeros: every logit is exactly 0
  int nonzero = 0;
  f32x2 hh = 0;
  for (long long i = tid; i < P.d / 8; i += kTopThreads) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(h) + i);
    nonzero |= ((a.x | a.y | a.z | a.w) & 0x7fff7fffu) != 0u;
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x2 x = pack_f32x2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
      hh = fma_f32x2(x, x, hh);
    }
  }
  uint32_t best_key = 0u;
  {
    const int n_vec = (n_keys + 3) / 4;  // rows are padded to whole vectors
#pragma unroll 4
    for (int i = tid; i < n_vec; i += kTopThreads) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(values) + i);
      uint4 k = make_uint4(ordered_key(group_value<G>(x.x)), ordered_key(group_value<G>(x.y)),
                           ordered_key(group_value<G>(x.z)), ordered_key(group_value<G>(x.w)));
      if (4 * i + 1 >= n_keys) k.y = 0u;
      if (4 * i + 2 >= n_keys) k.z = 0u;
      if (4 * i + 3 >= n_keys) k.w = 0u;
      best_key = max(max(best_key, max(k.x, k.y)), max(k.z, k.w));
      if (P.keys_in_smem) reinterpret_cast<uint4*>(keys_s)[i] = k;
    }
  }
  max_s[tid] = best_key;
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < PN; ++j) m = fmaxf(m, pv[j].x);
  for (int g = tid + PN * kTopThreads; g < P.n_parts; g += kTopThreads) m = fmaxf(m, P.part[(size_t)g * P.T + t].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float h0, h1;
  unpack_f32x2(hh, h0, h1);
  h0 += h1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) h0 += __shfl_xor_sync(0xffffffffu, h0, o);
  ww = __reduce_max_sync(0xffffffffu, ww);
  if (lane == 0) {
    red_s[0][warp] = m;
    red_s[3][warp] = h0;
    length_s[warp] = ww;
  }
  if (tid == 0) n_sel_s = 0;
  nonzero = __syncthreads_or(nonzero);

  // ---- row statistics: the partials at the row's maximum, summed in a fixed order
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red_s[0][w]);
  float s = 0.f, a = 0.f;
  auto add_part = [&](float2 p, float av) {
    if (p.y != 0.f) {
      const float dm = p.x - m, e = exp2f(dm);
      s = fmaf(p.y, e, s);
      a = fmaf(fmaf(p.y, dm, av), e, a);
    }
  };
#pragma unroll
  for (int j = 0; j < PN; ++j) add_part(pv[j], pa[j]);
  for (int g = tid + PN * kTopThreads; g < P.n_parts; g += kTopThreads)
    add_part(P.part[(size_t)g * P.T + t], P.part_a[(size_t)g * P.T + t]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    a += __shfl_xor_sync(0xffffffffu, a, o);
  }
  if (lane == 0) {
    red_s[1][warp] = s;
    red_s[2][warp] = a;
  }

  if (warp == 1) {
    float h2 = lane < kWarps ? red_s[3][lane] : 0.f;
    const uint32_t w2 = __reduce_max_sync(0xffffffffu, lane < kWarps ? length_s[lane] : 0u);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) h2 += __shfl_xor_sync(0xffffffffu, h2, o);
    if (lane == 0) error_s = top_accumulator_error(h2, __uint_as_float(w2), P.d);
  }
  uint32_t lo = 0u, reached = 0u;  // the keys from lo on are selected; k keys at least reach the other
  if (nonzero) {
    const int n = min(n_keys, P.k + kTopSpare + P.k / 16);
    // ---- a threshold that at least n keys reach, by bisection on the threads' maxima
    if (n < n_keys && warp == 0) {
      uint32_t v[kTopThreads / 32];
      uint32_t low = 0xffffffffu, top = 0u;
#pragma unroll
      for (int j = 0; j < kTopThreads / 128; ++j) {
        const uint4 x = reinterpret_cast<const uint4*>(max_s)[j * 32 + lane];
        v[4 * j] = x.x;
        v[4 * j + 1] = x.y;
        v[4 * j + 2] = x.z;
        v[4 * j + 3] = x.w;
      }
#pragma unroll
      for (int j = 0; j < kTopThreads / 32; ++j) {
        low = min(low, v[j]);
        top = max(top, v[j]);
      }
      uint32_t at = __reduce_min_sync(0xffffffffu, low);
      unsigned long long hi = (unsigned long long)__reduce_max_sync(0xffffffffu, top) + 1;
      int c_at = kTopThreads;
      while (c_at > n + kTopSpare / 2 && hi - at > 1) {
        const uint32_t mid = (uint32_t)(at + (hi - at) / 2);
        int c = 0;
#pragma unroll
        for (int j = 0; j < kTopThreads / 32; ++j) c += v[j] >= mid ? 1 : 0;
        c = (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
        if (c >= n) {
          at = mid;
          c_at = c;
        } else {
          hi = mid;
        }
      }
      if (lane == 0) lo_s = at;
    } else if (n >= n_keys && tid == 0) {
      lo_s = 0u;
    }
    __syncthreads();
    lo = reached = lo_s;
    for (int i = tid; i < n_keys; i += kTopThreads) {
      if (key(i) >= lo) {
        const int at = atomicAdd(&n_sel_s, 1);
        if (at < kTopSel) sel_key[at] = i;
      }
    }
    __syncthreads();
    if (n_sel_s > kTopSel) {
      // ---- bisection over all keys: count(key >= lo) >= n always holds, count(key >= hi) < n
      int c_lo = n_sel_s;
      unsigned long long hi = 1ull << 32;
      while (c_lo > kTopSel && hi - lo > 1) {
        const uint32_t mid = (uint32_t)(lo + (hi - lo) / 2);
        int c = 0;
        for (int i = tid; i < n_keys; i += kTopThreads) c += key(i) >= mid ? 1 : 0;
        c = block_sum(c, warp_s);
        if (c >= n) {
          lo = mid;
          c_lo = c;
        } else {
          hi = mid;
        }
      }
      reached = lo;
      if (c_lo > kTopSel) ++lo;  // more equal keys than slots: at first those above them, fewer than n
      if (tid == 0) n_sel_s = 0;
      __syncthreads();
      for (int i = tid; i < n_keys; i += kTopThreads)
        if (key(i) >= lo) sel_key[atomicAdd(&n_sel_s, 1)] = i;
      __syncthreads();
    }
  } else {
    // every logit is exactly 0: the first k tokens, or every column of the groups that hold them
    if (tid < P.k) sel_key[tid] = tid;
    if (tid == 0) n_sel_s = (P.k + G - 1) / G;
    __syncthreads();
  }
  // ---- rounds: the selected keys, then those that may still hold one of the k
  int n_sel = n_sel_s, n_best = 0;
  float least = 0.f;  // what lies below is not one of the k
  for (int pos = -1;;) {  // after the first round: where the keys that follow start
    int first = 0, cols = 0;  // candidates of this thread's key
    float v0 = -INFINITY, v1 = -INFINITY;
    if (tid < n_sel) {
      v0 = values[sel_key[tid]];
      if constexpr (GROUPS) v1 = group_value<G>(values[(size_t)P.T * P.ld_keys + sel_key[tid]]);
    }
    if (pos < 0) {
      if (tid < n_sel) {
        sel_v[tid] = group_value<G>(v0);
        sel_v[n_sel + tid] = v1;
      }
      __syncthreads();
      if (warp == 0) {
        // a value that at least k of those seen reach, and nearly no more
        constexpr int kSeen = (GROUPS ? 2 : 1) * kTopSel / 32;
        uint32_t v[kSeen];
        uint32_t top = reached;
#pragma unroll
        for (int j = 0; j < kSeen; ++j) {
          const int i = j * 32 + lane;
          v[j] = i < (GROUPS ? 2 : 1) * n_sel ? ordered_key(sel_v[i]) : 0u;
          top = max(top, v[j]);
        }
        uint32_t at = reached;
        unsigned long long hi = (unsigned long long)__reduce_max_sync(0xffffffffu, top) + 1;
        int c_at = 2 * kTopSel;
        while (c_at > P.k && hi - at > 1) {
          const uint32_t mid = (uint32_t)(at + (hi - at) / 2);
          int c = 0;
#pragma unroll
          for (int j = 0; j < kSeen; ++j) c += v[j] >= mid ? 1 : 0;
          c = (int)__reduce_add_sync(0xffffffffu, (unsigned)c);
          if (c >= P.k) {
            at = mid;
            c_at = c;
          } else {
            hi = mid;
          }
        }
        // A value that is dropped is off by as much as the k-th; the bits cut off from either are at most
        // G 2^-23 of the k-th (of a larger value above it, which stays anyway), with as much again for
        // these sums.
        const float kth = key_value(at);
        if (lane == 0) least_s = kth - 2.f * error_s - 2.f * (G * 2.384185791015625e-07f) * fabsf(kth);
      }
      __syncthreads();
      least = least_s;
    }
    if (tid < n_sel) {
      first = sel_key[tid] * G;
      cols = !nonzero || !(group_value<G>(v0) < least) ? 1 : 0;  // comparisons that a NaN fails keep
      if constexpr (GROUPS) {
        if (!nonzero || !(v1 < least)) cols = (int)min((long long)G, P.V - first);
        else first += (int)(__float_as_uint(v0) & (uint32_t)(G - 1));
      }
    }
    // where this key's candidates are: exclusive scan over the threads
    int my_at = cols;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, my_at, o);
      if (lane >= o) my_at += y;
    }
    if (lane == 31) warp_s[warp] = my_at;
    __syncthreads();
    my_at -= cols;
    int n_cand = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      my_at += w < warp ? warp_s[w] : 0;
      n_cand += warp_s[w];
    }
    // batches of candidates; the best so far take part in the next batch's ranking
    for (int b0 = 0; b0 < n_cand; b0 += kTopBatch) {
      const int have = n_best;
      const int count = have + min(kTopBatch, n_cand - b0);
      if (tid < have) {
        cand_z[tid] = best_i[tid];
        cand_id[tid] = best_id[tid];
      }
      for (int c = max(0, b0 - my_at); c < min(cols, b0 + kTopBatch - my_at); ++c)
        cand_id[have + my_at + c - b0] = first + c;
      __syncthreads();
#pragma unroll 1
      for (int i = have + warp; i < count; i += kWarps) {
        const double z = warp_score(h, P.W + (size_t)cand_id[i] * P.d, P.d, lane);
        if (lane == 0) cand_z[i] = ordered_i64(z);
      }
      __syncthreads();
      // rank by (score descending, id ascending), four threads per candidate
      for (int i0 = 0; i0 < count; i0 += kTopThreads / 4) {
        const int i = i0 + tid / 4;
        const long long z = i < count ? cand_z[i] : 0;
        const int id = i < count ? cand_id[i] : 0;
        int rank = 0;
#pragma unroll 4
        for (int j = tid % 4; j < count; j += 4) {
          const long long o = cand_z[j];
          rank += (o > z || (o == z && cand_id[j] < id)) ? 1 : 0;
        }
        rank += __shfl_xor_sync(0xffffffffu, rank, 1);
        rank += __shfl_xor_sync(0xffffffffu, rank, 2);
        if (tid % 4 == 0 && i < count && rank < P.k) {
          best_i[rank] = z;
          best_id[rank] = id;
        }
      }
      __syncthreads();
      n_best = min(P.k, count);
    }
    if (!nonzero || lo == 0u) break;  // all keys were selected
    if (n_best == P.k) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += red_s[1][w];
      if (sum != sum) break;  // a logit is NaN, or +inf without a softcap: so is all that this row answers
      const float kth = (float)ordered_f64(best_i[P.k - 1]);
      least = fmaxf(least, kth - error_s - (G * 2.384185791015625e-07f) * fabsf(kth));
    }
    if (pos < 0) {
      if (key_value(lo - 1u) < least) break;  // no key below lo can hold one of the k
      pos = 0;
    }
    // the next of them, in order
    n_sel = 0;
    while (pos < n_keys && n_sel < kTopSel) {
      const int i = pos + tid;
      const uint32_t x = i < n_keys ? key(i) : 0xffffffffu;
      const bool hit = x < lo && !(key_value(x) < least);
      const unsigned ballot = __ballot_sync(0xffffffffu, hit);
      __syncthreads();  // warp_s and next_s have been read
      if (lane == 0) warp_s[warp] = __popc(ballot);
      __syncthreads();
      int slot = n_sel + __popc(ballot & ((1u << lane) - 1u)), total = 0;
      for (int w = 0; w < kWarps; ++w) {
        slot += w < warp ? warp_s[w] : 0;
        total += warp_s[w];
      }
      if (hit && slot < kTopSel) sel_key[slot] = i;
      if (hit && slot == kTopSel) next_s = i;
      __syncthreads();
      pos = n_sel + total > kTopSel ? next_s : pos + kTopThreads;
      n_sel = min(n_sel + total, kTopSel);
    }
    if (n_sel == 0) break;
  }
  s = a = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    m = fmaxf(m, red_s[0][w]);
    s += red_s[1][w];
    a += red_s[2][w];
  }
  if (tid < P.k) {
    double x = ordered_f64(best_i[tid]);
    // a score that is not finite answers NaN: the softcap would bring it back to +-c
    if (isinf(x)) x = NAN;
    best_z[tid] = softcap_f64(x, P.cap);
  }
  __syncthreads();
  // The sums, with the best token's terms (1 of S, 0 of A) taken from its exact logit: the GEMM's is off by the
  // accumulation and the softcap's fast functions (1e-5 at c = 50), which would be all that is left of the
  // log-probability of a token that has nearly all of the mass.
  const double z_gemm = (double)m * 0.6931471805599453;
  double off = best_z[0] - z_gemm;
  if (!isfinite(off)) off = 0.;
  const double more = expm1(off), sum = (double)s + more, log_sum = log(sum);
  const double lse = z_gemm + log_sum;

  if constexpr (!SAMPLE) {
    for (int j = tid; j < P.k; j += kTopThreads) {
      P.ids[(size_t)t * P.k + j] = best_id[j];
      P.logps[(size_t)t * P.k + j] = dist_logp(best_z[j], lse);
    }
    if (tid == 0) {
      const float entropy = (float)(log_sum - ((double)a * 0.6931471805599453 + (1. + more) * off) / sum);
      P.entropy[t] = entropy < 0.f ? 0.f : entropy;  // (a NaN stays a NaN)
    }
    if (P.tokens != nullptr && warp == kTopThreads / 32 - 1) {
      const long long v = token;
      float lp = 0.f;
      if (v >= 0 && v < P.V) lp = dist_logp(softcap_f64(warp_score(h, P.W + (size_t)v * P.d, P.d, lane), P.cap), lse);
      if (lane == 0) P.token_logps[t] = lp;
    }
  } else {
    __shared__ double weight_s[kTopMax];
    if (tid < P.k) weight_s[tid] = exp((best_z[tid] - best_z[0]) / P.temperature);
    __syncthreads();
    if (warp != 0) return;
    // Inverse of the cumulative distribution of the kept prefix, in f64: kTopMax / 32 consecutive
    // ranks per lane and a scan over the lanes.
    constexpr int Q = kTopMax / 32;
    double w[Q], upto[Q];
    double run = 0.;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int j = lane * Q + q;
      w[q] = j < P.k ? weight_s[j] : 0.;
      run += w[q];
      upto[q] = run;
    }
    double incl = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    const double before = incl - run;
    const double total = __shfl_sync(0xffffffffu, incl, 31);
    const double limit = P.top_p * total;
    int kept = 0;
    double mass = 0.;  // of the kept prefix: the largest kept cumulative sum
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int j = lane * Q + q;
      upto[q] += before;
      if (j < P.k && (j == 0 || upto[q] - w[q] < limit)) {
        ++kept;
        mass = upto[q];
      }
    }
    const int n_kept = __reduce_add_sync(0xffffffffu, kept);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mass = fmax(mass, __shfl_xor_sync(0xffffffffu, mass, o));
    const double target = (double)P.uniform[t] * mass;
    int place = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (lane * Q + q < n_kept && upto[q] <= target) ++place;
    place = min((int)__reduce_add_sync(0xffffffffu, place), n_kept - 1);
    if (lane == 0) {
      P.sampled[t] = best_id[place];
      P.logps[t] = dist_logp(best_z[place], lse);
    }
  }
}

}  // namespace lpk
