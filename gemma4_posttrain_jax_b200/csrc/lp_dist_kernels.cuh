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
  float m, s, a;  // base 2: max, sum 2^(z-m), sum 2^(z-m) (z-m); s == 0: nothing yet
};

__device__ __forceinline__ DistAcc dist_merge(const DistAcc& x, const DistAcc& y) {
  if (y.s == 0.f) return x;
  if (x.s == 0.f) return y;
  DistAcc r;
  r.m = fmaxf(x.m, y.m);
  const float dx = x.m - r.m, dy = y.m - r.m;
  const float ex = exp2f(dx), ey = exp2f(dy);
  r.s = x.s * ex + y.s * ey;
  r.a = fmaf(x.s, dx, x.a) * ex + fmaf(y.s, dy, y.a) * ey;
  return r;
}

__device__ __forceinline__ float dist_lse(const DistAcc& x) { return x.m * kLn2 + logf(x.s); }
__device__ __forceinline__ float dist_entropy(const DistAcc& x) { return logf(x.s) - kLn2 * (x.a / x.s); }

// A log-probability is never above 0; the roundings of z and lse can leave it there by an ulp
// (a NaN stays a NaN).
__device__ __forceinline__ float dist_logp(float z, float lse) {
  const float lp = z - lse;
  return lp > 0.f ? 0.f : lp;
}

__device__ __forceinline__ float softcap_exact(float x, float cap) { return cap > 0.f ? cap * tanhf(x / cap) : x; }

// Raw dot product h . w over one warp (every lane returns it): 16-byte loads, products of two
// bf16 numbers are exact in f32.
__device__ __forceinline__ float warp_dot(const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ w,
                                          long long d, int lane) {
  float acc0 = 0.f, acc1 = 0.f;
  for (long long i = lane; i < d / 8; i += 32) {
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

// The same in f64. The products are exact and a sum of bf16 products rarely needs more than 53
// bits, so equal dot products compare equal whatever the order of the sum.
__device__ __forceinline__ double warp_dot_f64(const __nv_bfloat16* __restrict__ h,
                                               const __nv_bfloat16* __restrict__ w, long long d, int lane) {
  double acc0 = 0., acc1 = 0.;
  for (long long i = lane; i < d / 8; i += 32) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(h) + i);
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(w) + i);
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc0 += (double)(__uint_as_float(av[j] << 16) * __uint_as_float(bv[j] << 16));
      acc1 += (double)(__uint_as_float(av[j] & 0xffff0000u) * __uint_as_float(bv[j] & 0xffff0000u));
    }
  }
  double acc = acc0 + acc1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  return acc;
}

// Merges the GEMM's partials of R consecutive rows per block and computes the given tokens'
// logits, one warp per (row, token) pair.
//   stats (optional, [3, T]): m, S, A of this shard in natural units, for dist_combine_kernel
//   zt [T, K]: softcapped logit of tokens owned by this shard, else 0
//   lse, entropy, logp (optional): valid where the shard is the whole vocabulary; a token
//   outside [0, Vs) has logp 0
constexpr int kDistThreads = 256;

template <int R>
__global__ void __launch_bounds__(kDistThreads)
    dist_finalize_kernel(const float2* __restrict__ part, const float* __restrict__ part_a, int n_parts, int T,
                         const __nv_bfloat16* __restrict__ H, long long ldh, const __nv_bfloat16* __restrict__ W,
                         long long d, long long Vs, long long v_off, const int32_t* __restrict__ y, int K, float cap,
                         float* __restrict__ stats, float* __restrict__ zt, float* __restrict__ lse,
                         float* __restrict__ entropy, float* __restrict__ logp) {
  __shared__ DistAcc acc_s[kDistThreads];
  __shared__ float lse_s[R];
  const int t0 = blockIdx.x * R;
  const int r = threadIdx.x % R;
  const int t = t0 + r;
  DistAcc acc{-INFINITY, 0.f, 0.f};
  if (t < T) {
    for (int g = threadIdx.x / R; g < n_parts; g += kDistThreads / R) {
      const float2 p = part[(size_t)g * T + t];
      acc = dist_merge(acc, DistAcc{p.x, p.y, part_a[(size_t)g * T + t]});
    }
  }
  acc_s[threadIdx.x] = acc;
  __syncthreads();
#pragma unroll
  for (int o = kDistThreads / 2; o >= R; o >>= 1) {
    if ((int)threadIdx.x < o) acc_s[threadIdx.x] = dist_merge(acc_s[threadIdx.x], acc_s[threadIdx.x + o]);
    __syncthreads();
  }
  if (threadIdx.x < R && t < T) {
    acc = acc_s[threadIdx.x];
    const float l = dist_lse(acc);
    lse_s[threadIdx.x] = l;
    if (stats != nullptr) {
      stats[t] = acc.m * kLn2;
      stats[(size_t)T + t] = acc.s;
      stats[(size_t)2 * T + t] = acc.a * kLn2;
    }
    if (lse != nullptr) lse[t] = l;
    if (entropy != nullptr) entropy[t] = dist_entropy(acc);
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = min(R, T - t0);
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

// The given tokens' entries of a chunk's dZ, computed from their f32 logits and rounded once:
//   dZ[t, y] = softcap'(z) * (sum of g over the row's slots that hold y - p * (a + b log2 p))
// softcap'(z) = 1 - (z / c)^2. The first slot of a token writes the entry, so a token that a row
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
  const float z = zt[i];
  const float lp = fmaf(z, kLog2e, -row_const[2 * row_ld + t]);
  const float u = cap > 0.f ? z / cap : 0.f;
  const float w = fmaf(row_const[row_ld + t], lp, row_const[t]);
  dz[(size_t)t * ldz + v] = __float2bfloat16_rn(fmaf(-u, u, 1.f) * (sum - exp2f(lp) * w));
}

// ----------------------------------------------------------------------------- selection
// The k most likely tokens of a row, in the order of the exact dot products h . W_v (softcap is
// monotone), the lowest id first among equals. The GEMM only nominates: a key is either one
// accumulator (f32) or the largest of 32 neighbours with the second largest beside it. The
// k + kTopSpare largest keys are selected; of a selected group every column is a candidate if its
// second largest reaches the k-th largest value seen, else only its largest is. Candidates are
// scored again in f64 and ranked by that, so a rounding of the nomination (f32 accumulation, 2^-18
// for a group's low bits) can exchange neighbours only if more than kTopSpare values lie within it
// of the k-th.
constexpr int kTopMax = 128;
constexpr int kTopSpare = 16;
constexpr int kTopGroup = 32;
constexpr int kTopThreads = 512;
// selected keys: at most k + 2 kTopSpare, or any number up to this of equal ones
constexpr int kTopSel = kTopMax + 2 * kTopSpare;
constexpr int kTopCand = kTopSel * kTopGroup;
constexpr int kTopCandBytes = kTopCand * (int)(sizeof(double) + sizeof(int));
constexpr int kTopKeyBytes = 200 * 1024 - 16 * 1024;  // keys kept in shared memory, beside the static part

// Order-preserving map of f32 to u32; NaN comes last.
__device__ __forceinline__ uint32_t ordered_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
// A group's value without its column bits.
__device__ __forceinline__ float group_value(float x) { return __uint_as_float(__float_as_uint(x) & ~31u); }

struct TopParams {
  const float2* part;
  const float* part_a;
  int n_parts;
  int T;  // rows of this launch
  const __nv_bfloat16* H;
  long long ldh;
  const __nv_bfloat16* W;
  long long d, V;
  float cap;
  const float* logits;  // [T, ld_keys] accumulators, or
  const float2* groups;  // [T, ld_keys] the two largest of every 32
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
  float temperature, top_p;
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

template <bool SAMPLE, bool GROUPS>
__global__ void __launch_bounds__(kTopThreads) top_select_kernel(const TopParams P) {
  // keys while selecting, then the candidates' f64 scores and ids
  extern __shared__ __align__(16) uint8_t dyn_s[];
  uint32_t* keys_s = reinterpret_cast<uint32_t*>(dyn_s);
  double* cand_z = reinterpret_cast<double*>(dyn_s);
  int* cand_id = reinterpret_cast<int*>(dyn_s + kTopCand * sizeof(double));
  __shared__ DistAcc acc_s[kTopThreads / 32];
  __shared__ int warp_s[kTopThreads / 32];
  __shared__ int n_sel_s, n_cand_s;
  __shared__ int sel_key[kTopSel];
  __shared__ float sel_v[2 * kTopSel];  // values of the selected keys: [0, n) largest, [n, 2n) second
  __shared__ float kth_s;
  __shared__ double best_z[kTopMax];
  __shared__ int best_id[kTopMax];
  const int t = blockIdx.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n_keys = P.n_keys;
  const __nv_bfloat16* h = P.H + (size_t)t * P.ldh;

  auto load_key = [&](int i) -> uint32_t {
    if constexpr (GROUPS) return ordered_key(group_value(P.groups[(size_t)t * P.ld_keys + i].x));
    else return ordered_key(P.logits[(size_t)t * P.ld_keys + i]);
  };
  auto key = [&](int i) -> uint32_t { return P.keys_in_smem ? keys_s[i] : load_key(i); };

  // a row of zeros: every logit is exactly 0
  int nonzero = 0;
  for (long long i = tid; i < P.d / 8; i += kTopThreads) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(h) + i);
    nonzero |= ((a.x | a.y | a.z | a.w) & 0x7fff7fffu) != 0u;
  }
  if (P.keys_in_smem)
    for (int i = tid; i < n_keys; i += kTopThreads) keys_s[i] = load_key(i);
  // row statistics
  DistAcc acc{-INFINITY, 0.f, 0.f};
  for (int g = tid; g < P.n_parts; g += kTopThreads) {
    const float2 p = P.part[(size_t)g * P.T + t];
    acc = dist_merge(acc, DistAcc{p.x, p.y, P.part_a[(size_t)g * P.T + t]});
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    DistAcc b;
    b.m = __shfl_xor_sync(0xffffffffu, acc.m, o);
    b.s = __shfl_xor_sync(0xffffffffu, acc.s, o);
    b.a = __shfl_xor_sync(0xffffffffu, acc.a, o);
    acc = (lane & o) ? dist_merge(b, acc) : dist_merge(acc, b);
  }
  if (lane == 0) acc_s[warp] = acc;
  if (tid == 0) n_sel_s = n_cand_s = 0;
  nonzero = __syncthreads_or(nonzero);
  acc = acc_s[0];
#pragma unroll
  for (int w = 1; w < kTopThreads / 32; ++w) acc = dist_merge(acc, acc_s[w]);
  const float lse = dist_lse(acc);

  if (nonzero) {
    // Bisection on the ordered keys: count(key >= lo) >= n always holds, count(key >= hi) < n.
    const int n = min(n_keys, P.k + kTopSpare);
    uint32_t lo = 0u;
    unsigned long long hi = 1ull << 32;
    int c_lo = n_keys;
    while (c_lo > n + kTopSpare && hi - lo > 1) {
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
    const bool ties = c_lo > kTopSel;  // then hi = lo + 1: more equal keys than slots
    for (int i = tid; i < n_keys; i += kTopThreads) {
      const uint32_t x = key(i);
      if (ties ? x > lo : x >= lo) sel_key[atomicAdd(&n_sel_s, 1)] = i;
    }
    __syncthreads();
    if (ties) {
      // fewer than n keys lie above the tie; fill up to n with the lowest of the tie
      int have = n_sel_s;
      __syncthreads();
      for (int base = 0; base < n_keys && have < n; base += kTopThreads) {
        const int i = base + tid;
        const bool hit = i < n_keys && key(i) == lo;
        const unsigned ballot = __ballot_sync(0xffffffffu, hit);
        if (lane == 0) warp_s[warp] = __popc(ballot);
        __syncthreads();
        int before = 0, total = 0;
        for (int w = 0; w < kTopThreads / 32; ++w) {
          before += w < warp ? warp_s[w] : 0;
          total += warp_s[w];
        }
        const int slot = have + before + __popc(ballot & ((1u << lane) - 1u));
        if (hit && slot < n) sel_key[slot] = i;
        have = min(n, have + total);
        __syncthreads();
      }
      if (tid == 0) n_sel_s = n;
      __syncthreads();
    }
    const int n_sel = n_sel_s;  // the keys in shared memory are not read below
    if constexpr (GROUPS) {
      float b0 = -INFINITY, b1 = -INFINITY;
      if (tid < n_sel) {
        const float2 g = P.groups[(size_t)t * P.ld_keys + sel_key[tid]];
        b0 = g.x;
        b1 = group_value(g.y);
        sel_v[tid] = group_value(b0);
        sel_v[n_sel + tid] = b1;
      }
      if (tid == 0) kth_s = -INFINITY;
      __syncthreads();
      // the k-th largest of the values seen is a lower bound of the k-th largest logit
      for (int i = tid; i < 2 * n_sel; i += kTopThreads) {
        const float v = sel_v[i];
        int above = 0;
        for (int j = 0; j < 2 * n_sel; ++j) above += (sel_v[j] > v || (sel_v[j] == v && j < i)) ? 1 : 0;
        if (above == P.k - 1) kth_s = v;
      }
      __syncthreads();
      if (tid < n_sel) {
        const long long first = (long long)sel_key[tid] * kTopGroup;
        const int cols = (int)min((long long)kTopGroup, P.V - first);
        // 2^-16 of slack for the accumulation and the bits cut off
        const float least = kth_s - 1.52587890625e-05f * fabsf(kth_s);
        if (!(b1 < least)) {
          const int at = atomicAdd(&n_cand_s, cols);
          for (int c = 0; c < cols; ++c) cand_id[at + c] = (int)first + c;
        } else {
          cand_id[atomicAdd(&n_cand_s, 1)] = (int)first + (int)(__float_as_uint(b0) & 31u);
        }
      }
    } else {
      if (tid < n_sel) cand_id[tid] = sel_key[tid];
      if (tid == 0) n_cand_s = n_sel;
    }
  } else {
    if (tid < P.k) cand_id[tid] = tid;
    if (tid == 0) n_cand_s = P.k;
  }
  __syncthreads();
  const int n_cand = n_cand_s;

  for (int i = warp; i < n_cand; i += kTopThreads / 32) {
    const double z = warp_dot_f64(h, P.W + (size_t)cand_id[i] * P.d, P.d, lane);
    if (lane == 0) cand_z[i] = z == z ? z : -INFINITY;  // a NaN ranks last
  }
  __syncthreads();
  // rank by (z descending, id ascending)
  for (int i = tid; i < n_cand; i += kTopThreads) {
    const double z = cand_z[i];
    const int id = cand_id[i];
    int rank = 0;
    for (int j = 0; j < n_cand; ++j) rank += (cand_z[j] > z || (cand_z[j] == z && cand_id[j] < id)) ? 1 : 0;
    if (rank < P.k) {
      best_z[rank] = P.cap > 0.f ? (double)P.cap * tanh(z / (double)P.cap) : z;
      best_id[rank] = id;
    }
  }
  __syncthreads();

  if constexpr (!SAMPLE) {
    for (int j = tid; j < P.k; j += kTopThreads) {
      P.ids[(size_t)t * P.k + j] = best_id[j];
      P.logps[(size_t)t * P.k + j] = dist_logp((float)best_z[j], lse);
    }
    if (tid == 0) P.entropy[t] = dist_entropy(acc);
    if (P.tokens != nullptr && warp == kTopThreads / 32 - 1) {
      const long long v = P.tokens[t];
      float lp = 0.f;
      if (v >= 0 && v < P.V) lp = dist_logp(softcap_exact(warp_dot(h, P.W + (size_t)v * P.d, P.d, lane), P.cap), lse);
      if (lane == 0) P.token_logps[t] = lp;
    }
  } else if (warp == 0) {
    // Inverse of the cumulative distribution of the kept prefix, in f64: kTopMax / 32 consecutive
    // ranks per lane and a scan over the lanes.
    constexpr int Q = kTopMax / 32;
    double w[Q], upto[Q];
    double run = 0.;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int j = lane * Q + q;
      w[q] = j < P.k ? exp((best_z[j] - best_z[0]) / (double)P.temperature) : 0.;
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
    const double limit = (double)P.top_p * total;
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
      P.logps[t] = dist_logp((float)best_z[place], lse);
    }
  }
}

}  // namespace lpk
