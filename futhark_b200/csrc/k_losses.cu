// Two more losses of a training step and their gradients, on logits that exist.
//
// topk_distill: a student's logits S [n][v] against a teacher of which each row's top k logits T [n][k] and their
// words is [n][k] are kept (a word outside [0, v), or with a logit of -inf, is padding):
//   q_i = softmax_j(T_ij / tau) over the row's words,  lse_i = log sum_v exp(S_iv / tau)
//   loss_i = tau^2 sum_j q_ij (log q_ij - S_{i,is_ij} / tau + lse_i)
//   dS_iv  = dl_i tau (exp(S_iv / tau - lse_i) - sum_{j: is_ij = v} q_ij);     0 where a row has no word
//
// router_balance: R [n][e] logits of a router, is [n][k] the experts each token was sent to (outside [0, e): dropped),
// keep [n] (false: padding):
//   counts_e = #{(i, j): keep_i, is_ij = e},  norm = e / (sum counts * #keep),  p_i = softmax R_i
//   loss = norm sum_e counts_e sum_{i kept} p_ie
//   dR_ie = dl norm p_ie (counts_e - sum_f counts_f p_if);                     0 for padding
//
// All four are bound by memory: each direction reads its logits once and the gradients are written once.
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace fb {

constexpr float L_LOG2E = 1.4426950408889634f;
constexpr double L_LN2 = 0.69314718055994530942;

__device__ __forceinline__ float ex2_approx(float x) {   // 2^x: at most 2 units in the last place off, 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// ---- distillation -----------------------------------------------------------------------------------------
// A row is cut into parts of 2048 aligned 16-byte groups, 8 per thread of a CTA, all in flight at once; what of the
// first and last group lies outside the row is not read.  Rows of any length and start keep every SM busy this way,
// a single one included.
constexpr int D_THREADS = 256, D_PER = 8, D_GROUPS = D_THREADS * D_PER;

template <typename T> struct DistillRow {
  static constexpr int W = 16 / (int)sizeof(T);      // elements of a group
  const T *base;                                     // first element
  int64_t v;
  int off;                                           // elements of group 0 in front of the row
  __device__ DistillRow(const T *s, int64_t row, int64_t v_) : base(s + row * v_), v(v_), off((int)(((uintptr_t)base & 15) / sizeof(T))) {}
  __device__ int64_t first(int64_t group) const { return group * W - off; }      // column of the group's first element
  __device__ bool whole(int64_t group) const { return first(group) >= 0 && first(group) + W <= v; }
};

// The group's elements in f32; those outside the row are `fill`.
template <typename T>
__device__ __forceinline__ void load_group(const DistillRow<T> &r, int64_t group, float fill, float (&x)[16 / sizeof(T)]) {
  constexpr int W = DistillRow<T>::W;
  const int64_t c = r.first(group);
  if (r.whole(group)) {
    const int4 b = ld_stream_v4(r.base + c);
    const T *h = reinterpret_cast<const T *>(&b);
#pragma unroll
    for (int j = 0; j < W; j++) x[j] = to_f32<T>(h[j]);
  } else {
#pragma unroll
    for (int j = 0; j < W; j++) x[j] = c + j >= 0 && c + j < r.v ? to_f32<T>(r.base[c + j]) : fill;
  }
}

// One part of one row: maximum (in units of log 2, exactly what is subtracted) and sum.
template <typename T>
__global__ void __launch_bounds__(D_THREADS)
distill_part_kernel(const T *__restrict__ s, int64_t n, int64_t v, int parts, float scale, float2 *__restrict__ part) {
  constexpr int W = 16 / (int)sizeof(T);
  __shared__ float sm[D_THREADS / 32], ss[D_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t b = blockIdx.x; b < n * parts; b += gridDim.x) {
    const int64_t row = b / parts;
    const DistillRow<T> r(s, row, v);
    const int64_t g0 = (b - row * parts) * D_GROUPS + threadIdx.x;
    float x[D_PER][W];
#pragma unroll
    for (int i = 0; i < D_PER; i++) load_group<T>(r, g0 + i * D_THREADS, -INFINITY, x[i]);
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < D_PER; i++)
#pragma unroll
      for (int j = 0; j < W; j++) m = fmaxf(m, x[i][j]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    if (lane == 0) sm[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < D_THREADS / 32; w++) m = fmaxf(m, sm[w]);
    m *= scale;
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < D_PER; i++) {
      float t = 0.f;
#pragma unroll
      for (int j = 0; j < W; j++) t += ex2_approx(fmaf(x[i][j], scale, -ref));
      sum += t;
    }
    sum = warp_sum(sum);
    if (lane == 0) ss[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < D_THREADS / 32; w++) t += ss[w];
      part[b] = make_float2(m, t);
    }
    __syncthreads();                                 // sm and ss are used again
  }
}

__device__ __forceinline__ bool is_word(int32_t c, float t, int64_t v) { return c >= 0 && c < v && t != -INFINITY; }

// The teacher's softmax of a row over its words, one warp: maximum and sum of exp in the lanes' common registers.
__device__ __forceinline__ bool teacher_row(const int32_t *is, const float *t, int k, int64_t v, float inv_tau, int lane, float &m, float &sum) {
  m = -INFINITY;
  bool some = false;
  for (int j = lane; j < k; j += 32)
    if (is_word(is[j], t[j], v)) { some = true; m = fmaxf(m, t[j] * inv_tau); }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  sum = 0.f;
  for (int j = lane; j < k; j += 32)
    if (is_word(is[j], t[j], v)) sum += expf(t[j] * inv_tau - m);
  sum = warp_sum(sum);
  return __any_sync(kFull, some);
}

// One warp per row: fold of the parts, and the loss over the teacher's words (in f64: its terms cancel).
template <typename T>
__global__ void __launch_bounds__(256)
distill_loss_kernel(const T *__restrict__ s, const int32_t *__restrict__ is, const float *__restrict__ t, const float2 *__restrict__ part, int parts,
                    int64_t n, int64_t v, int k, float tau, float *__restrict__ loss, float *__restrict__ lse) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= n) return;
  float m = -INFINITY, sum = 0.f;
  for (int p = lane; p < parts; p += 32) {
    const float2 q = part[row * parts + p];
    const float mn = fmaxf(m, q.x), ref = mn == -INFINITY ? 0.f : mn;
    sum = sum * exp2f(m - ref) + q.y * exp2f(q.x - ref);
    m = mn;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float pm = __shfl_xor_sync(kFull, m, o), ps = __shfl_xor_sync(kFull, sum, o);
    const float mn = fmaxf(m, pm), ref = mn == -INFINITY ? 0.f : mn;
    sum = sum * exp2f(m - ref) + ps * exp2f(pm - ref);
    m = mn;
  }
  const double l = ((double)m + log2((double)sum)) * L_LN2;
  is += row * k; t += row * k; s += row * v;
  const float inv_tau = 1.f / tau;
  float tm, ts;
  const bool some = teacher_row(is, t, k, v, inv_tau, lane, tm, ts);
  const float logsum = logf(ts);
  double total = 0;
  if (some)
    for (int j = lane; j < k; j += 32) {
      const int64_t c = is[j];
      if (!is_word(is[j], t[j], v)) continue;
      const float lq = t[j] * inv_tau - tm - logsum, q = expf(lq);
      // a teacher's weight of exactly 0 adds nothing, whatever the student says
      if (q != 0.f) total += (double)q * ((double)lq - (double)to_f32<T>(s[c]) / (double)tau + l);
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
  if (lane == 0) {
    lse[row] = (float)l;
    loss[row] = (float)((double)tau * (double)tau * total);
  }
}

// One warp per row, before the gradient: per word of the teacher its weight, those of a word that stands there
// more than once added up (in the order of j) at the first place, -1 at the others.
__global__ void __launch_bounds__(256)
distill_teacher_kernel(const int32_t *__restrict__ is, const float *__restrict__ t, int64_t n, int64_t v, int k, float tau,
                       const float *__restrict__ dl, int32_t *__restrict__ words, float *__restrict__ weights, float2 *__restrict__ rows) {
  extern __shared__ float sh[];                      // [8][2][k]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + warp;
  if (row >= n) return;
  is += row * k; t += row * k;
  int *wi = reinterpret_cast<int *>(sh) + warp * 2 * k;
  float *wq = sh + warp * 2 * k + k;
  const float inv_tau = 1.f / tau;
  float tm, ts;
  const bool some = teacher_row(is, t, k, v, inv_tau, lane, tm, ts);
  const float inv = 1.f / ts;
  for (int j = lane; j < k; j += 32) {
    const int c = is[j];
    const bool in = is_word(c, t[j], v);
    wi[j] = in ? c : -1;
    wq[j] = in ? expf(t[j] * inv_tau - tm) * inv : 0.f;
  }
  __syncwarp();
  for (int j = lane; j < k; j += 32) {
    const int c = wi[j];
    float q = 0.f;
    bool first = c >= 0;
    if (c >= 0)
      for (int o = 0; o < k; o++)
        if (wi[o] == c) { if (o < j) { first = false; break; } q += wq[o]; }
    words[row * k + j] = first ? c : -1;
    weights[row * k + j] = q;
  }
  if (lane == 0) rows[row] = make_float2(dl[row] * tau, some ? 1.f : 0.f);
}

// One part of one row: the student's softmax, then the words of the teacher that lie in it once more.
template <typename T>
__global__ void __launch_bounds__(D_THREADS)
distill_grad_kernel(const T *__restrict__ s, int64_t n, int64_t v, int parts, float scale, int k, const int32_t *__restrict__ words,
                    const float *__restrict__ weights, const float2 *__restrict__ rows, const float *__restrict__ lse, T *__restrict__ ds) {
  constexpr int W = 16 / (int)sizeof(T);
  for (int64_t b = blockIdx.x; b < n * parts; b += gridDim.x) {
    const int64_t row = b / parts;
    const DistillRow<T> r(s, row, v);
    T *out = ds + row * v;
    const int64_t p0 = (b - row * parts) * D_GROUPS, g0 = p0 + threadIdx.x;
    float x[D_PER][W];
#pragma unroll
    for (int i = 0; i < D_PER; i++) load_group<T>(r, g0 + i * D_THREADS, 0.f, x[i]);
    const float2 rc = rows[row];
    const bool some = rc.y != 0.f;
    // exp(S / tau - lse) = 2^(S scale - hi) 2^-lo, hi + lo the exponent's constant term to more than 32 bits
    const double shift = (double)lse[row] / L_LN2;
    const float hi = (float)shift;
    const float f = exp2f((float)((double)hi - shift));
    auto value = [&](float xv, float q) {            // once the product with dl tau, as the definition has it
      const float p = ex2_approx(fmaf(xv, scale, -hi)) * f;
      return some ? (p - q) * rc.x : 0.f;
    };
#pragma unroll
    for (int i = 0; i < D_PER; i++) {
      const int64_t g = g0 + i * D_THREADS, c = r.first(g);
      __align__(16) T o[W];
#pragma unroll
      for (int j = 0; j < W; j++) o[j] = from_f32<T>(value(x[i][j], 0.f));
      if (r.whole(g) && ((uintptr_t)(out + c) & 15) == 0) {
        st_stream_v4(out + c, *reinterpret_cast<const int4 *>(o));
      } else {
#pragma unroll
        for (int j = 0; j < W; j++) if (c + j >= 0 && c + j < v) out[c + j] = o[j];
      }
    }
    __syncthreads();                                 // the words' places have been written
    const int64_t c0 = r.first(p0), c1 = r.first(p0 + D_GROUPS);
    for (int j = threadIdx.x; j < k; j += D_THREADS) {
      const int64_t c = words[row * k + j];
      if (c >= 0 && c >= c0 && c < c1) out[c] = from_f32<T>(value(to_f32<T>(r.base[c]), weights[row * k + j]));
    }
  }
}

static inline size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }
// parts of a row: its groups, one more if it does not start on a 16-byte boundary
static inline int64_t distill_parts(int64_t v, int elem) {
  const int64_t w = 16 / elem, groups = (v + w - 1) / w + 1;
  return (groups + D_GROUPS - 1) / D_GROUPS;
}
static inline unsigned part_grid(int64_t items) { return (unsigned)(items < (1ll << 30) ? items : (1ll << 30)); }

size_t distill_workspace_bytes(int64_t n, int64_t v, int64_t k, int elem, bool grad) {
  if (!grad) return up256((size_t)(n * distill_parts(v, elem)) * sizeof(float2));
  return up256((size_t)(n * k) * 4) * 2 + up256((size_t)n * sizeof(float2));
}

template <typename T>
static cudaError_t distill(void *workspace, const T *s, const int32_t *is, const float *t, float tau, int64_t n, int64_t v, int64_t k, float *loss,
                           float *lse, cudaStream_t stream) {
  if (n <= 0) return cudaSuccess;
  const int64_t parts = distill_parts(v, sizeof(T));
  float2 *part = reinterpret_cast<float2 *>(workspace);
  const float scale = (float)(1.0 / (L_LN2 * (double)tau));
  distill_part_kernel<T><<<part_grid(n * parts), D_THREADS, 0, stream>>>(s, n, v, (int)parts, scale, part);
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  distill_loss_kernel<T><<<(unsigned)((n + 7) / 8), 256, 0, stream>>>(s, is, t, part, (int)parts, n, v, (int)k, tau, loss, lse);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t distill_grad(void *workspace, const T *s, const int32_t *is, const float *t, float tau, const float *lse, const float *dl, int64_t n,
                                int64_t v, int64_t k, T *ds, cudaStream_t stream) {
  if (n <= 0 || v <= 0) return cudaSuccess;
  const int64_t parts = distill_parts(v, sizeof(T));
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  int32_t *words = reinterpret_cast<int32_t *>(ws);
  float *weights = reinterpret_cast<float *>(ws + up256((size_t)(n * k) * 4));
  float2 *rows = reinterpret_cast<float2 *>(ws + 2 * up256((size_t)(n * k) * 4));
  const float scale = (float)(1.0 / (L_LN2 * (double)tau));
  const size_t smem = (size_t)k * 8 * 2 * 4;
  cudaError_t err = cudaFuncSetAttribute(distill_teacher_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, DISTILL_MAX_K * 8 * 2 * 4);
  if (err != cudaSuccess) return err;
  distill_teacher_kernel<<<(unsigned)((n + 7) / 8), 256, smem, stream>>>(is, t, n, v, (int)k, tau, dl, words, weights, rows);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  distill_grad_kernel<T><<<part_grid(n * parts), D_THREADS, 0, stream>>>(s, n, v, (int)parts, scale, (int)k, words, weights, rows, lse, ds);
  return cudaGetLastError();
}

cudaError_t launch_topk_distill(void *workspace, int elem, const void *s, const int32_t *is, const float *t, float tau, int64_t n, int64_t v, int64_t k,
                                float *loss, float *lse, cudaStream_t stream) {
  if (elem == 2) return distill<__half>(workspace, reinterpret_cast<const __half *>(s), is, t, tau, n, v, k, loss, lse, stream);
  return distill<float>(workspace, reinterpret_cast<const float *>(s), is, t, tau, n, v, k, loss, lse, stream);
}
cudaError_t launch_topk_distill_grad(void *workspace, int elem, const void *s, const int32_t *is, const float *t, float tau, const float *lse,
                                     const float *dl, int64_t n, int64_t v, int64_t k, void *ds, cudaStream_t stream) {
  if (elem == 2)
    return distill_grad<__half>(workspace, reinterpret_cast<const __half *>(s), is, t, tau, lse, dl, n, v, k, reinterpret_cast<__half *>(ds), stream);
  return distill_grad<float>(workspace, reinterpret_cast<const float *>(s), is, t, tau, lse, dl, n, v, k, reinterpret_cast<float *>(ds), stream);
}

// ---- router balance ----------------------------------------------------------------------------------------
// A row belongs to G lanes of a warp (a power of two, at most 32), lane l of them has the columns l + G j, j < J.  The
// lanes keep their columns' sums in registers over all rows of the CTA, so that nothing but the row maxima and sums
// crosses lanes, and the column sums add in an order that does not depend on timing.
constexpr int R_THREADS = 256;

struct RouterShape { int g, j; };
static RouterShape router_shape(int64_t e) {
  RouterShape s = {1, 1};
  while (s.g < 32 && s.g < e) s.g *= 2;
  while ((int64_t)s.g * s.j < e) s.j *= 2;
  return s;
}

// p of the lane's columns; 0 in a row that is all -inf
template <typename T, int J>
__device__ __forceinline__ void router_softmax(const T *row, int e, int g, int l, float (&p)[J]) {
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < J; j++) {
    p[j] = l + g * j < e ? to_f32<T>(row[l + g * j]) : -INFINITY;
    m = fmaxf(m, p[j]);
  }
  for (int o = g / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < J; j++) { p[j] = ex2_approx((p[j] - ref) * L_LOG2E); sum += p[j]; }
  for (int o = g / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int j = 0; j < J; j++) p[j] *= inv;
}

// Partial results of a CTA: column sums of p [e], counts [e] and the number of rows kept.
template <typename T, int J>
__global__ void __launch_bounds__(R_THREADS)
router_part_kernel(const T *__restrict__ r, const uint8_t *__restrict__ keep, const int32_t *__restrict__ is, int64_t n, int e, int k, int g,
                   float *__restrict__ psum, int *__restrict__ pcount, int *__restrict__ ticket) {
  extern __shared__ float rsh[];                     // [8][g * J] column sums of the warps, then [e + 1] counts
  int *cnt = reinterpret_cast<int *>(rsh + (R_THREADS / 32) * g * J);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (g - 1), sub = lane / g, per_warp = 32 / g;
  for (int c = threadIdx.x; c <= e; c += R_THREADS) cnt[c] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;              // of the next kernel
  __syncthreads();
  float acc[J];
#pragma unroll
  for (int j = 0; j < J; j++) acc[j] = 0.f;
  const int64_t warps = (int64_t)gridDim.x * (R_THREADS / 32);
  int kept = 0;
  for (int64_t i0 = ((int64_t)blockIdx.x * (R_THREADS / 32) + warp) * per_warp; i0 < n; i0 += warps * per_warp) {
    const int64_t i = i0 + sub;
    const bool use = i < n && keep[i] != 0;
    float p[J];
    router_softmax<T, J>(r + (use ? i : i0) * e, e, g, l, p);        // every lane takes part in the shuffles
    if (use) {
#pragma unroll
      for (int j = 0; j < J; j++) acc[j] += p[j];
      if (l == 0) kept++;
    }
  }
#pragma unroll
  for (int j = 0; j < J; j++)
    for (int o = g; o < 32; o <<= 1) acc[j] += __shfl_xor_sync(kFull, acc[j], o);
  if (lane < g)
#pragma unroll
    for (int j = 0; j < J; j++) rsh[warp * g * J + lane + g * j] = acc[j];
  kept = warp_sum(kept);
  if (lane == 0 && kept) atomicAdd(&cnt[e], kept);
  for (int64_t o = (int64_t)blockIdx.x * R_THREADS + threadIdx.x; o < n * k; o += (int64_t)gridDim.x * R_THREADS) {
    const int c = is[o];
    if (c >= 0 && c < e && keep[o / k] != 0) atomicAdd(&cnt[c], 1);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < e; c += R_THREADS) {
    float t = 0.f;
    for (int w = 0; w < R_THREADS / 32; w++) t += rsh[w * g * J + c];
    psum[(int64_t)blockIdx.x * e + c] = t;
  }
  for (int c = threadIdx.x; c <= e; c += R_THREADS) pcount[(int64_t)blockIdx.x * (e + 1) + c] = cnt[c];
}

// 32 columns per CTA, the partial results of the CTAs over the warps, in f64; the CTA that ends last makes the loss.
__global__ void __launch_bounds__(1024)
router_loss_kernel(const float *__restrict__ psum, const int *__restrict__ pcount, int parts, int e, double *__restrict__ sums, int *__restrict__ kept,
                   int *__restrict__ ticket, int32_t *__restrict__ counts, float *__restrict__ loss, float *__restrict__ norm) {
  __shared__ double sp[32][33];
  __shared__ int sc[32][33];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  double p = 0;
  int q = 0;
  if (c <= e)
    for (int b = warp; b < parts; b += 32) {
      if (c < e) p += (double)psum[(int64_t)b * e + c];
      q += pcount[(int64_t)b * (e + 1) + c];
    }
  sp[warp][lane] = p;
  sc[warp][lane] = q;
  __syncthreads();
  if (warp == 0 && c <= e) {
    for (int w = 1; w < 32; w++) { p += sp[w][lane]; q += sc[w][lane]; }
    if (c < e) { sums[c] = p; counts[c] = q; } else *kept = q;
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(ticket, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last || warp != 0) return;
  __threadfence();
  double total = 0;
  long long all = 0;
  for (int x = lane; x < e; x += 32) {
    const int cx = __ldcg(counts + x);
    total += (double)cx * __ldcg(sums + x);
    all += cx;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { total += __shfl_xor_sync(kFull, total, o); all += __shfl_xor_sync(kFull, all, o); }
  if (lane == 0) {
    const double m = (double)__ldcg(kept);
    const double f = all > 0 && m > 0 ? (double)e / ((double)all * m) : 0.0;
    *norm = (float)f;
    *loss = all > 0 ? (float)(total * f) : 0.f;
  }
}

// Counts are taken around their mean (in integers): where they are nearly equal the gradient is what is left of a
// difference, and sum_f p_if = 1 makes the shift cancel.
template <typename T, int J>
__global__ void __launch_bounds__(R_THREADS)
router_grad_kernel(const T *__restrict__ r, const uint8_t *__restrict__ keep, const int32_t *__restrict__ counts, const float *__restrict__ norm,
                   const float *__restrict__ dl, int64_t n, int e, int g, T *__restrict__ dr) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (g - 1), sub = lane / g, per_warp = 32 / g;
  long long all = 0;
  for (int x = lane; x < e; x += 32) all += counts[x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(kFull, all, o);
  const int mean = (int)(all / e);
  float cf[J];
#pragma unroll
  for (int j = 0; j < J; j++) cf[j] = l + g * j < e ? (float)(counts[l + g * j] - mean) : 0.f;
  const float f = (float)((double)*norm * (double)*dl);
  const int64_t warps = (int64_t)gridDim.x * (R_THREADS / 32);
  for (int64_t i0 = ((int64_t)blockIdx.x * (R_THREADS / 32) + warp) * per_warp; i0 < n; i0 += warps * per_warp) {
    const int64_t i = i0 + sub;
    const bool use = i < n && keep[i] != 0;
    float p[J];
    router_softmax<T, J>(r + (use ? i : i0) * e, e, g, l, p);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < J; j++) dot = fmaf(p[j], cf[j], dot);
    for (int o = g / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
    if (i < n)
#pragma unroll
      for (int j = 0; j < J; j++)
        if (l + g * j < e) dr[i * e + l + g * j] = from_f32<T>(use ? p[j] * (cf[j] - dot) * f : 0.f);
  }
}

static int64_t router_grid(int64_t n, int64_t e, int num_sms) {
  const RouterShape s = router_shape(e);
  const int64_t rows = (int64_t)(R_THREADS / 32) * (32 / s.g);
  const int64_t want = (n + rows - 1) / rows, most = (int64_t)num_sms * 4;
  return want < 1 ? 1 : want < most ? want : most;
}

size_t router_workspace_bytes(int64_t n, int64_t e, int num_sms) {
  const int64_t grid = router_grid(n, e, num_sms);
  return up256((size_t)(grid * e) * 4) + up256((size_t)(grid * (e + 1)) * 4) + up256((size_t)e * 8) + 256;
}

template <typename T, int J>
static cudaError_t router_part(const T *r, const uint8_t *keep, const int32_t *is, int64_t n, int e, int k, int g, int grid, float *psum, int *pcount,
                               int *ticket, cudaStream_t stream) {
  const size_t smem = (size_t)(R_THREADS / 32) * g * J * 4 + (size_t)(e + 1) * 4;
  router_part_kernel<T, J><<<grid, R_THREADS, smem, stream>>>(r, keep, is, n, e, k, g, psum, pcount, ticket);
  return cudaGetLastError();
}
template <typename T, int J>
static cudaError_t router_grad(const T *r, const uint8_t *keep, const int32_t *counts, const float *norm, const float *dl, int64_t n, int e, int g,
                               int grid, T *dr, cudaStream_t stream) {
  router_grad_kernel<T, J><<<grid, R_THREADS, 0, stream>>>(r, keep, counts, norm, dl, n, e, g, dr);
  return cudaGetLastError();
}

#define FB_ROUTER_J(J_, CALL)                     \
  switch (J_) {                                   \
    case 1: { constexpr int J = 1; CALL; break; } \
    case 2: { constexpr int J = 2; CALL; break; } \
    case 4: { constexpr int J = 4; CALL; break; } \
    case 8: { constexpr int J = 8; CALL; break; } \
    case 16: { constexpr int J = 16; CALL; break; } \
    default: { constexpr int J = 32; CALL; break; } \
  }

cudaError_t launch_router_balance(void *workspace, int elem, const void *r, const uint8_t *keep, const int32_t *is, int64_t n, int64_t e, int64_t k,
                                  float *loss, int32_t *counts, float *norm, int num_sms, cudaStream_t stream) {
  const RouterShape s = router_shape(e);
  const int grid = (int)router_grid(n, e, num_sms);
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  float *psum = reinterpret_cast<float *>(ws);
  int *pcount = reinterpret_cast<int *>(ws + up256((size_t)grid * e * 4));
  double *sums = reinterpret_cast<double *>(reinterpret_cast<uint8_t *>(pcount) + up256((size_t)grid * (e + 1) * 4));
  int *kept = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(sums) + up256((size_t)e * 8));
  int *ticket = kept + 1;
  cudaError_t err = cudaSuccess;
  if (elem == 2) { FB_ROUTER_J(s.j, (err = router_part<__half, J>(reinterpret_cast<const __half *>(r), keep, is, n, (int)e, (int)k, s.g, grid, psum, pcount, ticket, stream))) }
  else { FB_ROUTER_J(s.j, (err = router_part<float, J>(reinterpret_cast<const float *>(r), keep, is, n, (int)e, (int)k, s.g, grid, psum, pcount, ticket, stream))) }
  if (err != cudaSuccess) return err;
  router_loss_kernel<<<(unsigned)((e + 1 + 31) / 32), 1024, 0, stream>>>(psum, pcount, grid, (int)e, sums, kept, ticket, counts, loss, norm);
  return cudaGetLastError();
}

cudaError_t launch_router_balance_grad(int elem, const void *r, const uint8_t *keep, const int32_t *counts, const float *norm, const float *dl, int64_t n,
                                       int64_t e, void *dr, int num_sms, cudaStream_t stream) {
  if (n <= 0 || e <= 0) return cudaSuccess;
  const RouterShape s = router_shape(e);
  const int grid = (int)router_grid(n, e, num_sms);
  cudaError_t err = cudaSuccess;
  if (elem == 2) { FB_ROUTER_J(s.j, (err = router_grad<__half, J>(reinterpret_cast<const __half *>(r), keep, counts, norm, dl, n, (int)e, s.g, grid, reinterpret_cast<__half *>(dr), stream))) }
  else { FB_ROUTER_J(s.j, (err = router_grad<float, J>(reinterpret_cast<const float *>(r), keep, counts, norm, dl, n, (int)e, s.g, grid, reinterpret_cast<float *>(dr), stream))) }
  return err;
}

}  // namespace fb
