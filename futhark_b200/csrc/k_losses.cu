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
// A row is read in aligned 16-byte groups; what of the first and last group lies outside the row is not read.  It is cut
// into parts of at most 2048 groups, each worked on by `tpr` threads (32 to 256; CTAs have 256 and as many rows as
// fit) with up to 8 groups per thread, all in flight at once.  Rows of any length and start keep every SM busy this way,
// a single one included.
constexpr int D_THREADS = 256;
struct DistillShape {
  int parts, tpr, per;               // parts of a row, threads of a part, groups of a thread (1, 2, 4 or 8)
};
static DistillShape distill_shape(int64_t v, int elem) {
  const int64_t w = 16 / elem, groups = (v + w - 1) / w + 1;          // one more if the row starts inside a group
  DistillShape s;
  s.parts = (int)((groups + D_THREADS * 8 - 1) / (D_THREADS * 8));
  const int64_t g = (groups + s.parts - 1) / s.parts;
  s.tpr = 32;
  while (s.tpr < D_THREADS && s.tpr * 8 < g) s.tpr *= 2;
  s.per = 1;
  while (s.per < 8 && s.tpr * s.per < g) s.per *= 2;
  return s;
}

template <typename T> struct DistillRow {
  static constexpr int W = 16 / (int)sizeof(T);      // elements of a group
  const T *base;                                     // first element
  int v;
  int off;                                           // elements of group 0 in front of the row
  __device__ DistillRow(const T *s, int64_t row, int64_t v_) : base(s + row * v_), v((int)v_), off((int)(((uintptr_t)base & 15) / sizeof(T))) {}
  __device__ int first(int group) const { return group * W - off; }      // column of the group's first element
  __device__ bool whole(int group) const { return first(group) >= 0 && first(group) + W <= v; }
};

// The group's elements as they lie in memory; those outside the row are -inf.
template <typename T>
__device__ __forceinline__ int4 load_group(const DistillRow<T> &r, int group) {
  constexpr int W = DistillRow<T>::W;
  const int c = r.first(group);
  if (r.whole(group)) return ld_stream_v4(r.base + c);
  __align__(16) T x[W];
#pragma unroll
  for (int j = 0; j < W; j++) x[j] = c + j >= 0 && c + j < r.v ? r.base[c + j] : from_f32<T>(-INFINITY);
  return *reinterpret_cast<const int4 *>(x);
}
__device__ __forceinline__ void unpack(const int4 &b, float (&x)[4]) {
  x[0] = __int_as_float(b.x); x[1] = __int_as_float(b.y); x[2] = __int_as_float(b.z); x[3] = __int_as_float(b.w);
}
__device__ __forceinline__ void unpack(const int4 &b, float (&x)[8]) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&b);
#pragma unroll
  for (int j = 0; j < 4; j++) { const float2 f = __half22float2(h[j]); x[2 * j] = f.x; x[2 * j + 1] = f.y; }
}
__device__ __forceinline__ int4 pack(const float (&x)[4]) {
  return make_int4(__float_as_int(x[0]), __float_as_int(x[1]), __float_as_int(x[2]), __float_as_int(x[3]));
}
__device__ __forceinline__ int4 pack(const float (&x)[8]) {
  int4 b;
  __half2 *h = reinterpret_cast<__half2 *>(&b);
#pragma unroll
  for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
  return b;
}

// (maximum in units of log 2, exactly what was subtracted; sum): the fold of two
__device__ __forceinline__ void fold_pair(float &m, float &s, float om, float os) {
  const float mn = fmaxf(m, om), ref = mn == -INFINITY ? 0.f : mn;
  s = s * exp2f(m - ref) + os * exp2f(om - ref);
  m = mn;
}

// One part of one row.
template <typename T, int PER>
__global__ void __launch_bounds__(D_THREADS, 4)
distill_part_kernel(const T *__restrict__ s, int64_t n, int64_t v, int parts, int tpr, float scale, float2 *__restrict__ part) {
  constexpr int W = 16 / (int)sizeof(T);
  __shared__ float2 sm[D_THREADS / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = threadIdx.x & (tpr - 1), rpc = D_THREADS / tpr;
  const int64_t items = n * parts;
  for (int64_t b0 = (int64_t)blockIdx.x * rpc; b0 < items; b0 += (int64_t)gridDim.x * rpc) {
    const int64_t b = b0 + threadIdx.x / tpr;
    float m = -INFINITY, sum = 0.f;
    if (b < items) {                                 // uniform over the warp
      const int64_t row = b / parts;
      const DistillRow<T> r(s, row, v);
      const int g0 = (int)(b - row * parts) * (tpr * PER) + t;
      int4 x[PER];
#pragma unroll
      for (int i = 0; i < PER; i++) x[i] = load_group<T>(r, g0 + i * tpr);
#pragma unroll
      for (int i = 0; i < PER; i++) {
        float f[W];
        unpack(x[i], f);
#pragma unroll
        for (int j = 0; j < W; j++) m = fmaxf(m, f[j]);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
      m *= scale;
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        float f[W], a = 0.f, c = 0.f;
        unpack(x[i], f);
#pragma unroll
        for (int j = 0; j < W; j += 2) { a += ex2_approx(fmaf(f[j], scale, -ref)); c += ex2_approx(fmaf(f[j + 1], scale, -ref)); }
        sum += a + c;
      }
      sum = warp_sum(sum);
    }
    if (tpr > 32) {
      if (lane == 0) sm[warp] = make_float2(m, sum);
      __syncthreads();
      if (t == 0)
        for (int w = 1; w < tpr / 32; w++) fold_pair(m, sum, sm[warp + w].x, sm[warp + w].y);
      __syncthreads();                               // sm is used again
    }
    if (t == 0 && b < items) part[b] = make_float2(m, sum);
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
    fold_pair(m, sum, q.x, q.y);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float pm = __shfl_xor_sync(kFull, m, o), ps = __shfl_xor_sync(kFull, sum, o);
    fold_pair(m, sum, pm, ps);
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
// more than once added up (in the order of j) at the first place, -1 at the others.  Whether one does is seen by a hash
// table of the words; only then are they compared with one another.
__global__ void __launch_bounds__(256)
distill_teacher_kernel(const int32_t *__restrict__ is, const float *__restrict__ t, int64_t n, int64_t v, int k, int table, float tau,
                       const float *__restrict__ dl, int32_t *__restrict__ words, float *__restrict__ weights, float2 *__restrict__ rows) {
  extern __shared__ float sh[];                      // per warp: words [k], weights [k], places [table]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + warp;
  if (row >= n) return;
  is += row * k; t += row * k;
  int *wi = reinterpret_cast<int *>(sh) + warp * (2 * k + table);
  float *wq = reinterpret_cast<float *>(wi + k);
  int *place = wi + 2 * k;
  const float inv_tau = 1.f / tau;
  float tm, ts;
  const bool some = teacher_row(is, t, k, v, inv_tau, lane, tm, ts);
  const float inv = 1.f / ts;
  for (int h = lane; h < table; h += 32) place[h] = -1;
  for (int j = lane; j < k; j += 32) {
    const int c = is[j];
    const bool in = is_word(c, t[j], v);
    wi[j] = in ? c : -1;
    wq[j] = in ? expf(t[j] * inv_tau - tm) * inv : 0.f;
  }
  __syncwarp();
  bool twice = false;
  for (int j = lane; j < k; j += 32) {
    const int c = wi[j];
    if (c < 0) continue;
    for (int h = (int)(((uint32_t)c * 2654435761u) >> 16) & (table - 1);; h = (h + 1) & (table - 1)) {   // at least half of the table is free
      const int at = atomicCAS(place + h, -1, c);
      if (at == -1) break;
      if (at == c) { twice = true; break; }
    }
  }
  twice = __any_sync(kFull, twice);
  for (int j = lane; j < k; j += 32) {
    const int c = wi[j];
    float q = wq[j];
    bool first = c >= 0;
    if (twice && c >= 0) {
      q = 0.f;
      for (int o = 0; o < k; o++)
        if (wi[o] == c) { if (o < j) first = false; q += wq[o]; }
    }
    words[row * k + j] = first ? c : -1;
    weights[row * k + j] = q;
  }
  if (lane == 0) rows[row] = make_float2(dl[row] * tau, some ? 1.f : 0.f);
}

// One part of one row: the student's softmax, then the words of the teacher that lie in it once more.
template <typename T, int PER>
__global__ void __launch_bounds__(D_THREADS, 4)
distill_grad_kernel(const T *__restrict__ s, int64_t n, int64_t v, int parts, int tpr, float scale, int k, const int32_t *__restrict__ words,
                    const float *__restrict__ weights, const float2 *__restrict__ rows, const float *__restrict__ lse, T *__restrict__ ds) {
  constexpr int W = 16 / (int)sizeof(T);
  const int t = threadIdx.x & (tpr - 1), rpc = D_THREADS / tpr;
  const int64_t items = n * parts;
  for (int64_t b0 = (int64_t)blockIdx.x * rpc; b0 < items; b0 += (int64_t)gridDim.x * rpc) {
    const int64_t b = b0 + threadIdx.x / tpr;
    const bool active = b < items;
    const int64_t row = active ? b / parts : 0;
    const DistillRow<T> r(s, row, v);
    T *out = ds + row * v;
    const int p0 = (int)(b - row * parts) * (tpr * PER), g0 = p0 + t;
    // exp(S / tau - lse) = 2^(S scale - hi) 2^-lo, hi + lo the exponent's constant term to more than 32 bits
    float hi = 0.f, f = 0.f, c = 0.f;
    bool some = false;
    if (active) {
      int4 x[PER];
#pragma unroll
      for (int i = 0; i < PER; i++) x[i] = load_group<T>(r, g0 + i * tpr);
      const float2 rc = rows[row];
      const double shift = (double)lse[row] / L_LN2;
      c = rc.x;
      some = rc.y != 0.f;
      hi = (float)shift;
      f = exp2f((float)((double)hi - shift));
      const float fc = f * c;
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int g = g0 + i * tpr, col = r.first(g);
        float y[W];
        unpack(x[i], y);
#pragma unroll
        for (int j = 0; j < W; j++) y[j] = some ? ex2_approx(fmaf(y[j], scale, -hi)) * fc : 0.f;
        if (r.whole(g) && ((uintptr_t)(out + col) & 15) == 0) {
          st_stream_v4(out + col, pack(y));
        } else {
#pragma unroll
          for (int j = 0; j < W; j++) if (col + j >= 0 && col + j < r.v) out[col + j] = from_f32<T>(y[j]);
        }
      }
    }
    __syncthreads();                                 // the words' places have been written
    if (active && some) {
      const int c0 = r.first(p0), c1 = r.first(p0 + tpr * PER);
      for (int j = t; j < k; j += tpr) {
        const int w = words[row * k + j];
        if (w >= 0 && w >= c0 && w < c1) {
          const float p = ex2_approx(fmaf(to_f32<T>(r.base[w]), scale, -hi)) * f;
          out[w] = from_f32<T>((p - weights[row * k + j]) * c);
        }
      }
    }
  }
}

static inline size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }
static inline unsigned part_grid(int64_t items, int per_cta) {
  const int64_t g = (items + per_cta - 1) / per_cta;
  return (unsigned)(g < (1ll << 30) ? g : (1ll << 30));
}

size_t distill_workspace_bytes(int64_t n, int64_t v, int64_t k, int elem, bool grad) {
  if (!grad) return up256((size_t)n * distill_shape(v, elem).parts * sizeof(float2));
  return up256((size_t)(n * k) * 4) * 2 + up256((size_t)n * sizeof(float2));
}

#define FB_DISTILL_PER(PER_, CALL)                    \
  switch (PER_) {                                     \
    case 1: { constexpr int PER = 1; CALL; break; }   \
    case 2: { constexpr int PER = 2; CALL; break; }   \
    case 4: { constexpr int PER = 4; CALL; break; }   \
    default: { constexpr int PER = 8; CALL; break; }  \
  }

template <typename T>
static cudaError_t distill(void *workspace, const T *s, const int32_t *is, const float *t, float tau, int64_t n, int64_t v, int64_t k, float *loss,
                           float *lse, cudaStream_t stream) {
  if (n <= 0) return cudaSuccess;
  const DistillShape sh = distill_shape(v, sizeof(T));
  float2 *part = reinterpret_cast<float2 *>(workspace);
  const float scale = (float)(1.0 / (L_LN2 * (double)tau));
  const unsigned grid = part_grid(n * sh.parts, D_THREADS / sh.tpr);
  FB_DISTILL_PER(sh.per, (distill_part_kernel<T, PER><<<grid, D_THREADS, 0, stream>>>(s, n, v, sh.parts, sh.tpr, scale, part)))
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  distill_loss_kernel<T><<<(unsigned)((n + 7) / 8), 256, 0, stream>>>(s, is, t, part, sh.parts, n, v, (int)k, tau, loss, lse);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t distill_grad(void *workspace, const T *s, const int32_t *is, const float *t, float tau, const float *lse, const float *dl, int64_t n,
                                int64_t v, int64_t k, T *ds, cudaStream_t stream) {
  if (n <= 0 || v <= 0) return cudaSuccess;
  const DistillShape sh = distill_shape(v, sizeof(T));
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  int32_t *words = reinterpret_cast<int32_t *>(ws);
  float *weights = reinterpret_cast<float *>(ws + up256((size_t)(n * k) * 4));
  float2 *rows = reinterpret_cast<float2 *>(ws + 2 * up256((size_t)(n * k) * 4));
  const float scale = (float)(1.0 / (L_LN2 * (double)tau));
  int table = 32;
  while (table < 2 * k) table *= 2;
  cudaError_t err = cudaFuncSetAttribute(distill_teacher_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * (2 * DISTILL_MAX_K + 2 * DISTILL_MAX_K) * 4);
  if (err != cudaSuccess) return err;
  distill_teacher_kernel<<<(unsigned)((n + 7) / 8), 256, (size_t)8 * (2 * k + table) * 4, stream>>>(is, t, n, v, (int)k, table, tau, dl, words, weights, rows);
  err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  const unsigned grid = part_grid(n * sh.parts, D_THREADS / sh.tpr);
  FB_DISTILL_PER(sh.per, (distill_grad_kernel<T, PER><<<grid, D_THREADS, 0, stream>>>(s, n, v, sh.parts, sh.tpr, scale, (int)k, words, weights, rows, lse, ds)))
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
// A row belongs to G lanes of a warp (a power of two, at most 32), each of which has J groups of W consecutive columns
// (W = 4 where rows are made of whole aligned groups, 1 otherwise).  The lanes keep their columns' sums in
// registers over all rows of the CTA, so that nothing but the row maxima and sums crosses lanes, and the column sums
// add in an order that does not depend on timing.  The next row is loaded before this one is worked on: a warp's
// rows are short chains of dependent steps, and two rows in flight per warp are what hides them.
constexpr int R_THREADS = 256;

struct RouterShape { int w, g, j; };
static RouterShape router_shape(const void *r, int64_t e, int elem) {
  RouterShape s = {e % 4 == 0 && ((uintptr_t)r & (4 * elem - 1)) == 0 ? 4 : 1, 1, 1};
  while (s.g < 32 && s.g * s.w < e) s.g *= 2;
  while ((int64_t)s.g * s.w * s.j < e) s.j *= 2;
  return s;
}

template <typename T, int W> struct RouterGroup;
template <> struct RouterGroup<float, 4> { using type = float4; };
template <> struct RouterGroup<float, 1> { using type = float; };
template <> struct RouterGroup<__half, 4> { using type = uint2; };
template <> struct RouterGroup<__half, 1> { using type = __half; };

template <typename T, int W, int J> struct RouterRow {
  typename RouterGroup<T, W>::type x[J];
  __device__ __forceinline__ void load(const T *row, int e, int g, int l) {
#pragma unroll
    for (int j = 0; j < J; j++)
      if ((l + g * j) * W < e) x[j] = *reinterpret_cast<const typename RouterGroup<T, W>::type *>(row + (l + g * j) * W);
  }
  // p of the lane's columns; 0 in a row that is all -inf
  __device__ __forceinline__ void softmax(int e, int g, int l, float (&p)[J * W]) const {
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; j++) {
      const T *t = reinterpret_cast<const T *>(&x[j]);
#pragma unroll
      for (int i = 0; i < W; i++) {
        p[j * W + i] = (l + g * j) * W < e ? to_f32<T>(t[i]) : -INFINITY;
        m = fmaxf(m, p[j * W + i]);
      }
    }
    for (int o = g / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
    const float ref = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < J * W; j++) { p[j] = ex2_approx((p[j] - ref) * L_LOG2E); sum += p[j]; }
    for (int o = g / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < J * W; j++) p[j] *= inv;
  }
};

// Partial results of a CTA: column sums of p [e], counts [e] and the number of rows kept.
template <typename T, int W, int J>
__global__ void __launch_bounds__(R_THREADS)
router_part_kernel(const T *__restrict__ r, const uint8_t *__restrict__ keep, const int32_t *__restrict__ is, int64_t n, int e, int k, int g,
                   float *__restrict__ psum, int *__restrict__ pcount, int *__restrict__ ticket) {
  extern __shared__ float rsh[];                     // [8][g * J * W] column sums of the warps, then [e + 1] counts
  const int span = g * J * W;
  int *cnt = reinterpret_cast<int *>(rsh + (R_THREADS / 32) * span);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (g - 1), sub = lane / g, per_warp = 32 / g;
  for (int c = threadIdx.x; c <= e; c += R_THREADS) cnt[c] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;              // of the next kernel
  __syncthreads();
  float acc[J * W];
#pragma unroll
  for (int j = 0; j < J * W; j++) acc[j] = 0.f;
  const int64_t step = (int64_t)gridDim.x * (R_THREADS / 32) * per_warp;
  int64_t i = ((int64_t)blockIdx.x * (R_THREADS / 32) + warp) * per_warp + sub;
  int kept = 0;
  RouterRow<T, W, J> next;
  bool use = i < n && keep[i] != 0;
  if (use) next.load(r + i * e, e, g, l);
  for (; i - sub < n; i += step) {                   // uniform over the warp: every lane takes part in the shuffles
    const RouterRow<T, W, J> row = next;
    const bool mine = use;
    use = i + step < n && keep[i + step] != 0;
    if (use) next.load(r + (i + step) * e, e, g, l);
    float p[J * W];
    row.softmax(e, g, l, p);
    if (mine) {
#pragma unroll
      for (int j = 0; j < J * W; j++) acc[j] += p[j];
      if (l == 0) kept++;
    }
  }
#pragma unroll
  for (int j = 0; j < J * W; j++)
    for (int o = g; o < 32; o <<= 1) acc[j] += __shfl_xor_sync(kFull, acc[j], o);
  if (lane < g)
#pragma unroll
    for (int j = 0; j < J; j++)
#pragma unroll
      for (int x = 0; x < W; x++) rsh[warp * span + (lane + g * j) * W + x] = acc[j * W + x];
  kept = warp_sum(kept);
  if (lane == 0 && kept) atomicAdd(&cnt[e], kept);
  for (int64_t o = (int64_t)blockIdx.x * R_THREADS + threadIdx.x; o < n * k; o += (int64_t)gridDim.x * R_THREADS) {
    const int c = is[o];
    if (c >= 0 && c < e && keep[(uint32_t)o / (uint32_t)k] != 0) atomicAdd(&cnt[c], 1);      // n k is below 2^31
  }
  __syncthreads();
  for (int c = threadIdx.x; c < e; c += R_THREADS) {
    float t = 0.f;
    for (int w = 0; w < R_THREADS / 32; w++) t += rsh[w * span + c];
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
  if (c < e) {
#pragma unroll 8
    for (int b = warp; b < parts; b += 32) p += (double)psum[(int64_t)b * e + c];
  }
  if (c <= e) {
#pragma unroll 8
    for (int b = warp; b < parts; b += 32) q += pcount[(int64_t)b * (e + 1) + c];
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
template <typename T, int W, int J>
__global__ void __launch_bounds__(R_THREADS)
router_grad_kernel(const T *__restrict__ r, const uint8_t *__restrict__ keep, const int32_t *__restrict__ counts, const float *__restrict__ norm,
                   const float *__restrict__ dl, int64_t n, int e, int g, T *__restrict__ dr) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (g - 1), sub = lane / g, per_warp = 32 / g;
  const int64_t step = (int64_t)gridDim.x * (R_THREADS / 32) * per_warp;
  int64_t i = ((int64_t)blockIdx.x * (R_THREADS / 32) + warp) * per_warp + sub;
  RouterRow<T, W, J> next;
  bool use = i < n && keep[i] != 0;
  if (use) next.load(r + i * e, e, g, l);
  long long all = 0;
  for (int x = lane; x < e; x += 32) all += counts[x];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(kFull, all, o);
  const int mean = (int)(all / e);
  float cf[J * W];
#pragma unroll
  for (int j = 0; j < J; j++)
#pragma unroll
    for (int x = 0; x < W; x++) cf[j * W + x] = (l + g * j) * W < e ? (float)(counts[(l + g * j) * W + x] - mean) : 0.f;
  const float f = (float)((double)*norm * (double)*dl);
  for (; i - sub < n; i += step) {
    const RouterRow<T, W, J> row = next;
    const bool mine = use;
    use = i + step < n && keep[i + step] != 0;
    if (use) next.load(r + (i + step) * e, e, g, l);
    float p[J * W];
    row.softmax(e, g, l, p);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < J * W; j++) dot = fmaf(p[j], cf[j], dot);
    for (int o = g / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
    if (i < n) {
#pragma unroll
      for (int j = 0; j < J; j++)
        if ((l + g * j) * W < e) {
          typename RouterGroup<T, W>::type y;
          T *t = reinterpret_cast<T *>(&y);
#pragma unroll
          for (int x = 0; x < W; x++) t[x] = from_f32<T>(mine ? p[j * W + x] * (cf[j * W + x] - dot) * f : 0.f);
          *reinterpret_cast<typename RouterGroup<T, W>::type *>(dr + i * e + (l + g * j) * W) = y;
        }
    }
  }
}

static int64_t router_grid(int64_t n, const RouterShape &s, int num_sms) {
  const int64_t rows = (int64_t)(R_THREADS / 32) * (32 / s.g);
  const int64_t want = (n + rows - 1) / rows, most = (int64_t)num_sms * 4;
  return want < 1 ? 1 : want < most ? want : most;
}

size_t router_workspace_bytes(const void *r, int elem, int64_t n, int64_t e, int num_sms) {
  const int64_t grid = router_grid(n, router_shape(r, e, elem), num_sms);
  return up256((size_t)(grid * e) * 4) + up256((size_t)(grid * (e + 1)) * 4) + up256((size_t)e * 8) + 256;
}

// F is instantiated for the row's shape: W = 4 has up to 8 groups per lane, W = 1 up to 32
#define FB_ROUTER_SHAPE(S, F)                                                                       \
  switch ((S).w * 100 + (S).j) {                                                                    \
    case 101: F(1, 1); break; case 102: F(1, 2); break; case 104: F(1, 4); break; case 108: F(1, 8); break; \
    case 116: F(1, 16); break; case 132: F(1, 32); break;                                           \
    case 401: F(4, 1); break; case 402: F(4, 2); break; case 404: F(4, 4); break; default: F(4, 8); break;  \
  }

template <typename T>
static cudaError_t router(void *workspace, const T *r, const uint8_t *keep, const int32_t *is, int64_t n, int64_t e, int64_t k, float *loss,
                          int32_t *counts, float *norm, int num_sms, cudaStream_t stream) {
  const RouterShape s = router_shape(r, e, sizeof(T));
  const int grid = (int)router_grid(n, s, num_sms);
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  float *psum = reinterpret_cast<float *>(ws);
  int *pcount = reinterpret_cast<int *>(ws + up256((size_t)grid * e * 4));
  double *sums = reinterpret_cast<double *>(reinterpret_cast<uint8_t *>(pcount) + up256((size_t)grid * (e + 1) * 4));
  int *kept = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(sums) + up256((size_t)e * 8));
  int *ticket = kept + 1;
  const size_t smem = (size_t)(R_THREADS / 32) * s.g * s.j * s.w * 4 + (size_t)(e + 1) * 4;
#define FB_PART(W, J) router_part_kernel<T, W, J><<<grid, R_THREADS, smem, stream>>>(r, keep, is, n, (int)e, (int)k, s.g, psum, pcount, ticket)
  FB_ROUTER_SHAPE(s, FB_PART)
#undef FB_PART
  const cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  router_loss_kernel<<<(unsigned)((e + 1 + 31) / 32), 1024, 0, stream>>>(psum, pcount, grid, (int)e, sums, kept, ticket, counts, loss, norm);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t router_grad(const T *r, const uint8_t *keep, const int32_t *counts, const float *norm, const float *dl, int64_t n, int64_t e, T *dr,
                               int num_sms, cudaStream_t stream) {
  if (n <= 0 || e <= 0) return cudaSuccess;
  const RouterShape s = router_shape(r, e, sizeof(T));               // the result starts on a 256-byte boundary
  const int grid = (int)router_grid(n, s, num_sms);
#define FB_GRAD(W, J) router_grad_kernel<T, W, J><<<grid, R_THREADS, 0, stream>>>(r, keep, counts, norm, dl, n, (int)e, s.g, dr)
  FB_ROUTER_SHAPE(s, FB_GRAD)
#undef FB_GRAD
  return cudaGetLastError();
}

cudaError_t launch_router_balance(void *workspace, int elem, const void *r, const uint8_t *keep, const int32_t *is, int64_t n, int64_t e, int64_t k,
                                  float *loss, int32_t *counts, float *norm, int num_sms, cudaStream_t stream) {
  if (elem == 2) return router<__half>(workspace, reinterpret_cast<const __half *>(r), keep, is, n, e, k, loss, counts, norm, num_sms, stream);
  return router<float>(workspace, reinterpret_cast<const float *>(r), keep, is, n, e, k, loss, counts, norm, num_sms, stream);
}

cudaError_t launch_router_balance_grad(int elem, const void *r, const uint8_t *keep, const int32_t *counts, const float *norm, const float *dl, int64_t n,
                                       int64_t e, void *dr, int num_sms, cudaStream_t stream) {
  if (elem == 2) return router_grad<__half>(reinterpret_cast<const __half *>(r), keep, counts, norm, dl, n, e, reinterpret_cast<__half *>(dr), num_sms, stream);
  return router_grad<float>(reinterpret_cast<const float *>(r), keep, counts, norm, dl, n, e, reinterpret_cast<float *>(dr), num_sms, stream);
}

}  // namespace fb
