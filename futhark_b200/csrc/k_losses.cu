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
// All four are bound by memory: each direction reads its logits once and the gradients are written once.  One at a time, 4096 x 131072
// binary16: distill_part 171 us (6.3 TB/s), distill_grad 346 us (6.2 TB/s), and 12 and 8 us for losses and teachers; 2049 x 50001 f32: 64 us (6.4),
// 125 us (6.6), 6 and 6 us; 131072 x 256 f32: router_part 25 us (5.3 TB/s), router_loss 10 us, router_grad 38 us (7.0 TB/s, some of the writes
// still in L2).
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "kernels.h"

namespace fb {

constexpr float L_LOG2E = 1.4426950408889634f;
constexpr double L_LN2 = 0.69314718055994530942;

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// ---- distillation -----------------------------------------------------------------------------------------
// A row is read in aligned 16-byte groups; what of the first and last group lies outside the row is not read.  It is cut
// into chunks of 32 x 4 groups, and those into runs that a warp works off one after the other: a lane has up to 4 groups
// in registers and the 4 of its next chunk (of whatever row) in flight.  Nothing is shared between warps, so rows of any
// length and start keep every SM busy, a single one included; lanes meet only at the end of a run, since with one chunk per
// meeting the steps around a chunk's elements took as many instructions as the elements (10.7 per element in all, issue-bound).
constexpr int D_THREADS = 256, D_WARPS = D_THREADS / 32, D_PER = 4, D_CTAS = 4;
struct DistillShape {
  int chunks, groups;                // chunks of a row, groups of a chunk
  int run, runs;                     // chunks of a run, runs of a row
};
static DistillShape distill_shape(const void *s, int64_t n, int64_t v, int elem, int num_sms, int longest) {
  const int64_t w = 16 / elem, slack = ((uintptr_t)s & 15) == 0 && v % w == 0 ? 0 : 1;      // rows may start inside a group
  const int64_t groups = (v + w - 1) / w + slack, most = 32 * D_PER;
  DistillShape d;
  d.chunks = groups <= most ? 1 : (int)((groups + most - 1) / most);
  d.groups = (int)(groups < most ? groups : most);
  // as long as there are four runs for every warp that is resident
  const int64_t warps = (int64_t)num_sms * D_CTAS * D_WARPS;
  d.run = 1;
  while (d.run < longest && d.run < d.chunks && n * ((d.chunks + 2 * d.run - 1) / (2 * d.run)) >= 4 * warps) d.run *= 2;
  d.runs = (d.chunks + d.run - 1) / d.run;
  return d;
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
  if (r.whole(group)) return ld_chain_v4(r.base + c);
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

// Its largest element; NaN does not count here, it is seen in the sum.
__device__ __forceinline__ float group_max(const int4 &b, const float *) {
  return fmaxf(fmaxf(__int_as_float(b.x), __int_as_float(b.y)), fmaxf(__int_as_float(b.z), __int_as_float(b.w)));
}
__device__ __forceinline__ float group_max(const int4 &b, const __half *) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&b);
  const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Maxima are kept in units in which what was subtracted from the logits is known exactly.  SCALED: log 2, the unit of the
// exponents: x scale - m in one step, whose rounding of m (|m| 2^-24) goes into the sum as a power of two and out again with m.  Otherwise the
// logit's own, (x - m) scale.  That is how f32 does it, since a logit of the type's lowest value (a mask) times the scale would be no
// finite number, and binary16 below the temperature of D_FAR, since there the rounding of m would leave the exponents' range.
template <bool SCALED> struct LogitUnit {
  static __device__ __forceinline__ float of(float x, float scale) { return SCALED ? x * scale : x; }             // of a logit
  static __device__ __forceinline__ float log2(float d, float scale) { return SCALED ? d : d * scale; }           // of a difference
};
// (maximum, sum): the fold of two
template <bool SCALED>
__device__ __forceinline__ void fold_pair(float &m, float &s, float om, float os, float scale) {
  const float mn = fmaxf(m, om), ref = mn == -INFINITY ? 0.f : mn;
  s = s * exp2f(LogitUnit<SCALED>::log2(m - ref, scale)) + os * exp2f(LogitUnit<SCALED>::log2(om - ref, scale));
  m = mn;
}
// of a row's runs, by a warp, eight per lane in flight
template <bool SCALED>
__device__ __forceinline__ void fold_runs(const float2 *part, int runs, float scale, int lane, float &m, float &sum) {
  m = -INFINITY;
  sum = 0.f;
  for (int p0 = lane; p0 < runs; p0 += 256) {
    float2 q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = p0 + 32 * j < runs ? __ldcg(part + p0 + 32 * j) : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int j = 0; j < 8; j++) fold_pair<SCALED>(m, sum, q[j].x, q[j].y, scale);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float pm = __shfl_xor_sync(kFull, m, o), ps = __shfl_xor_sync(kFull, sum, o);
    fold_pair<SCALED>(m, sum, pm, ps, scale);
  }
}

// Where a warp is: run `item` of all rows, at one of its chunks.
struct DistillAt {
  int64_t item, row;
  int chunk, last;                                   // the chunk, and the one behind the run's last
  __device__ __forceinline__ void start(int64_t items, const DistillShape &d, bool small) {
    if (item >= items) return;
    row = small ? (int64_t)((uint32_t)item / (uint32_t)d.runs) : item / d.runs;
    chunk = (int)(item - row * d.runs) * d.run;
    last = min(chunk + d.run, d.chunks);
  }
  __device__ __forceinline__ void next(int64_t items, int64_t step, const DistillShape &d, bool small) {
    if (++chunk == last) { item += step; start(items, d, small); }
  }
};
// The lane's groups of a chunk.  Away from the ends of the row every group is whole.
template <typename T>
__device__ __forceinline__ void load_chunk(const DistillRow<T> &r, int chunk, int groups, int lane, int4 (&x)[D_PER]) {
  const int g0 = chunk * groups;
  if (r.first(g0) >= 0 && groups == 32 * D_PER && r.first(g0 + groups) <= r.v) {
    const T *p = r.base + r.first(g0 + lane);
#pragma unroll
    for (int i = 0; i < D_PER; i++) x[i] = ld_chain_v4(p + i * 32 * DistillRow<T>::W);
  } else {
#pragma unroll
    for (int i = 0; i < D_PER; i++)
      if (lane + 32 * i < groups) x[i] = load_group<T>(r, g0 + lane + 32 * i);
  }
}

// exponents of 2 of two logits, relative to the reference whose negative is nr
template <bool SCALED> __device__ __forceinline__ float2 exponents(float2 x, float2 scale, float2 nr) {
  return SCALED ? fma2(x, scale, nr) : mul2(add2(x, nr), scale);
}

__device__ __forceinline__ bool is_word(int32_t c, float t, int64_t v) { return c >= 0 && c < v && t != -INFINITY; }

// The teacher's softmax of a row over its words, by one warp in shared memory: its words (-1: padding), and log q or q.  The lanes
// read what they wrote themselves until the caller's __syncwarp.  False if the row has no word.
template <bool LOG>
__device__ __forceinline__ bool teacher_row(const int32_t *is, const float *t, int k, int64_t v, float inv_tau, int lane, int *wi, float *wq) {
  float m = -INFINITY;
#pragma unroll 4
  for (int j = lane; j < k; j += 32) {
    const int c = is[j];
    const float x = t[j];
    const bool in = is_word(c, x, v);
    wi[j] = in ? c : -1;
    wq[j] = x;
    if (in) m = fmaxf(m, x);
  }
  bool some = false;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
  float sum = 0.f;
  for (int j = lane; j < k; j += 32)
    if (wi[j] >= 0) {
      some = true;
      const float x = (wq[j] - m) * inv_tau, e = expf(x);
      wq[j] = LOG ? x : e;
      sum += e;
    }
  sum = warp_sum(sum);
  const float c = LOG ? logf(sum) : 1.f / sum;
  for (int j = lane; j < k; j += 32)
    if (wi[j] >= 0) wq[j] = LOG ? wq[j] - c : wq[j] * c;
  return __any_sync(kFull, some);
}

// The loss of a row by one warp, over the teacher's words (in f64: its terms cancel), after the fold of the row's runs.
struct DistillLoss {
  const int32_t *is;
  const float *t;
  int k;
  float tau;
  float *loss, *lse;
};
template <typename T, bool SCALED>
__device__ __forceinline__ void distill_row(const DistillLoss &a, const T *s, int64_t v, const float2 *part, int runs, float scale, int64_t row, int lane, int *wi,
                                            float *wq) {
  const int k = a.k;
  const bool some = teacher_row<true>(a.is + row * k, a.t + row * k, k, v, 1.f / a.tau, lane, wi, wq);
  float m, sum;
  fold_runs<SCALED>(part + row * runs, runs, scale, lane, m, sum);
  const double inv_tau = 1.0 / (double)a.tau, l = (double)m * (SCALED ? L_LN2 : inv_tau) + log((double)sum);
  double total = 0;
  if (some) {
#pragma unroll 4
    for (int j = lane; j < k; j += 32) {
      const int c = wi[j];
      const float lq = wq[j], q = c >= 0 ? expf(lq) : 0.f;
      // a teacher's weight of exactly 0 adds nothing, whatever the student says
      if (q != 0.f) total += (double)q * ((double)lq - (double)to_f32<T>(s[row * v + c]) * inv_tau + l);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(kFull, total, o);
  if (lane == 0) {
    a.lse[row] = (float)l;
    a.loss[row] = (float)((double)a.tau * (double)a.tau * total);
  }
}

// (maximum, sum) of every run.  JOIN: of few rows, whose losses the CTA that ends last then makes; `ticket` is 0 between launches.
template <typename T, bool SCALED, bool JOIN>
__global__ void __launch_bounds__(D_THREADS, D_CTAS)
distill_part_kernel(const T *s, int64_t n, int64_t v, const DistillShape d, float scale, float2 *part,
                    uint32_t *ticket, const DistillLoss a) {
  constexpr int W = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t items = n * d.runs, step = (int64_t)gridDim.x * D_WARPS;
  const bool small = items < (1ll << 31);
  DistillAt at;
  at.item = (int64_t)blockIdx.x * D_WARPS + (threadIdx.x >> 5);
  at.start(items, d, small);
  chain_wait();
  int4 next[D_PER];
  if (at.item < items) load_chunk<T>(DistillRow<T>(s, at.row, v), at.chunk, d.groups, lane, next);
  float m = -INFINITY, sum = 0.f;
  while (at.item < items) {
    int4 x[D_PER];
#pragma unroll
    for (int i = 0; i < D_PER; i++) x[i] = next[i];
    const DistillAt here = at;
    at.next(items, step, d, small);
    if (at.item < items) load_chunk<T>(DistillRow<T>(s, at.row, v), at.chunk, d.groups, lane, next);
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < D_PER; i++)
      if (lane + 32 * i < d.groups) mx = fmaxf(mx, group_max(x[i], (const T *)nullptr));
    mx = fmaxf(m, LogitUnit<SCALED>::of(mx, scale));
    const float ref = mx == -INFINITY ? 0.f : mx;
    const float2 sc = make_float2(scale, scale), nr = make_float2(-ref, -ref);
    float2 u = make_float2(sum * ex2(LogitUnit<SCALED>::log2(m - ref, scale)), 0.f), b = make_float2(0.f, 0.f);
    m = mx;
#pragma unroll
    for (int i = 0; i < D_PER; i++)
      if (lane + 32 * i < d.groups) {
        float f[W];
        unpack(x[i], f);
#pragma unroll
        for (int j = 0; j < W; j += 4) {
          const float2 e = exponents<SCALED>(make_float2(f[j], f[j + 1]), sc, nr), g = exponents<SCALED>(make_float2(f[j + 2], f[j + 3]), sc, nr);
          u = add2(u, make_float2(ex2(e.x), ex2(e.y)));
          b = add2(b, make_float2(ex2(g.x), ex2(g.y)));
        }
      }
    sum = (u.x + u.y) + (b.x + b.y);
    if (here.chunk + 1 == here.last) {               // the lanes meet
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(kFull, m, o), os = __shfl_xor_sync(kFull, sum, o);
        fold_pair<SCALED>(m, sum, om, os, scale);
      }
      if (lane == 0) part[here.item] = make_float2(m, sum);
      m = -INFINITY;
      sum = 0.f;
    }
  }
  if (JOIN) {
    extern __shared__ float sh[];                    // per warp: words [k], log q [k]
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      last = atomicAdd(ticket, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    int *wi = reinterpret_cast<int *>(sh) + (threadIdx.x >> 5) * 2 * a.k;
    for (int64_t row = threadIdx.x >> 5; row < n; row += D_WARPS)
      distill_row<T, SCALED>(a, s, v, part, d.runs, scale, row, lane, wi, reinterpret_cast<float *>(wi + a.k));
    if (threadIdx.x == 0) *ticket = 0;
  }
}

template <typename T, bool SCALED>
__global__ void __launch_bounds__(256)
distill_loss_kernel(const T *s, const float2 *part, int runs, int64_t n, int64_t v, float scale, const DistillLoss a) {
  extern __shared__ float sh[];                      // per warp: words [k], log q [k]
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  chain_wait();
  int *wi = reinterpret_cast<int *>(sh) + (threadIdx.x >> 5) * 2 * a.k;
  if (row < n) distill_row<T, SCALED>(a, s, v, part, runs, scale, row, threadIdx.x & 31, wi, reinterpret_cast<float *>(wi + a.k));
}

// What the gradient needs of a row's teacher, by one warp in shared memory: per word its weight; of places with the same word one has
// the sum of their weights and the others -1.  Which places those are is found without comparing all with all: in a round every
// place that has not met its word yet writes itself into the word's slot of a hash table, and who then finds a place with its
// own word there has met it (all places of a word do so in the same round, and in every slot someone does).  False if the row has no word.
struct DistillTeacher {
  const int32_t *is;
  const float *t;
  int k, table;                                      // slots of the hash table: a power of two, at least 2 k
  float tau;
  const float *dl, *lse;
  __host__ __device__ __forceinline__ int shared() const { return 3 * k + table; }       // 32-bit words a warp needs
};
__device__ __forceinline__ bool teacher_weights(const DistillTeacher &a, int64_t row, int64_t v, int lane, int *wi, float *wq) {
  const int k = a.k, table = a.table;
  int *met = wi + 2 * k, *slot = wi + 3 * k;         // the place met, and the table
  const bool some = teacher_row<false>(a.is + row * k, a.t + row * k, k, v, 1.f / a.tau, lane, wi, wq);
  for (int j = lane; j < k; j += 32) met[j] = wi[j] < 0 ? j : -1;
  uint32_t mul = 2654435761u;
  for (bool left = true; left; mul = mul * 1664525u + 1013904224u | 1u) {
    for (int j = lane; j < k; j += 32)
      if (met[j] < 0) slot[(((uint32_t)wi[j] * mul) >> 16) & (table - 1)] = j;
    __syncwarp();
    left = false;
    for (int j = lane; j < k; j += 32)
      if (met[j] < 0) {
        const int w = slot[(((uint32_t)wi[j] * mul) >> 16) & (table - 1)];
        if (wi[w] == wi[j]) met[j] = w; else left = true;
      }
    left = __any_sync(kFull, left);
    __syncwarp();
  }
  for (int j0 = 0; j0 < k; j0 += 32) {
    const int j = j0 + lane;
    for (;;) {                                       // one word that stands more than once, the whole warp
      const unsigned more = __ballot_sync(kFull, j < k && met[j] != j);
      if (more == 0) break;
      const int w = __shfl_sync(kFull, j < k ? met[j] : 0, __ffs(more) - 1);
      float q = 0.f;
      for (int o = lane; o < k; o += 32)
        if (met[o] == w && wi[o] >= 0) {
          q += wq[o];
          if (o != w) { wi[o] = -1; met[o] = o; }
        }
      q = warp_sum(q);
      if (lane == 0) wq[w] = q;
      __syncwarp();
    }
  }
  return some;
}
// Per row: dl tau, whether there is a word, and the reference of its exponents with the factor that makes it exact: for binary16
// exp(S / tau - lse) = 2^(S scale - hi) f, with hi + log f to more than 32 bits; for f32 lse itself, exp(S / tau - lse).
__device__ __forceinline__ float4 teacher_record(const DistillTeacher &a, int64_t row, bool some, bool wide) {
  const float lse = a.lse[row];
  const double shift = (double)lse * (1.0 / L_LN2);
  const float hi = (float)shift;
  return make_float4(a.dl[row] * a.tau, some ? 1.f : 0.f, wide ? lse : hi, wide ? 1.f : exp2f((float)((double)hi - shift)));
}
// Below D_FAR an lse in f32 says too little about the row: the record then has the maximum of the row's logits and 1 / the sum of
// exp((S - maximum) / tau), from runs that distill_part_kernel has worked off again.
struct DistillFar {
  const float2 *part;                                // or nullptr
  int runs;
  float scale;                                       // log2 e / tau
};
// Both for every row, one warp per row.
__global__ void __launch_bounds__(256)
distill_teacher_kernel(bool wide, const DistillTeacher a, const DistillFar far, int64_t n, int64_t v, int32_t *words, float *weights, float4 *rows) {
  extern __shared__ float sh[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + warp;
  chain_wait();
  if (row >= n) return;
  int *wi = reinterpret_cast<int *>(sh) + warp * a.shared();
  float *wq = reinterpret_cast<float *>(wi + a.k);
  const bool some = teacher_weights(a, row, v, lane, wi, wq);
  for (int j = lane; j < a.k; j += 32) {
    words[row * a.k + j] = wi[j];
    weights[row * a.k + j] = wq[j];
  }
  float4 record = teacher_record(a, row, some, wide);
  if (far.part != nullptr) {
    float m, sum;
    fold_runs<false>(far.part + row * far.runs, far.runs, far.scale, lane, m, sum);
    record.z = m;
    record.w = 1.f / sum;
  }
  if (lane == 0) rows[row] = record;
}

// The gradient is read and written by neighbouring warps at neighbouring places, which HBM likes better than long runs: with runs
// of 1, 2, 4 and 16 chunks 131.5, 138, 142 and 147 us (f32, 2049 x 50001) and 377, 352, 362 and 388 us (binary16, 4096 x 131072,
// where a chunk is twice the elements per instruction around them).
template <typename T> constexpr int D_GRAD_RUN = sizeof(T) == 2 ? 2 : 1;

// exponents of 2 of two logits less the row's reference, whose negative is nr: scale is log2 e / tau (binary16, or far) or 1 / tau (f32)
template <typename T, bool FAR> __device__ __forceinline__ float2 row_exponents(float2 x, float2 scale, float2 nr) {
  if (FAR) return exponents<false>(x, scale, nr);
  const float2 y = fma2(x, scale, nr);
  return sizeof(T) == 2 ? y : mul2(y, make_float2(L_LOG2E, L_LOG2E));
}

// Every chunk: the student's softmax; after a run the words of the teacher that lie in it once more.
// OWN: every warp has one run at most, and finds what it needs of its row's teacher for itself.
// FAR: the rows' records have their own maxima and sums.
template <typename T, bool OWN, bool FAR>
__global__ void __launch_bounds__(D_THREADS, D_CTAS)
distill_grad_kernel(const T *s, int64_t n, int64_t v, const DistillShape d, float scale, const DistillTeacher a,
                    const int32_t *words, const float *weights, const float4 *rows, T *ds) {
  extern __shared__ float sh[];
  constexpr int W = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 31;
  const int64_t items = n * d.runs, step = (int64_t)gridDim.x * D_WARPS;
  const bool small = items < (1ll << 31);
  DistillAt at;
  at.item = (int64_t)blockIdx.x * D_WARPS + (threadIdx.x >> 5);
  at.start(items, d, small);
  chain_wait();
  int4 next[D_PER];
  if (at.item < items) load_chunk<T>(DistillRow<T>(s, at.row, v), at.chunk, d.groups, lane, next);
  float4 rc = make_float4(0.f, 0.f, 0.f, 0.f);
  bool fresh = true;
  int *wi = reinterpret_cast<int *>(sh) + (threadIdx.x >> 5) * a.shared();
  float *wq = reinterpret_cast<float *>(wi + a.k);
  if (OWN && at.item < items) {
    rc = teacher_record(a, at.row, teacher_weights(a, at.row, v, lane, wi, wq), sizeof(T) == 4);
    __syncwarp();
  }
  while (at.item < items) {
    int4 x[D_PER];
#pragma unroll
    for (int i = 0; i < D_PER; i++) x[i] = next[i];
    const DistillAt here = at;
    if (!OWN && fresh) rc = rows[here.row];
    at.next(items, step, d, small);
    if (at.item < items) load_chunk<T>(DistillRow<T>(s, at.row, v), at.chunk, d.groups, lane, next);
    const DistillRow<T> r(s, here.row, v);
    T *out = ds + here.row * v;
    const bool some = rc.y != 0.f;                   // uniform over the warp
    const int g0 = here.chunk * d.groups;
    const float2 sc = make_float2(scale, scale), nr = make_float2(-rc.z, -rc.z);
    const float fc = rc.w * rc.x;
    const bool inner = r.first(g0) >= 0 && d.groups == 32 * D_PER && r.first(g0 + d.groups) <= r.v && ((uintptr_t)(out + r.first(g0)) & 15) == 0;
#pragma unroll
    for (int i = 0; i < D_PER; i++)
      if (lane + 32 * i < d.groups) {
        float y[W];
        unpack(x[i], y);
#pragma unroll
        for (int j = 0; j < W; j += 2) {
          const float2 e = row_exponents<T, FAR>(make_float2(y[j], y[j + 1]), sc, nr);
          y[j] = ex2(e.x) * fc;
          y[j + 1] = ex2(e.y) * fc;
        }
        if (!some) {
#pragma unroll
          for (int j = 0; j < W; j++) y[j] = 0.f;
        }
        const int col = r.first(g0 + lane + 32 * i);
        if (inner) {
          st_stream_v4(out + col, pack(y));
        } else {
#pragma unroll
          for (int j = 0; j < W; j++) if (col + j >= 0 && col + j < r.v) out[col + j] = from_f32<T>(y[j]);
        }
      }
    fresh = here.chunk + 1 == here.last;
    if (fresh) {
      __syncwarp();                                  // the words' places have been written
      if (some) {
        const int c0 = r.first((here.last - 1) / d.run * d.run * d.groups), c1 = r.first(here.last * d.groups);
        for (int j = lane; j < a.k; j += 32) {
          const int word = OWN ? wi[j] : words[here.row * a.k + j];
          if (word >= 0 && word >= c0 && word < c1) {
            const float xw = to_f32<T>(r.base[word]), p = ex2(row_exponents<T, FAR>(make_float2(xw, xw), sc, nr).x) * rc.w;
            out[word] = from_f32<T>((p - (OWN ? wq[j] : weights[here.row * a.k + j])) * rc.x);
          }
        }
      }
    }
  }
}

static inline size_t up256(size_t b) { return (b + 255) & ~(size_t)255; }
static unsigned chunk_grid(int64_t items, int num_sms) {
  const int64_t g = (items + D_WARPS - 1) / D_WARPS, most = (int64_t)num_sms * D_CTAS;
  return (unsigned)(g < most ? g : most);
}
// Warps of a CTA that has a row per warp: few rows are spread over more SMs.
static int row_warps(int64_t n, int num_sms) { return n >= (int64_t)num_sms * 8 ? 8 : 2; }

// Small calls, where a kernel less is 4 us on the GPU and 2 on the host: what the runs leave of a row is then done by the kernel that works them
// off.  Of the forward the last CTA makes the losses, at most two rows of 256 runs per warp; in the gradient, where a warp has a run at most, it
// finds the weights of its row's teacher itself, in what shared memory leaves each of four CTAs.  One row of 32000 f32 with 8 words of its
// teacher, both directions: 25 us instead of 28.5; 16 rows of 2000000 binary16, 1954 runs, would be 64 instead of 58.5.
constexpr int D_OWN_K = 256;
static bool own_loss(const DistillShape &d, int64_t n, int64_t k) { return n <= 2 * D_WARPS && d.runs <= 256 && k <= D_OWN_K; }
static bool own_teacher(const DistillShape &d, int64_t n, int64_t k, int num_sms) {
  return n * d.runs <= (int64_t)num_sms * D_CTAS * D_WARPS && k <= D_OWN_K;
}

// Temperatures below which logits over the temperature need more than the 24 bits of an f32: a logit of 65504 there is 2^22 or more, and
// neither the rounding of a scaled maximum (at most 0.4 above) nor that of the lse can be left aside.  The gradient then reads the logits
// once more for statistics of its own (2049 x 50001 f32: 210 us instead of 139).
constexpr float D_FAR = 0x1p-6f;
static bool distill_far(float tau) { return tau < D_FAR; }
constexpr int D_LONGEST = 16;                        // chunks of a run whose elements are only read

size_t distill_workspace_bytes(const void *s, float tau, int64_t n, int64_t v, int64_t k, int elem, bool grad, int num_sms) {
  const size_t part = up256((size_t)n * distill_shape(s, n, v, elem, num_sms, D_LONGEST).runs * sizeof(float2));
  if (!grad) return part;
  const DistillShape d = distill_shape(s, n, v, elem, num_sms, elem == 2 ? D_GRAD_RUN<__half> : D_GRAD_RUN<float>);
  if (!distill_far(tau) && own_teacher(d, n, k, num_sms)) return 0;
  return up256((size_t)(n * k) * 4) * 2 + up256((size_t)n * sizeof(float4)) + (distill_far(tau) ? part : 0);
}

template <typename T, bool SCALED>
static cudaError_t distill(void *workspace, uint32_t *ticket, const T *s, const int32_t *is, const float *t, float tau, int64_t n, int64_t v, int64_t k,
                           float *loss, float *lse, int num_sms, cudaStream_t stream) {
  if (n <= 0) return cudaSuccess;
  const DistillShape d = distill_shape(s, n, v, sizeof(T), num_sms, D_LONGEST);
  float2 *part = reinterpret_cast<float2 *>(workspace);
  const float scale = (float)(1.0 / (L_LN2 * (double)tau));
  const DistillLoss a = {is, t, (int)k, tau, loss, lse};
  const unsigned grid = chunk_grid(n * d.runs, num_sms);
  if (own_loss(d, n, k))
    return launch_after(distill_part_kernel<T, SCALED, true>, grid, D_THREADS, (size_t)D_WARPS * 2 * k * 4, stream, s, n, v, d, scale, part, ticket, a);
  cudaError_t err = launch_after(distill_part_kernel<T, SCALED, false>, grid, D_THREADS, 0, stream, s, n, v, d, scale, part, ticket, a);
  if (err != cudaSuccess) return err;
  const int rw = row_warps(n, num_sms);
  static unsigned long long allowed = 0;
  err = allow_smem(reinterpret_cast<const void *>(distill_loss_kernel<T, SCALED>), 8 * 2 * DISTILL_MAX_K * 4, allowed);
  if (err != cudaSuccess) return err;
  return launch_after(distill_loss_kernel<T, SCALED>, (unsigned)((n + rw - 1) / rw), 32 * rw, (size_t)rw * 2 * k * 4, stream, s, part, d.runs, n, v, scale, a);
}

template <typename T>
static cudaError_t distill_grad(void *workspace, const T *s, const int32_t *is, const float *t, float tau, const float *lse, const float *dl, int64_t n,
                                int64_t v, int64_t k, T *ds, int num_sms, cudaStream_t stream) {
  if (n <= 0 || v <= 0) return cudaSuccess;
  const DistillShape d = distill_shape(s, n, v, sizeof(T), num_sms, D_GRAD_RUN<T>);
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  int32_t *words = reinterpret_cast<int32_t *>(ws);
  float *weights = reinterpret_cast<float *>(ws + up256((size_t)(n * k) * 4));
  float4 *rows = reinterpret_cast<float4 *>(ws + 2 * up256((size_t)(n * k) * 4));
  const bool far = distill_far(tau);
  const float scale = (float)(1.0 / ((sizeof(T) == 2 || far ? L_LN2 : 1.0) * (double)tau));
  DistillTeacher a = {is, t, (int)k, 32, tau, dl, lse};
  while (a.table < 2 * k) a.table *= 2;
  const unsigned grid = chunk_grid(n * d.runs, num_sms);
  if (!far && own_teacher(d, n, k, num_sms))
    return launch_after(distill_grad_kernel<T, true, false>, grid, D_THREADS, (size_t)D_WARPS * a.shared() * 4, stream, s, n, v, d, scale, a, words, weights, rows,
                        ds);
  DistillFar f = {nullptr, 0, scale};
  if (far) {
    const DistillShape p = distill_shape(s, n, v, sizeof(T), num_sms, D_LONGEST);
    float2 *part = reinterpret_cast<float2 *>(reinterpret_cast<uint8_t *>(rows) + up256((size_t)n * sizeof(float4)));
    const cudaError_t err = launch_after(distill_part_kernel<T, false, false>, chunk_grid(n * p.runs, num_sms), D_THREADS, 0, stream, s, n, v, p, scale, part,
                                         nullptr, DistillLoss{});
    if (err != cudaSuccess) return err;
    f.part = part;
    f.runs = p.runs;
  }
  const int rw = row_warps(n, num_sms);
  static unsigned long long allowed = 0;
  cudaError_t err = allow_smem(reinterpret_cast<const void *>(distill_teacher_kernel), 8 * (3 * DISTILL_MAX_K + 2 * DISTILL_MAX_K) * 4, allowed);
  if (err != cudaSuccess) return err;
  err = launch_after(distill_teacher_kernel, (unsigned)((n + rw - 1) / rw), 32 * rw, (size_t)rw * a.shared() * 4, stream, sizeof(T) == 4, a, f, n, v, words,
                     weights, rows);
  if (err != cudaSuccess) return err;
  if (far) return launch_after(distill_grad_kernel<T, false, true>, grid, D_THREADS, 0, stream, s, n, v, d, scale, a, words, weights, rows, ds);
  return launch_after(distill_grad_kernel<T, false, false>, grid, D_THREADS, 0, stream, s, n, v, d, scale, a, words, weights, rows, ds);
}

cudaError_t launch_topk_distill(void *workspace, void *ticket, int elem, const void *s, const int32_t *is, const float *t, float tau, int64_t n, int64_t v,
                                int64_t k, float *loss, float *lse, int num_sms, cudaStream_t stream) {
  uint32_t *tk = reinterpret_cast<uint32_t *>(ticket);
  const __half *h = reinterpret_cast<const __half *>(s);
  if (elem == 2)
    return distill_far(tau) ? distill<__half, false>(workspace, tk, h, is, t, tau, n, v, k, loss, lse, num_sms, stream)
                            : distill<__half, true>(workspace, tk, h, is, t, tau, n, v, k, loss, lse, num_sms, stream);
  return distill<float, false>(workspace, tk, reinterpret_cast<const float *>(s), is, t, tau, n, v, k, loss, lse, num_sms, stream);
}
cudaError_t launch_topk_distill_grad(void *workspace, int elem, const void *s, const int32_t *is, const float *t, float tau, const float *lse,
                                     const float *dl, int64_t n, int64_t v, int64_t k, void *ds, int num_sms, cudaStream_t stream) {
  if (elem == 2)
    return distill_grad<__half>(workspace, reinterpret_cast<const __half *>(s), is, t, tau, lse, dl, n, v, k, reinterpret_cast<__half *>(ds), num_sms, stream);
  return distill_grad<float>(workspace, reinterpret_cast<const float *>(s), is, t, tau, lse, dl, n, v, k, reinterpret_cast<float *>(ds), num_sms, stream);
}

// ---- router balance ----------------------------------------------------------------------------------------
// A row belongs to G lanes of a warp (a power of two, at most 32), each of which has J groups of W consecutive columns
// (W = 4 where rows are made of whole aligned groups, 1 otherwise).  Sixteen columns per lane where there are as many: a warp
// per row of 100 columns spent 250 instructions on it, most of them on crossing lanes, and was bound by them.  The lanes
// keep their columns' sums in registers over all rows of the CTA, so that nothing but the row maxima and sums crosses
// lanes, and the column sums add in an order that does not depend on timing.  The next row is loaded before this one is worked on.
//
// One CTA per SM, so that there are few partial results to add up, of as many warps as leave a lane the registers for its
// row, the next one and the sums: with sixteen columns 16, 20, 24 and 32 warps took 83, 78, 86 and 95 us for both directions of 131072
// x 256 f32, and 80, 66, 61 and 65 us of 200000 x 100 binary16.
constexpr int router_warps(int cols, int elem) { return cols <= 8 ? 32 : cols <= 16 ? (elem == 4 ? 20 : 24) : 16; }
struct RouterShape {
  int w, g, j, elem;
  int cols() const { return w * j; }                 // columns of a lane
  int warps() const { return router_warps(cols(), elem); }
};
static RouterShape router_shape(const void *r, int64_t e, int elem) {
  RouterShape s = {e % 4 == 0 && ((uintptr_t)r & (4 * elem - 1)) == 0 ? 4 : 1, 1, 1, elem};
  while (s.g < 32 && s.g * 16 < e) s.g *= 2;
  while ((int64_t)s.g * s.w * s.j < e) s.j *= 2;
  return s;
}
// lanes of a row known at compile time unroll their exchanges
template <typename F>
__device__ __forceinline__ float over_lanes(float x, int g, F f) {
  if (g == 32) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(kFull, x, o));
  } else if (g == 16) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(kFull, x, o));
  } else if (g > 1) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1)
      if (o < g) x = f(x, __shfl_xor_sync(kFull, x, o));
  }
  return x;
}
__device__ __forceinline__ float lanes_max(float x, int g) { return over_lanes(x, g, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ float lanes_sum(float x, int g) { return over_lanes(x, g, [](float a, float b) { return a + b; }); }

template <typename T, int W> struct RouterGroup;
template <> struct RouterGroup<float, 4> { using type = float4; };
template <> struct RouterGroup<float, 1> { using type = float; };
template <> struct RouterGroup<__half, 4> { using type = uint2; };
template <> struct RouterGroup<__half, 1> { using type = __half; };

template <typename T, int W, int J> struct RouterRow {
  static constexpr int COLS = W * J, WARPS = router_warps(COLS, sizeof(T)), THREADS = 32 * WARPS;
  typename RouterGroup<T, W>::type x[J];
  // columns behind the last one are -inf and stay so: nothing is loaded over them
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < J; j++) {
      T *t = reinterpret_cast<T *>(&x[j]);
#pragma unroll
      for (int i = 0; i < W; i++) t[i] = from_f32<T>(-INFINITY);
    }
  }
  // `at` is the lane's first group of the row, the others `gap` columns apart; the lane has `left` columns' worth of them
  __device__ __forceinline__ void load(const T *at, int gap, int left) {
#pragma unroll
    for (int j = 0; j < J; j++)
      if (gap * j < left) x[j] = *reinterpret_cast<const typename RouterGroup<T, W>::type *>(at + gap * j);
  }
  __device__ __forceinline__ void unpack(float (&p)[COLS]) const {
#pragma unroll
    for (int j = 0; j < J; j++) {
      const T *t = reinterpret_cast<const T *>(&x[j]);
#pragma unroll
      for (int i = 0; i < W; i++) p[j * W + i] = to_f32<T>(t[i]);
    }
  }
};
// Logits to exp(logit - maximum), in place; returns the factor that makes them add up to 1 (0 in a row that is all -inf).
// The difference is taken first: a logit of the type's lowest value (a mask) times log2 e would be no finite number.
template <int COLS>
__device__ __forceinline__ float router_exp(float (&p)[COLS], int g) {
  float m = p[0];
#pragma unroll
  for (int j = 1; j < COLS; j++) m = fmaxf(m, p[j]);
  m = lanes_max(m, g);
  const float ref = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
  if (COLS % 2 == 0) {
    const float2 nr = make_float2(-ref, -ref), scale = make_float2(L_LOG2E, L_LOG2E);
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < COLS - 1; j += 2) {
      const float2 d = mul2(add2(make_float2(p[j], p[j + 1]), nr), scale);
      p[j] = ex2(d.x);
      p[j + 1] = ex2(d.y);
      s = add2(s, make_float2(p[j], p[j + 1]));
    }
    sum = s.x + s.y;
  } else {
#pragma unroll
    for (int j = 0; j < COLS; j++) { p[j] = ex2((p[j] - ref) * L_LOG2E); sum += p[j]; }
  }
  sum = lanes_sum(sum, g);
  return sum == 0.f ? 0.f : __fdividef(1.f, sum);       // at most 2 units in the last place off; sum is at most 1024
}

// Partial results that a thread of the last CTA adds up at most.  More are left to a kernel of their own: 148 of 256 experts took one SM
// 2.4 us longer than that kernel, and 148 of 1024 experts 37 us.  It costs small calls 2 us.
constexpr int R_JOIN = 4;
// Columns of the CTAs' partial results: the experts and the number of rows kept, in whole groups of 4.
static __host__ __device__ __forceinline__ int router_groups(int e) { return e / 4 + 1; }
// Slices of the CTAs that the last one adds up side by side.
static __host__ __device__ __forceinline__ int router_slices(int threads, int e) { const int s = threads / router_groups(e); return s < 16 ? s : 16; }

// Partial results of a CTA: column sums of p, counts and, behind them, the number of rows kept.  `ticket`, which is 0 between
// launches: where there are few partial results the CTA that ends last adds them all up, in f64 and in the order of the CTAs, and makes the loss.
template <typename T, int W, int J>
__global__ void __launch_bounds__(RouterRow<T, W, J>::THREADS)
router_part_kernel(const T *r, const uint8_t *keep, const int32_t *is, int64_t n, int e, int k, int g,
                   float *psum, int *pcount, uint32_t *ticket, int32_t *counts,
                   float *loss, float *norm) {
  constexpr int R_WARPS = RouterRow<T, W, J>::WARPS, R_THREADS = RouterRow<T, W, J>::THREADS;
  extern __shared__ __align__(16) float rsh[];       // [R_WARPS][g * J * W] column sums of the warps, then [e + 1] counts
  const int span = g * J * W;
  int *cnt = reinterpret_cast<int *>(rsh + R_WARPS * span);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (g - 1), sub = lane / g, per_warp = 32 / g;
  const int64_t step = (int64_t)gridDim.x * R_WARPS * per_warp;
  int64_t i = ((int64_t)blockIdx.x * R_WARPS + warp) * per_warp + sub;
  const int gap = g * W, left = e - l * W;
  const T *at = r + i * e + l * W;                   // the lane's part of row i, and of its experts
  const int32_t *ex = is + i * k + l;
  RouterRow<T, W, J> next;
  chain_wait();
  uint8_t use = 0;                                   // whether the row counts: loaded beside it, not before it
  int sent = -1;                                     // the lane's first expert of the row
  next.clear();
  if (i < n) {
    next.load(at, gap, left);
    use = keep[i];
    if (l < k) sent = *ex;
  }
  for (int c = threadIdx.x; c <= e; c += R_THREADS) cnt[c] = 0;
  __syncthreads();
  float acc[J * W];
#pragma unroll
  for (int j = 0; j < J * W; j++) acc[j] = 0.f;
  int kept = 0;
  for (; i - sub < n; i += step) {                   // uniform over the warp: every lane takes part in the shuffles
    float p[J * W];
    next.unpack(p);
    const bool mine = use != 0;
    const int to = sent;
    const int32_t *here = ex;
    use = 0;
    at += step * e;
    ex += step * k;
    if (i + step < n) {
      next.load(at, gap, left);
      use = keep[i + step];
      if (l < k) sent = *ex;
    }
    const float inv = router_exp(p, g);
    if (mine) {
      if (J * W % 2 == 0) {
#pragma unroll
        for (int j = 0; j < J * W - 1; j += 2) {
          const float2 a = fma2(make_float2(p[j], p[j + 1]), make_float2(inv, inv), make_float2(acc[j], acc[j + 1]));
          acc[j] = a.x;
          acc[j + 1] = a.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < J * W; j++) acc[j] = fmaf(p[j], inv, acc[j]);
      }
      if (l == 0) kept++;
      if (to >= 0 && to < e) atomicAdd(&cnt[to], 1);
      for (int j = g; j < k - l; j += g) {
        const int c = here[j];
        if (c >= 0 && c < e) atomicAdd(&cnt[c], 1);
      }
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
  __syncthreads();
  const int groups = router_groups(e), span4 = 4 * groups, parts = (int)gridDim.x;
  for (int c = threadIdx.x; c < span4; c += R_THREADS) {
    float t = 0.f;
    if (c < e) {
#pragma unroll
      for (int w = 0; w < R_WARPS; w++) t += rsh[w * span + c];
    }
    psum[(int64_t)blockIdx.x * span4 + c] = t;
    pcount[(int64_t)blockIdx.x * span4 + c] = c <= e ? cnt[c] : 0;
  }
  if (ticket == nullptr) return;
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  // a slice of the CTAs and a group of 4 columns per thread
  const int slices = router_slices(R_THREADS, e);
  double *dsum = reinterpret_cast<double *>(rsh);    // [slices][span4]
  int *dcnt = reinterpret_cast<int *>(dsum + slices * span4);
  if ((int)threadIdx.x < slices * groups) {
    const int sl = threadIdx.x / groups, c = 4 * (threadIdx.x - sl * groups);
    double p0 = 0, p1 = 0, p2 = 0, p3 = 0;
    int4 q = make_int4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < R_JOIN; j++) {
      const int b = sl + j * slices;
      if (b >= parts) break;
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(psum + (int64_t)b * span4 + c));
      const int4 y = __ldcg(reinterpret_cast<const int4 *>(pcount + (int64_t)b * span4 + c));
      p0 += (double)x.x; p1 += (double)x.y; p2 += (double)x.z; p3 += (double)x.w;
      q.x += y.x; q.y += y.y; q.z += y.z; q.w += y.w;
    }
    double *dp = dsum + sl * span4 + c;
    dp[0] = p0; dp[1] = p1; dp[2] = p2; dp[3] = p3;
    *reinterpret_cast<int4 *>(dcnt + sl * span4 + c) = q;
  }
  __syncthreads();
  __shared__ double stotal[32];
  __shared__ long long sall[32];
  __shared__ int skept;
  double total = 0;
  long long all = 0;
  for (int c = threadIdx.x; c <= e; c += R_THREADS) {
    double p = 0;
    int q = 0;
    for (int sl = 0; sl < slices; sl++) { p += dsum[sl * span4 + c]; q += dcnt[sl * span4 + c]; }
    if (c == e) { skept = q; break; }
    counts[c] = q;
    total += (double)q * p;
    all += q;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { total += __shfl_xor_sync(kFull, total, o); all += __shfl_xor_sync(kFull, all, o); }
  if (lane == 0) { stotal[warp] = total; sall[warp] = all; }
  __syncthreads();
  if (warp != 0) return;
  total = lane < R_WARPS ? stotal[lane] : 0;
  all = lane < R_WARPS ? sall[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) { total += __shfl_xor_sync(kFull, total, o); all += __shfl_xor_sync(kFull, all, o); }
  if (lane == 0) {
    const double m = (double)skept, f = all > 0 && m > 0 ? (double)e / ((double)all * m) : 0.0;
    *norm = (float)f;
    *loss = all > 0 ? (float)(total * f) : 0.f;
    *ticket = 0;
  }
}

// 32 columns per CTA, the partial results of the CTAs over the warps, in f64; the CTA that ends last makes the loss.
__global__ void __launch_bounds__(1024)
router_loss_kernel(const float *psum, const int *pcount, int parts, int e, double *sums, int *kept,
                   uint32_t *ticket, int32_t *counts, float *loss, float *norm) {
  __shared__ double sp[32][33];
  __shared__ int sc[32][33];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, span4 = 4 * router_groups(e);
  double p = 0;
  int q = 0;
  chain_wait();
  if (c <= e) {
#pragma unroll 5
    for (int b = warp; b < parts; b += 32) {
      q += pcount[(int64_t)b * span4 + c];
      p += (double)psum[(int64_t)b * span4 + c];
    }
  }
  sp[warp][lane] = p;
  sc[warp][lane] = q;
  __syncthreads();
  p = warp_sum(sp[lane][warp]);                      // the warp's column of the 32
  q = warp_sum(sc[lane][warp]);
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine <= e) {
    if (mine < e) { sums[mine] = p; counts[mine] = q; } else *kept = q;
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(ticket, 1u) == gridDim.x - 1;
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
    *ticket = 0;
  }
}

// Counts are taken around their mean (in integers): where they are nearly equal the gradient is what is left of a
// difference, and sum_f p_if = 1 makes the shift cancel.
template <typename T, int W, int J>
__global__ void __launch_bounds__(RouterRow<T, W, J>::THREADS)
router_grad_kernel(const T *r, const uint8_t *keep, const int32_t *counts, const float *norm,
                   const float *dl, int64_t n, int e, int g, T *dr) {
  constexpr int R_WARPS = RouterRow<T, W, J>::WARPS;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (g - 1), sub = lane / g, per_warp = 32 / g;
  const int64_t step = (int64_t)gridDim.x * R_WARPS * per_warp;
  int64_t i = ((int64_t)blockIdx.x * R_WARPS + warp) * per_warp + sub;
  const int gap = g * W, left = e - l * W;
  const T *at = r + i * e + l * W;
  T *out = dr + i * e + l * W;
  RouterRow<T, W, J> next;
  chain_wait();
  uint8_t use = 0;
  next.clear();
  if (i < n) { next.load(at, gap, left); use = keep[i]; }
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
    float p[J * W];
    next.unpack(p);
    const bool mine = use != 0;
    at += step * e;
    if (i + step < n) { next.load(at, gap, left); use = keep[i + step]; }
    const float inv = router_exp(p, g);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < J * W; j++) dot = fmaf(p[j], cf[j], dot);
    dot = lanes_sum(dot, g) * inv;
    const float s = inv * f;
    if (i < n) {
#pragma unroll
      for (int j = 0; j < J; j++)
        if (gap * j < left) {
          typename RouterGroup<T, W>::type y;
          T *t = reinterpret_cast<T *>(&y);
#pragma unroll
          for (int x = 0; x < W; x++) t[x] = from_f32<T>(mine ? p[j * W + x] * s * (cf[j * W + x] - dot) : 0.f);
          *reinterpret_cast<typename RouterGroup<T, W>::type *>(out + gap * j) = y;
        }
    }
    out += step * e;
  }
}

static int64_t router_grid(int64_t n, const RouterShape &s, int num_sms) {
  const int64_t rows = (int64_t)s.warps() * (32 / s.g);
  const int64_t want = (n + rows - 1) / rows, most = num_sms;
  return want < 1 ? 1 : want < most ? want : most;
}

size_t router_workspace_bytes(const void *r, int elem, int64_t n, int64_t e, int num_sms) {
  const int64_t grid = router_grid(n, router_shape(r, e, elem), num_sms);
  return 2 * up256((size_t)grid * 16 * router_groups((int)e)) + up256((size_t)e * 8) + 256;
}

// F is instantiated for the row's shape: W = 4 has up to 8 groups per lane, W = 1 up to 32
#define FB_ROUTER_SHAPE(S, F)                                                                       \
  switch ((S).w * 100 + (S).j) {                                                                    \
    case 101: F(1, 1); break; case 102: F(1, 2); break; case 104: F(1, 4); break; case 108: F(1, 8); break; \
    case 116: F(1, 16); break; case 132: F(1, 32); break;                                           \
    case 401: F(4, 1); break; case 402: F(4, 2); break; case 404: F(4, 4); break; default: F(4, 8); break;  \
  }

template <typename T>
static cudaError_t router(void *workspace, uint32_t *ticket, const T *r, const uint8_t *keep, const int32_t *is, int64_t n, int64_t e, int64_t k,
                          float *loss, int32_t *counts, float *norm, int num_sms, cudaStream_t stream) {
  const RouterShape s = router_shape(r, e, sizeof(T));
  const int grid = (int)router_grid(n, s, num_sms), threads = 32 * s.warps(), span4 = 4 * router_groups((int)e);
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  float *psum = reinterpret_cast<float *>(ws);
  int *pcount = reinterpret_cast<int *>(ws + up256((size_t)grid * span4 * 4));
  double *sums = reinterpret_cast<double *>(reinterpret_cast<uint8_t *>(pcount) + up256((size_t)grid * span4 * 4));
  int *kept = reinterpret_cast<int *>(reinterpret_cast<uint8_t *>(sums) + up256((size_t)e * 8));
  const bool join = grid <= R_JOIN * router_slices(threads, (int)e);
  const size_t rows = (size_t)s.warps() * s.g * s.cols() * 4 + (size_t)(e + 1) * 4, joined = join ? (size_t)router_slices(threads, (int)e) * span4 * 12 : 0;
  const size_t smem = rows > joined ? rows : joined;
  cudaError_t err = cudaSuccess;
#define FB_PART(W, J)                                                                                                     \
  {                                                                                                                       \
    static unsigned long long allowed = 0;                                                                                \
    err = allow_smem(reinterpret_cast<const void *>(router_part_kernel<T, W, J>), 160 << 10, allowed);                    \
    if (err == cudaSuccess)                                                                                               \
      err = launch_after(router_part_kernel<T, W, J>, grid, threads, smem, stream, r, keep, is, n, (int)e, (int)k, s.g, psum, pcount,   \
                         join ? ticket : nullptr, counts, loss, norm);                                                    \
  }
  FB_ROUTER_SHAPE(s, FB_PART)
#undef FB_PART
  if (err != cudaSuccess || join) return err;
  return launch_after(router_loss_kernel, (unsigned)((e + 1 + 31) / 32), 1024, 0, stream, psum, pcount, grid, (int)e, sums, kept, ticket, counts, loss, norm);
}

template <typename T>
static cudaError_t router_grad(const T *r, const uint8_t *keep, const int32_t *counts, const float *norm, const float *dl, int64_t n, int64_t e, T *dr,
                               int num_sms, cudaStream_t stream) {
  if (n <= 0 || e <= 0) return cudaSuccess;
  const RouterShape s = router_shape(r, e, sizeof(T));               // the result starts on a 256-byte boundary
  const int grid = (int)router_grid(n, s, num_sms);
#define FB_GRAD(W, J) return launch_after(router_grad_kernel<T, W, J>, grid, 32 * s.warps(), 0, stream, r, keep, counts, norm, dl, n, (int)e, s.g, dr)
  FB_ROUTER_SHAPE(s, FB_GRAD)
#undef FB_GRAD
  return cudaSuccess;
}

cudaError_t launch_router_balance(void *workspace, void *ticket, int elem, const void *r, const uint8_t *keep, const int32_t *is, int64_t n, int64_t e,
                                  int64_t k, float *loss, int32_t *counts, float *norm, int num_sms, cudaStream_t stream) {
  uint32_t *tk = reinterpret_cast<uint32_t *>(ticket);
  if (elem == 2) return router<__half>(workspace, tk, reinterpret_cast<const __half *>(r), keep, is, n, e, k, loss, counts, norm, num_sms, stream);
  return router<float>(workspace, tk, reinterpret_cast<const float *>(r), keep, is, n, e, k, loss, counts, norm, num_sms, stream);
}

cudaError_t launch_router_balance_grad(int elem, const void *r, const uint8_t *keep, const int32_t *counts, const float *norm, const float *dl, int64_t n,
                                       int64_t e, void *dr, int num_sms, cudaStream_t stream) {
  if (elem == 2) return router_grad<__half>(reinterpret_cast<const __half *>(r), keep, counts, norm, dl, n, e, reinterpret_cast<__half *>(dr), num_sms, stream);
  return router_grad<float>(reinterpret_cast<const float *>(r), keep, counts, norm, dl, n, e, reinterpret_cast<float *>(dr), num_sms, stream);
}

}  // namespace fb
