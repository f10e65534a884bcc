// Entry points of the training losses (k_vocab.cu, k_losses.cu): argument checks, results, workspaces from the context's
// pool (given back in stream order at the end of the call), launches on the context's stream, and the records
// they return.  They follow entries.cu in everything a caller sees.
#include <stdlib.h>

#include <string>

#include "common.cuh"
#include "kernels.h"
#include "runtime.h"

static std::string kv(const char *k, int64_t v) { return std::string("\"") + k + "\":" + std::to_string(v); }

template <typename T>
static inline T *dptr(const memblock_device &m) { return reinterpret_cast<T *>((uintptr_t)m.mem); }

static int refuse(futhark_context *ctx, const char *why) {
  fb_set_error(ctx, "%s", why);
  return 1;
}
static int bad_sizes(futhark_context *ctx) { return refuse(ctx, "Error: entry point arguments have invalid sizes.\n"); }
static int not_ready(futhark_context *ctx) { return refuse(ctx, "The context failed to initialise; no entry point can run."); }

// Blocks and objects of a call that go back to the pool unless the call succeeds (`keep`), and its workspace, which
// always does: later work of the stream may have it.
struct Call {
  futhark_context *ctx;
  int rc = FUTHARK_SUCCESS;
  memblock_device ws = {nullptr, 0, 0, nullptr};
  struct Made { void *obj; memblock_device *mem; };
  Made made[4];
  int count = 0;
  // A captured call would write, at every replay, blocks that the pool has meanwhile given to others.
  explicit Call(futhark_context *c) : ctx(c) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(c->stream, &st) != cudaSuccess || st != cudaStreamCaptureStatusNone)
      rc = refuse(c, "Error: entry points that allocate their results cannot be captured.\n");
  }

  template <typename ARR>
  ARR *array(std::initializer_list<int64_t> shape, size_t elem, const char *desc) {
    if (rc != FUTHARK_SUCCESS) return nullptr;
    ARR *arr = (ARR *)malloc(sizeof(ARR));
    if (arr == nullptr) { rc = 1; return nullptr; }
    int64_t n = 1;
    int i = 0;
    for (const int64_t s : shape) { arr->shape[i++] = s; n *= s; }
    rc = fb_alloc(ctx, (size_t)n * elem, desc, &arr->mem);
    if (rc != FUTHARK_SUCCESS) { free(arr); return nullptr; }
    made[count++] = {arr, &arr->mem};
    return arr;
  }
  template <typename REC>
  REC *record() {
    if (rc != FUTHARK_SUCCESS) return nullptr;
    REC *r = (REC *)malloc(sizeof(REC));
    if (r == nullptr) { rc = 1; return nullptr; }
    made[count++] = {r, nullptr};
    return r;
  }
  void *workspace(size_t bytes, const char *desc) {
    if (rc != FUTHARK_SUCCESS) return nullptr;
    rc = fb_alloc(ctx, bytes, desc, &ws);
    return dptr<void>(ws);
  }
  template <typename DETAILS, typename LAUNCH>
  void launch(const char *name, const char *prov, DETAILS details, LAUNCH f) {       // details are only made where someone reads them
    if (rc != FUTHARK_SUCCESS) return;
    LaunchScope ls(ctx, name, prov, ctx->logging || ctx->profiling ? details() : std::string());
    rc = fb_cuda_check(ctx, f(), name);
  }
  ~Call() {
    fb_unref(ctx, &ws);
    if (rc == FUTHARK_SUCCESS) return;
    for (int i = 0; i < count; i++) {
      if (made[i].mem != nullptr) fb_unref(ctx, made[i].mem);
      free(made[i].obj);
    }
  }
};

static bool aligned16(const memblock_device &m) { return (m.mem & 15) == 0; }
static bool fits(int64_t a) { return a < ((int64_t)1 << 31); }

typedef struct futhark_opaque_tup2_arr1d_f32_arr1d_f32 losses_t;
typedef struct futhark_opaque_tup2_arr2d_f16_arr2d_f16 grads_t;
typedef struct futhark_opaque_tup3_arr1d_f32_arr1d_i32_arr1d_f32 balance_t;

// ---- cross entropy over a vocabulary ------------------------------------------------------------------
// sizes that are 32-bit numbers in the kernels, tiles among them
static bool vocab_fits(int64_t n, int64_t v, int64_t d) { return fits(n) && fits(v) && fits(d + 8) && n / 256 * (v / 128) < ((int64_t)1 << 30); }
static std::string vocab_details(int64_t n, int64_t v, int64_t d, const std::string &more = "") {
  return "{" + kv("n", n) + "," + kv("v", v) + "," + kv("d", d) + more + "}";
}

extern "C" {

int futhark_entry_vocab_xent_f16(struct futhark_context *ctx, losses_t **out0, const struct futhark_f16_2d *in0, const struct futhark_f16_2d *in1,
                                 const struct futhark_i32_1d *in2) {
  if (!ctx->ready) return not_ready(ctx);
  CtxGuard g(ctx);
  const int64_t n = in0->shape[0], d = in0->shape[1], v = in1->shape[0];
  if (in1->shape[1] != d || in2->shape[0] != n) return bad_sizes(ctx);
  if (!vocab_fits(n, v, d)) return refuse(ctx, "Error: vocab_xent_f16: sizes must be below 2^31 and n v below 2^45.\n");
  Call call(ctx);
  auto *loss = call.array<futhark_f32_1d>({n}, 4, "vocab_xent_f16.loss"), *lse = call.array<futhark_f32_1d>({n}, 4, "vocab_xent_f16.lse");
  auto *rec = call.record<losses_t>();
  const fb::VocabPlan plan = fb::vocab_plan(n, v, d, aligned16(in0->mem), aligned16(in1->mem), false, ctx->num_sms);
  void *ws = call.workspace(plan.bytes, "vocab_xent_f16.workspace");
  call.launch("vocab_xent_f16.segred", "map2 (\\x t -> log (sum (map exp (map (dot x) W))) - dot x W[t]) X ts", [&] { return vocab_details(n, v, d); }, [&] {
    ctx->failure_is_an_option = true;
    return fb::launch_vocab_xent(plan, ws, ctx->reduce_scratch, dptr<uint16_t>(in0->mem), dptr<uint16_t>(in1->mem), dptr<int32_t>(in2->mem), dptr<float>(loss->mem),
                                 dptr<float>(lse->mem), n, v, d, ctx->d_failure, ctx->num_sms, ctx->stream);
  });
  if (call.rc != FUTHARK_SUCCESS) return call.rc;
  rec->v0 = loss; rec->v1 = lse;
  *out0 = rec;
  return FUTHARK_SUCCESS;
}

int futhark_entry_vocab_xent_grad_f16(struct futhark_context *ctx, grads_t **out0, const struct futhark_f16_2d *in0, const struct futhark_f16_2d *in1,
                                      const struct futhark_i32_1d *in2, const struct futhark_f32_1d *in3, const struct futhark_f32_1d *in4,
                                      const struct futhark_f32_1d *in5) {
  if (!ctx->ready) return not_ready(ctx);
  CtxGuard g(ctx);
  const int64_t n = in0->shape[0], d = in0->shape[1], v = in1->shape[0];
  if (in1->shape[1] != d || in2->shape[0] != n || in3->shape[0] != n || in4->shape[0] != n || in5->shape[0] != n) return bad_sizes(ctx);
  if (!vocab_fits(n, v, d)) return refuse(ctx, "Error: vocab_xent_grad_f16: sizes must be below 2^31 and n v below 2^45.\n");
  Call call(ctx);
  auto *dx = call.array<futhark_f16_2d>({n, d}, 2, "vocab_xent_grad_f16.dx"), *dw = call.array<futhark_f16_2d>({v, d}, 2, "vocab_xent_grad_f16.dw");
  auto *rec = call.record<grads_t>();
  const fb::VocabPlan plan = fb::vocab_plan(n, v, d, aligned16(in0->mem), aligned16(in1->mem), true, ctx->num_sms);
  void *ws = call.workspace(plan.bytes, "vocab_xent_grad_f16.workspace");
  call.launch("vocab_xent_grad_f16.segmap_segred", "vjp of vocab_xent_f16", [&] { return vocab_details(n, v, d, "," + kv("pieces", plan.pieces) + "," + kv("parts", plan.splits)); }, [&] {
    ctx->failure_is_an_option = true;
    return fb::launch_vocab_xent_grad(plan, ws, dptr<uint16_t>(in0->mem), dptr<uint16_t>(in1->mem), dptr<int32_t>(in2->mem), dptr<float>(in3->mem),
                                      dptr<float>(in4->mem), dptr<float>(in5->mem), dptr<uint16_t>(dx->mem), dptr<uint16_t>(dw->mem), n, v, d,
                                      ctx->d_failure, ctx->num_sms, ctx->stream);
  });
  if (call.rc != FUTHARK_SUCCESS) return call.rc;
  rec->v0 = dx; rec->v1 = dw;
  *out0 = rec;
  return FUTHARK_SUCCESS;
}

}  // extern "C"

// ---- distillation ------------------------------------------------------------------------------------------
static int distill_refusal(futhark_context *ctx, float tau, int64_t n, int64_t v, int64_t k) {
  if (!(tau >= 0x1p-60f && tau <= 0x1p60f)) return refuse(ctx, "Error: topk_distill: the temperature must be in [2^-60, 2^60].\n");
  if (k > fb::DISTILL_MAX_K) return refuse(ctx, "Error: topk_distill: at most 1024 logits per row.\n");
  if (!fits(n) || !fits(v + 16384)) return refuse(ctx, "Error: topk_distill: sizes must be below 2^31 - 2^14.\n");
  return 0;
}
static std::string distill_details(int64_t n, int64_t v, int64_t k) { return "{" + kv("n", n) + "," + kv("v", v) + "," + kv("k", k) + "}"; }

template <typename MAT>
static int topk_distill(futhark_context *ctx, const char *name, int elem, losses_t **out0, float tau, const MAT *s, const futhark_i32_2d *is,
                        const futhark_f32_2d *t) {
  if (!ctx->ready) return not_ready(ctx);
  CtxGuard g(ctx);
  const int64_t n = s->shape[0], v = s->shape[1], k = is->shape[1];
  if (is->shape[0] != n || t->shape[0] != n || t->shape[1] != k) return bad_sizes(ctx);
  if (distill_refusal(ctx, tau, n, v, k)) return 1;
  Call call(ctx);
  auto *loss = call.array<futhark_f32_1d>({n}, 4, "topk_distill.loss"), *lse = call.array<futhark_f32_1d>({n}, 4, "topk_distill.lse");
  auto *rec = call.record<losses_t>();
  void *ws = call.workspace(fb::distill_workspace_bytes(dptr<void>(s->mem), tau, n, v, k, elem, false, ctx->num_sms), "topk_distill.workspace");
  call.launch(name, "map3 (\\s is t -> tau**2 * sum (map2 (\\q i -> q * (log q - s[i]/tau + lse s)) (softmax t) is)) S iss T", [&] { return distill_details(n, v, k); }, [&] {
    return fb::launch_topk_distill(ws, ctx->reduce_scratch, elem, dptr<void>(s->mem), dptr<int32_t>(is->mem), dptr<float>(t->mem), tau, n, v, k, dptr<float>(loss->mem),
                                   dptr<float>(lse->mem), ctx->num_sms, ctx->stream);
  });
  if (call.rc != FUTHARK_SUCCESS) return call.rc;
  rec->v0 = loss; rec->v1 = lse;
  *out0 = rec;
  return FUTHARK_SUCCESS;
}

template <typename MAT>
static int topk_distill_grad(futhark_context *ctx, const char *name, int elem, MAT **out0, float tau, const MAT *s, const futhark_i32_2d *is,
                             const futhark_f32_2d *t, const futhark_f32_1d *lse, const futhark_f32_1d *dl) {
  if (!ctx->ready) return not_ready(ctx);
  CtxGuard g(ctx);
  const int64_t n = s->shape[0], v = s->shape[1], k = is->shape[1];
  if (is->shape[0] != n || t->shape[0] != n || t->shape[1] != k || lse->shape[0] != n || dl->shape[0] != n) return bad_sizes(ctx);
  if (distill_refusal(ctx, tau, n, v, k)) return 1;
  Call call(ctx);
  auto *ds = call.array<MAT>({n, v}, elem, "topk_distill_grad.ds");
  void *ws = call.workspace(fb::distill_workspace_bytes(dptr<void>(s->mem), tau, n, v, k, elem, true, ctx->num_sms), "topk_distill_grad.workspace");
  call.launch(name, "vjp of topk_distill", [&] { return distill_details(n, v, k); }, [&] {
    return fb::launch_topk_distill_grad(ws, elem, dptr<void>(s->mem), dptr<int32_t>(is->mem), dptr<float>(t->mem), tau, dptr<float>(lse->mem),
                                        dptr<float>(dl->mem), n, v, k, dptr<void>(ds->mem), ctx->num_sms, ctx->stream);
  });
  if (call.rc != FUTHARK_SUCCESS) return call.rc;
  *out0 = ds;
  return FUTHARK_SUCCESS;
}

extern "C" {

int futhark_entry_topk_distill_f32(struct futhark_context *ctx, losses_t **out0, const float in0, const struct futhark_f32_2d *in1,
                                   const struct futhark_i32_2d *in2, const struct futhark_f32_2d *in3) {
  return topk_distill(ctx, "topk_distill_f32.segred", 4, out0, in0, in1, in2, in3);
}
int futhark_entry_topk_distill_f16(struct futhark_context *ctx, losses_t **out0, const float in0, const struct futhark_f16_2d *in1,
                                   const struct futhark_i32_2d *in2, const struct futhark_f32_2d *in3) {
  return topk_distill(ctx, "topk_distill_f16.segred", 2, out0, in0, in1, in2, in3);
}
int futhark_entry_topk_distill_grad_f32(struct futhark_context *ctx, struct futhark_f32_2d **out0, const float in0, const struct futhark_f32_2d *in1,
                                        const struct futhark_i32_2d *in2, const struct futhark_f32_2d *in3, const struct futhark_f32_1d *in4,
                                        const struct futhark_f32_1d *in5) {
  return topk_distill_grad(ctx, "topk_distill_grad_f32.segmap", 4, out0, in0, in1, in2, in3, in4, in5);
}
int futhark_entry_topk_distill_grad_f16(struct futhark_context *ctx, struct futhark_f16_2d **out0, const float in0, const struct futhark_f16_2d *in1,
                                        const struct futhark_i32_2d *in2, const struct futhark_f32_2d *in3, const struct futhark_f32_1d *in4,
                                        const struct futhark_f32_1d *in5) {
  return topk_distill_grad(ctx, "topk_distill_grad_f16.segmap", 2, out0, in0, in1, in2, in3, in4, in5);
}

}  // extern "C"

// ---- router balance ----------------------------------------------------------------------------------------
template <typename MAT>
static int router_balance(futhark_context *ctx, const char *name, int elem, balance_t **out0, const MAT *r, const futhark_bool_1d *keep,
                          const futhark_i32_2d *is) {
  if (!ctx->ready) return not_ready(ctx);
  CtxGuard g(ctx);
  const int64_t n = r->shape[0], e = r->shape[1], k = is->shape[1];
  if (keep->shape[0] != n || is->shape[0] != n) return bad_sizes(ctx);
  if (e > fb::ROUTER_MAX_E) return refuse(ctx, "Error: router_balance: at most 1024 experts.\n");
  if (!fits(n) || !fits(k) || !fits(n * k)) return refuse(ctx, "Error: router_balance: the number of assignments must be below 2^31.\n");
  Call call(ctx);
  auto *loss = call.array<futhark_f32_1d>({1}, 4, "router_balance.loss");
  auto *counts = call.array<futhark_i32_1d>({e}, 4, "router_balance.counts");
  auto *norm = call.array<futhark_f32_1d>({1}, 4, "router_balance.norm");
  auto *rec = call.record<balance_t>();
  void *ws = call.workspace(fb::router_workspace_bytes(dptr<void>(r->mem), elem, n, e, ctx->num_sms), "router_balance.workspace");
  call.launch(name, "(norm * sum (map2 (*) counts (reduce (map2 (+)) (map softmax R))), hist (+) 0 e is, norm)",
              [&] { return "{" + kv("n", n) + "," + kv("e", e) + "," + kv("k", k) + "}"; }, [&] {
    return fb::launch_router_balance(ws, ctx->reduce_scratch, elem, dptr<void>(r->mem), dptr<uint8_t>(keep->mem), dptr<int32_t>(is->mem), n, e, k, dptr<float>(loss->mem),
                                     dptr<int32_t>(counts->mem), dptr<float>(norm->mem), ctx->num_sms, ctx->stream);
  });
  if (call.rc != FUTHARK_SUCCESS) return call.rc;
  rec->v0 = loss; rec->v1 = counts; rec->v2 = norm;
  *out0 = rec;
  return FUTHARK_SUCCESS;
}

template <typename MAT>
static int router_balance_grad(futhark_context *ctx, const char *name, int elem, MAT **out0, const MAT *r, const futhark_bool_1d *keep,
                               const futhark_i32_1d *counts, const futhark_f32_1d *norm, const futhark_f32_1d *dl) {
  if (!ctx->ready) return not_ready(ctx);
  CtxGuard g(ctx);
  const int64_t n = r->shape[0], e = r->shape[1];
  if (keep->shape[0] != n || counts->shape[0] != e || norm->shape[0] != 1 || dl->shape[0] != 1) return bad_sizes(ctx);
  if (e > fb::ROUTER_MAX_E) return refuse(ctx, "Error: router_balance: at most 1024 experts.\n");
  Call call(ctx);
  auto *dr = call.array<MAT>({n, e}, elem, "router_balance_grad.dr");
  call.launch(name, "vjp of router_balance", [&] { return "{" + kv("n", n) + "," + kv("e", e) + "}"; }, [&] {
    return fb::launch_router_balance_grad(elem, dptr<void>(r->mem), dptr<uint8_t>(keep->mem), dptr<int32_t>(counts->mem), dptr<float>(norm->mem),
                                          dptr<float>(dl->mem), n, e, dptr<void>(dr->mem), ctx->num_sms, ctx->stream);
  });
  if (call.rc != FUTHARK_SUCCESS) return call.rc;
  *out0 = dr;
  return FUTHARK_SUCCESS;
}

extern "C" {

int futhark_entry_router_balance_f32(struct futhark_context *ctx, balance_t **out0, const struct futhark_f32_2d *in0, const struct futhark_bool_1d *in1,
                                     const struct futhark_i32_2d *in2) {
  return router_balance(ctx, "router_balance_f32.seghist_segred", 4, out0, in0, in1, in2);
}
int futhark_entry_router_balance_f16(struct futhark_context *ctx, balance_t **out0, const struct futhark_f16_2d *in0, const struct futhark_bool_1d *in1,
                                     const struct futhark_i32_2d *in2) {
  return router_balance(ctx, "router_balance_f16.seghist_segred", 2, out0, in0, in1, in2);
}
int futhark_entry_router_balance_grad_f32(struct futhark_context *ctx, struct futhark_f32_2d **out0, const struct futhark_f32_2d *in0,
                                          const struct futhark_bool_1d *in1, const struct futhark_i32_1d *in2, const struct futhark_f32_1d *in3,
                                          const struct futhark_f32_1d *in4) {
  return router_balance_grad(ctx, "router_balance_grad_f32.segmap", 4, out0, in0, in1, in2, in3, in4);
}
int futhark_entry_router_balance_grad_f16(struct futhark_context *ctx, struct futhark_f16_2d **out0, const struct futhark_f16_2d *in0,
                                          const struct futhark_bool_1d *in1, const struct futhark_i32_1d *in2, const struct futhark_f32_1d *in3,
                                          const struct futhark_f32_1d *in4) {
  return router_balance_grad(ctx, "router_balance_grad_f16.segmap", 2, out0, in0, in1, in2, in3, in4);
}

// ---- records: `new` and the projections share the blocks of the fields (docs/c-api.rst:366-391) -----------------
}  // extern "C"

template <typename ARR>
static ARR *shared_with(const ARR *a) {
  ARR *c = (ARR *)malloc(sizeof(ARR));
  if (c == nullptr) return nullptr;
  *c = *a;
  fb_ref(&c->mem);
  return c;
}
template <typename ARR>
static int project(futhark_context *ctx, ARR **out, const ARR *field) {
  CtxGuard g(ctx);
  *out = shared_with(field);
  return *out == nullptr;
}
template <typename ARR>
static void drop(futhark_context *ctx, ARR *a) {       // with the context's lock held
  if (a == nullptr) return;
  fb_unref(ctx, &a->mem);
  free(a);
}

template <typename REC, typename ARR>
static int new_pair(futhark_context *ctx, REC **out, const ARR *v0, const ARR *v1) {
  CtxGuard g(ctx);
  REC *r = (REC *)malloc(sizeof(REC));
  if (r == nullptr) return 1;
  r->v0 = shared_with(v0);
  r->v1 = shared_with(v1);
  if (r->v0 == nullptr || r->v1 == nullptr) { drop(ctx, r->v0); drop(ctx, r->v1); free(r); return 1; }
  *out = r;
  return 0;
}
template <typename REC>
static int free_pair(futhark_context *ctx, REC *obj) {
  if (obj == nullptr) return 0;
  CtxGuard g(ctx);
  drop(ctx, obj->v0);
  drop(ctx, obj->v1);
  free(obj);
  return 0;
}

extern "C" {

int futhark_free_opaque_tup2_arr1d_f32_arr1d_f32(struct futhark_context *ctx, losses_t *obj) { return free_pair(ctx, obj); }
int futhark_new_opaque_tup2_arr1d_f32_arr1d_f32(struct futhark_context *ctx, losses_t **out, const struct futhark_f32_1d *v0,
                                                const struct futhark_f32_1d *v1) { return new_pair(ctx, out, v0, v1); }
int futhark_project_opaque_tup2_arr1d_f32_arr1d_f32_0(struct futhark_context *ctx, struct futhark_f32_1d **out, const losses_t *obj) {
  return project(ctx, out, obj->v0);
}
int futhark_project_opaque_tup2_arr1d_f32_arr1d_f32_1(struct futhark_context *ctx, struct futhark_f32_1d **out, const losses_t *obj) {
  return project(ctx, out, obj->v1);
}
int futhark_free_opaque_tup2_arr2d_f16_arr2d_f16(struct futhark_context *ctx, grads_t *obj) { return free_pair(ctx, obj); }
int futhark_new_opaque_tup2_arr2d_f16_arr2d_f16(struct futhark_context *ctx, grads_t **out, const struct futhark_f16_2d *v0,
                                                const struct futhark_f16_2d *v1) { return new_pair(ctx, out, v0, v1); }
int futhark_project_opaque_tup2_arr2d_f16_arr2d_f16_0(struct futhark_context *ctx, struct futhark_f16_2d **out, const grads_t *obj) {
  return project(ctx, out, obj->v0);
}
int futhark_project_opaque_tup2_arr2d_f16_arr2d_f16_1(struct futhark_context *ctx, struct futhark_f16_2d **out, const grads_t *obj) {
  return project(ctx, out, obj->v1);
}
int futhark_free_opaque_tup3_arr1d_f32_arr1d_i32_arr1d_f32(struct futhark_context *ctx, balance_t *obj) {
  if (obj == nullptr) return 0;
  CtxGuard g(ctx);
  drop(ctx, obj->v0);
  drop(ctx, obj->v1);
  drop(ctx, obj->v2);
  free(obj);
  return 0;
}
int futhark_new_opaque_tup3_arr1d_f32_arr1d_i32_arr1d_f32(struct futhark_context *ctx, balance_t **out, const struct futhark_f32_1d *v0,
                                                          const struct futhark_i32_1d *v1, const struct futhark_f32_1d *v2) {
  CtxGuard g(ctx);
  balance_t *r = (balance_t *)malloc(sizeof(balance_t));
  if (r == nullptr) return 1;
  r->v0 = shared_with(v0);
  r->v1 = shared_with(v1);
  r->v2 = shared_with(v2);
  if (r->v0 == nullptr || r->v1 == nullptr || r->v2 == nullptr) { drop(ctx, r->v0); drop(ctx, r->v1); drop(ctx, r->v2); free(r); return 1; }
  *out = r;
  return 0;
}
int futhark_project_opaque_tup3_arr1d_f32_arr1d_i32_arr1d_f32_0(struct futhark_context *ctx, struct futhark_f32_1d **out, const balance_t *obj) {
  return project(ctx, out, obj->v0);
}
int futhark_project_opaque_tup3_arr1d_f32_arr1d_i32_arr1d_f32_1(struct futhark_context *ctx, struct futhark_i32_1d **out, const balance_t *obj) {
  return project(ctx, out, obj->v1);
}
int futhark_project_opaque_tup3_arr1d_f32_arr1d_i32_arr1d_f32_2(struct futhark_context *ctx, struct futhark_f32_1d **out, const balance_t *obj) {
  return project(ctx, out, obj->v2);
}

}  // extern "C"
