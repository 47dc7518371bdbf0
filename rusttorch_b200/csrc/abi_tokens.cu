// abi_tokens.cu — C-ABI entry points of the token operators (embedding,
// softmax cross entropy against token ids) and of AdamW over many tensors.
// Every argument is checked on the host before the CUDA runtime is touched.
#include "rt_abi_util.h"
#include "rt_tma.cuh"

#include <algorithm>
#include <cmath>
#include <new>

using namespace rt;

namespace {

bool store_type(int dtype, StoreType* t) {
  switch (dtype) {
    case RTC_F32: *t = kF32; return true;
    case RTC_BF16: *t = kBF16; return true;
    case RTC_F16: *t = kF16; return true;
  }
  return false;
}

// What an error is about: "op (argument)", or a name by itself.  Put together
// for an error alone.
struct What {
  const char* op;
  const char* argument;
  std::string text;
  What(const char* o, const char* a) : op(o), argument(a) {}
  What(std::string t) : op(nullptr), argument(nullptr), text(std::move(t)) {}
  std::string get() const {
    return op ? std::string(op) + " (" + argument + ")" : text;
  }
};

rtc_result need_float(const rtc_tensor* t, const What& what, StoreType* out) {
  if (!store_type(t->dtype, out))
    return dtype_mismatch(what.get(), "float32, bfloat16 or float16", dtype_display(t->dtype));
  return ok();
}

rtc_result need_ids(const rtc_tensor* t, const What& what) {
  if (t->dtype != RTC_I32 && t->dtype != RTC_I64)
    return dtype_mismatch(what.get(), "int32 or int64", dtype_display(t->dtype));
  return ok();
}

rtc_result need_dtype(const rtc_tensor* t, int dtype, const What& what) {
  if (t->dtype != dtype)
    return dtype_mismatch(what.get(), dtype_display(dtype), dtype_display(t->dtype));
  return ok();
}

// t has `lead`'s shape, then `last` unless that is kNone.
constexpr size_t kNone = ~size_t(0);
rtc_result need_shape(const rtc_tensor* t, const rtc_tensor* lead, size_t last,
                      const What& what) {
  const size_t extra = last != kNone;
  bool same = t->ndim == lead->ndim + extra && (!extra || t->shape[lead->ndim] == last);
  for (size_t i = 0; same && i < lead->ndim; i++) same = t->shape[i] == lead->shape[i];
  if (same) return ok();
  std::vector<size_t> want = shape_vec(lead);
  if (extra) want.push_back(last);
  return shape_mismatch_vec(what.get(), want, shape_vec(t));
}

rtc_result one_device(const rtc_tensor* a, const rtc_tensor* b) {
  if (a->device != b->device)
    return invalid_argument("device", "all tensors of one call must be on the same device");
  return ok();
}

rtc_result apart(const rtc_tensor* out, const rtc_tensor* in, const char* what) {
  if (!overlap(out, in)) return ok();
  return invalid_argument(what, "must not overlap another tensor of the call");
}

// `out` may be `in` itself, but not another range over the same bytes.
rtc_result apart_or_same(const rtc_tensor* out, const rtc_tensor* in, const char* what) {
  return out->data == in->data ? ok() : apart(out, in, what);
}

constexpr size_t kMaxVocab = 0x7fffffff;

// What a first call sets up (the memory pool, attributes of kernels, occupancy)
// queues nothing: a capture in progress, this thread's or another's, need not
// end for it.
struct SetupInCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  SetupInCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~SetupInCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};

// Runs launch(scratch, flag) on the tensors' device.
template <class F>
rtc_result on_device(int device, size_t scratch_bytes, const char* what, F launch) {
  DeviceScope scope(device);
  if (!scope.ok()) return backend_error("cudaSetDevice", scope.error());
  SetupInCapture setup;
  int* bad = bad_index_flag(device);
  if (!bad) return backend_error(what, cudaErrorInvalidValue);
  if (scratch_bytes == 0) return launched(launch(nullptr, bad), what);
  Scratch scratch(device, scratch_bytes, thread_stream());
  if (scratch.error() != cudaSuccess) return backend_error(what, scratch.error());
  return launched(launch(scratch.get(), bad), what);
}

}  // namespace

// ------------------------------------------------------------------ embedding

extern "C" rtc_result rtc_embedding(const rtc_tensor* weight, const rtc_tensor* ids, float scale,
                                    const rtc_tensor* out) {
  RTC_OP_RANGE();
  const char* ctx = "embedding";
  TRY(check_token_desc(weight, "weight"));
  TRY(check_token_desc(ids, "ids"));
  TRY(check_token_desc(out, "out"));
  StoreType type;
  TRY(need_float(weight, {"embedding", "weight"}, &type));
  TRY(need_ids(ids, {"embedding", "ids"}));
  TRY(need_dtype(out, weight->dtype, {"embedding", "output"}));
  if (weight->ndim != 2)
    return invalid_argument("weight", "must have two dimensions, got " +
                                          std::to_string(weight->ndim));
  const size_t vocab = weight->shape[0], width = weight->shape[1];
  TRY(need_shape(out, ids, width, {"embedding", "output"}));
  if (vocab > kMaxVocab) return invalid_argument("weight", "must have fewer than 2^31 rows");
  TRY(one_device(weight, ids));
  TRY(one_device(weight, out));
  TRY(apart(out, weight, "out"));
  TRY(apart(out, ids, "out"));
  if (out->numel == 0) return ok();
  return on_device(weight->device, 0, ctx, [&](void*, int* bad) {
    return launch_embedding(type, weight->data, ids->data, ids->dtype == RTC_I64, ids->numel,
                            vocab, width, scale, out->data, bad, thread_stream());
  });
}

extern "C" rtc_result rtc_embedding_backward(const rtc_tensor* grad_output, const rtc_tensor* ids,
                                             float scale, int64_t padding_idx, int accumulate,
                                             const rtc_tensor* grad_weight) {
  RTC_OP_RANGE();
  const char* ctx = "embedding_backward";
  TRY(check_token_desc(grad_output, "grad_output"));
  TRY(check_token_desc(ids, "ids"));
  TRY(check_token_desc(grad_weight, "grad_weight"));
  StoreType type, wtype;
  TRY(need_float(grad_output, {"embedding_backward", "grad_output"}, &type));
  TRY(need_ids(ids, {"embedding_backward", "ids"}));
  TRY(need_float(grad_weight, {"embedding_backward", "grad_weight"}, &wtype));
  if (wtype != kF32 && wtype != type)
    return dtype_mismatch("embedding_backward (grad_weight)",
                          "float32 or " + dtype_display(grad_output->dtype),
                          dtype_display(grad_weight->dtype));
  if (grad_weight->ndim != 2)
    return invalid_argument("grad_weight", "must have two dimensions, got " +
                                               std::to_string(grad_weight->ndim));
  const size_t vocab = grad_weight->shape[0], width = grad_weight->shape[1];
  TRY(need_shape(grad_output, ids, width, {"embedding_backward", "grad_output"}));
  if (vocab > kMaxVocab) return invalid_argument("grad_weight", "must have fewer than 2^31 rows");
  if (ids->numel > kMaxVocab) return invalid_argument("ids", "must be fewer than 2^31");
  if (padding_idx >= 0 && (size_t)padding_idx >= vocab)
    return invalid_argument("padding_idx", "must be below the number of rows (" +
                                               std::to_string(vocab) + "), got " +
                                               std::to_string(padding_idx));
  TRY(one_device(grad_output, ids));
  TRY(one_device(grad_output, grad_weight));
  TRY(apart(grad_weight, grad_output, "grad_weight"));
  TRY(apart(grad_weight, ids, "grad_weight"));
  if (grad_weight->numel == 0) return ok();
  return on_device(grad_output->device, embedding_backward_scratch(type, ids->numel, width), ctx,
                   [&](void* scratch, int* bad) {
                     return launch_embedding_backward(
                         type, grad_output->data, ids->data, ids->dtype == RTC_I64, ids->numel,
                         vocab, width, scale, (long long)padding_idx, accumulate != 0,
                         grad_weight->data, wtype != kF32, scratch, bad, thread_stream());
                   });
}

// ------------------------------------------------------ softmax cross entropy

namespace {

rtc_result check_loss(const rtc_tensor* logits, const rtc_tensor* targets, int64_t ignore_index,
                      int reduction, const char* ctx, TokenLoss* a) {
  TRY(check_token_desc(logits, "logits"));
  TRY(check_token_desc(targets, "targets"));
  TRY(need_float(logits, {ctx, "logits"}, &a->type));
  TRY(need_ids(targets, {ctx, "targets"}));
  if (reduction < RTC_REDUCE_NONE || reduction > RTC_REDUCE_SUM)
    return invalid_argument("reduction", "must be RTC_REDUCE_NONE, _MEAN or _SUM");
  if (logits->ndim == 0) return invalid_argument("logits", "must have a last dimension");
  const size_t vocab = logits->shape[logits->ndim - 1];
  TRY(need_shape(logits, targets, vocab, {ctx, "logits vs targets"}));
  if (vocab == 0) return empty_tensor(ctx);
  if (vocab > kMaxVocab) return invalid_argument("logits", "must have fewer than 2^31 classes");
  TRY(one_device(logits, targets));
  a->logits = logits->data;
  a->targets = targets->data;
  a->wide = targets->dtype == RTC_I64;
  a->rows = targets->numel;
  a->vocab = vocab;
  a->ignore = ignore_index;
  a->reduction = reduction;
  a->bad = a->gave_up = nullptr;
  return ok();
}

// One f32 per row, or one in all.
rtc_result check_row_values(const rtc_tensor* t, const rtc_tensor* logits,
                            const rtc_tensor* targets, int reduction, const char* name,
                            const char* ctx) {
  TRY(check_token_desc(t, name));
  TRY(need_dtype(t, RTC_F32, {ctx, name}));
  if (reduction == RTC_REDUCE_NONE)
    TRY(need_shape(t, targets, kNone, {ctx, name}));
  else if (t->numel != 1)
    return invalid_argument(name, "must have one element, got " + std::to_string(t->numel));
  return one_device(logits, t);
}

rtc_result check_grad_logits(const rtc_tensor* logits, const rtc_tensor* targets,
                             const rtc_tensor* grad, const char* ctx) {
  TRY(check_token_desc(grad, "grad_logits"));
  TRY(need_dtype(grad, logits->dtype, {ctx, "grad_logits"}));
  TRY(need_shape(grad, logits, kNone, {ctx, "grad_logits"}));
  TRY(one_device(logits, grad));
  TRY(apart(grad, targets, "grad_logits"));
  return apart_or_same(grad, logits, "grad_logits");
}

rtc_result check_stats(const rtc_tensor* stats, const rtc_tensor* logits,
                       const rtc_tensor* targets, const char* ctx) {
  TRY(check_token_desc(stats, "stats"));
  TRY(need_dtype(stats, RTC_F32, {ctx, "stats"}));
  TRY(need_shape(stats, targets, 3, {ctx, "stats"}));
  return one_device(logits, stats);
}

}  // namespace

extern "C" rtc_result rtc_softmax_cross_entropy(const rtc_tensor* logits,
                                                const rtc_tensor* targets, int64_t ignore_index,
                                                int reduction, const rtc_tensor* loss,
                                                const rtc_tensor* stats) {
  RTC_OP_RANGE();
  const char* ctx = "softmax_cross_entropy";
  TokenLoss a;
  TRY(check_loss(logits, targets, ignore_index, reduction, ctx, &a));
  TRY(check_row_values(loss, logits, targets, reduction, "loss", ctx));
  TRY(apart(loss, logits, "loss"));
  TRY(apart(loss, targets, "loss"));
  if (stats) {
    TRY(check_stats(stats, logits, targets, ctx));
    TRY(apart(stats, logits, "stats"));
    TRY(apart(stats, targets, "stats"));
    TRY(apart(stats, loss, "stats"));
  }
  if (a.rows == 0 && reduction == RTC_REDUCE_NONE) return ok();
  return on_device(logits->device, token_loss_scratch(a), ctx, [&](void* scratch, int* bad) {
    a.bad = bad;
    a.gave_up = wait_timeout_flag(logits->device);
    return launch_token_loss(a, f(loss), stats ? f(stats) : nullptr, scratch, thread_stream());
  });
}

extern "C" rtc_result rtc_softmax_cross_entropy_backward(
    const rtc_tensor* grad_output, const rtc_tensor* logits, const rtc_tensor* targets,
    const rtc_tensor* stats, int64_t ignore_index, int reduction, const rtc_tensor* grad_logits) {
  RTC_OP_RANGE();
  const char* ctx = "softmax_cross_entropy_backward";
  TokenLoss a;
  TRY(check_loss(logits, targets, ignore_index, reduction, ctx, &a));
  TRY(check_row_values(grad_output, logits, targets, reduction, "grad_output", ctx));
  TRY(check_stats(stats, logits, targets, ctx));
  TRY(check_grad_logits(logits, targets, grad_logits, ctx));
  TRY(apart(grad_logits, grad_output, "grad_logits"));
  TRY(apart(grad_logits, stats, "grad_logits"));
  if (a.rows == 0) return ok();
  return on_device(logits->device, token_loss_scratch(a), ctx, [&](void* scratch, int* bad) {
    a.bad = bad;
    a.gave_up = wait_timeout_flag(logits->device);
    return launch_token_loss_backward(a, cf(grad_output), cf(stats), grad_logits->data, scratch,
                                      thread_stream());
  });
}

extern "C" rtc_result rtc_softmax_cross_entropy_grad(const rtc_tensor* logits,
                                                     const rtc_tensor* targets,
                                                     int64_t ignore_index, int reduction,
                                                     float grad_scale, const rtc_tensor* loss,
                                                     const rtc_tensor* grad_logits) {
  RTC_OP_RANGE();
  const char* ctx = "softmax_cross_entropy_grad";
  TokenLoss a;
  TRY(check_loss(logits, targets, ignore_index, reduction, ctx, &a));
  TRY(check_row_values(loss, logits, targets, reduction, "loss", ctx));
  TRY(check_grad_logits(logits, targets, grad_logits, ctx));
  TRY(apart(loss, logits, "loss"));
  TRY(apart(loss, targets, "loss"));
  TRY(apart(loss, grad_logits, "loss"));
  if (a.rows == 0 && reduction == RTC_REDUCE_NONE) return ok();
  return on_device(logits->device, token_loss_scratch(a), ctx, [&](void* scratch, int* bad) {
    a.bad = bad;
    a.gave_up = wait_timeout_flag(logits->device);
    return launch_token_loss_grad(a, grad_scale, f(loss), grad_logits->data, scratch,
                                  thread_stream());
  });
}

// ---------------------------------------------------------- AdamW, many tensors

namespace {

std::string of(const char* list, size_t i) {
  return std::string(list) + "[" + std::to_string(i) + "]";
}

constexpr size_t kMaxListed = size_t(1) << 20;

// The bytes of one tensor of the lists; `list` names it if it is written.
struct Range {
  uintptr_t begin, end;
  size_t i;
  const char* list;
};

// Every tensor of a call, list by list.
struct Ranges {
  static constexpr int kLists = 7;
  std::vector<Range> list[kLists];

  explicit Ranges(size_t n) {
    for (auto& l : list) l.reserve(n);
  }
  void add(int k, const rtc_tensor* t, size_t i, const char* name) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(t->data);
    if (t->numel) list[k].push_back({b, b + t->numel * dtype_bytes(t->dtype), i, name});
  }

  // Whether each list's tensors follow one another in memory and no two lists'
  // spans meet, as where a list was cut from one buffer.
  bool laid_out() const {
    for (const auto& l : list)
      for (size_t i = 1; i < l.size(); i++)
        if (l[i].begin < l[i - 1].end) return false;
    for (int a = 0; a < kLists; a++)
      for (int b = 0; b < a; b++)
        if (!list[a].empty() && !list[b].empty() && list[a].front().begin < list[b].back().end &&
            list[b].front().begin < list[a].back().end)
          return false;
    return true;
  }
};

// No written tensor may share bytes with another (the same parameter twice in
// one call, say): the blocks of both would race.
rtc_result no_shared_writes(const Ranges& ranges) {
  if (ranges.laid_out()) return ok();
  std::vector<Range> r;
  for (const auto& l : ranges.list) r.insert(r.end(), l.begin(), l.end());
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  const Range* written = nullptr;   // of those before: the written one, and the
  const Range* any = nullptr;       // one at all, that reach furthest
  for (const Range& x : r) {
    const Range* hit = written && written->end > x.begin ? written : nullptr;
    if (!hit && x.list && any && any->end > x.begin) hit = &x;
    if (hit)
      return invalid_argument(of(hit->list, hit->i),
                              "must not overlap another tensor of the call");
    if (x.list && (!written || x.end > written->end)) written = &x;
    if (!any || x.end > any->end) any = &x;
  }
  return ok();
}

rtc_result check_moments(const rtc_tensor* p, const rtc_tensor* codes, const rtc_tensor* scales,
                         const std::string& name, const std::string& scale_name) {
  TRY(need_dtype(codes, RTC_F8E4M3, name));
  TRY(check_token_desc(scales, scale_name.c_str()));
  TRY(need_dtype(scales, RTC_F32, scale_name));
  const size_t blocks = (p->numel + kMomentBlock - 1) / kMomentBlock;
  if (scales->numel != blocks)
    return invalid_argument(scale_name, "must have one element per " +
                                            std::to_string(kMomentBlock) + " (" +
                                            std::to_string(blocks) + "), got " +
                                            std::to_string(scales->numel));
  return one_device(p, scales);
}

// Tensor i of the lists, with the errors that its checks give.
rtc_result check_listed(const rtc_tensor* params, const rtc_tensor* grads, const rtc_tensor* m,
                        const rtc_tensor* v, const rtc_tensor* m_scales,
                        const rtc_tensor* v_scales, const rtc_tensor* copies, size_t i) {
  const rtc_tensor* p = &params[i];
  TRY(check_token_desc(p, of("params", i).c_str()));
  TRY(check_token_desc(&grads[i], of("grads", i).c_str()));
  TRY(check_token_desc(&m[i], of("m", i).c_str()));
  TRY(check_token_desc(&v[i], of("v", i).c_str()));
  StoreType type;
  TRY(need_dtype(p, RTC_F32, of("params", i)));
  TRY(need_float(&grads[i], of("grads", i), &type));
  if (!same_shape(p, &grads[i])) return shape_mismatch(of("grads", i), p, &grads[i]);
  if (!same_shape(p, &m[i])) return shape_mismatch(of("m", i), p, &m[i]);
  if (!same_shape(p, &v[i])) return shape_mismatch(of("v", i), p, &v[i]);
  TRY(one_device(&params[0], p));
  TRY(one_device(p, &grads[i]));
  TRY(one_device(p, &m[i]));
  TRY(one_device(p, &v[i]));
  if (m_scales) {
    TRY(check_moments(p, &m[i], &m_scales[i], of("m", i), of("m_scales", i)));
    TRY(check_moments(p, &v[i], &v_scales[i], of("v", i), of("v_scales", i)));
  } else {
    TRY(need_dtype(&m[i], RTC_F32, of("m", i)));
    TRY(need_dtype(&v[i], RTC_F32, of("v", i)));
  }
  if (copies) {
    TRY(check_token_desc(&copies[i], of("copies", i).c_str()));
    if (copies[i].dtype != RTC_BF16 && copies[i].dtype != RTC_F16)
      return dtype_mismatch(of("copies", i), "bfloat16 or float16", dtype_display(copies[i].dtype));
    if (!same_shape(p, &copies[i])) return shape_mismatch(of("copies", i), p, &copies[i]);
    TRY(one_device(p, &copies[i]));
  }
  return ok();
}

// Whether a tensor passes check_listed as most do: contiguous without strides,
// on p's device, of the type and shape that its list wants.  A short-cut:
// what it does not know goes to check_listed.
bool plain(const rtc_tensor* t) {
  if (t->strides || t->device < 0 || (t->ndim > 0 && !t->shape)) return false;
  unsigned __int128 prod = 1;
  for (size_t i = 0; i < t->ndim; i++) {
    prod *= t->shape[i];
    if (prod > SIZE_MAX) return false;
  }
  return prod == t->numel && (t->numel == 0 || t->data) &&
         (reinterpret_cast<uintptr_t>(t->data) & (dtype_bytes(t->dtype) - 1)) == 0;
}
bool plain_f32(const rtc_tensor* t) { return t->dtype == RTC_F32 && plain(t); }
// p is plain.
bool plain_like(const rtc_tensor* t, const rtc_tensor* p) {
  if (t->strides || t->device != p->device || t->ndim != p->ndim || t->numel != p->numel ||
      (t->ndim > 0 && !t->shape))
    return false;
  for (size_t i = 0; i < t->ndim; i++)
    if (t->shape[i] != p->shape[i]) return false;
  return (t->numel == 0 || t->data) &&
         (reinterpret_cast<uintptr_t>(t->data) & (dtype_bytes(t->dtype) - 1)) == 0;
}
bool plain_moment(const rtc_tensor* t, const rtc_tensor* p, bool eight) {
  return t->dtype == (eight ? int(RTC_F8E4M3) : int(RTC_F32)) && plain_like(t, p);
}
bool plain_grad(const rtc_tensor* t, const rtc_tensor* p) {
  StoreType type;
  return store_type(t->dtype, &type) && plain_like(t, p);
}
bool plain_copy(const rtc_tensor* t, const rtc_tensor* p) {
  return (t->dtype == RTC_BF16 || t->dtype == RTC_F16) && plain_like(t, p);
}
bool plain_scales(const rtc_tensor* t, const rtc_tensor* p) {
  return t->dtype == RTC_F32 && plain(t) && t->device == p->device &&
         t->numel == (p->numel + kMomentBlock - 1) / kMomentBlock;
}

}  // namespace

extern "C" rtc_result rtc_adamw_update_multi(
    const rtc_tensor* params, const rtc_tensor* grads, const rtc_tensor* m, const rtc_tensor* v,
    const rtc_tensor* m_scales, const rtc_tensor* v_scales, const rtc_tensor* copies, size_t n,
    double learning_rate, double beta1, double beta2, double epsilon, double weight_decay,
    uint64_t timestep, uint64_t seed) try {
  RTC_OP_RANGE();
  if (n == 0) return ok();
  if (!params) return invalid_argument("params", "must not be null");
  if (!grads) return invalid_argument("grads", "must not be null");
  if (!m) return invalid_argument("m", "must not be null");
  if (!v) return invalid_argument("v", "must not be null");
  if (!m_scales != !v_scales)
    return invalid_argument("v_scales", "m_scales and v_scales must both be given or both be null");
  const bool eight = m_scales != nullptr;
  if (n > kMaxListed)
    return invalid_argument("n", "must be at most " + std::to_string(kMaxListed) + " tensors");
  if (weight_decay < 0.0)
    return invalid_argument("weight_decay", "must be non-negative, got " + rust_f64(weight_decay));
  std::vector<AdamTensor> list(n);
  Ranges ranges(n);
  for (size_t i = 0; i < n; i++) {
    const rtc_tensor* p = &params[i];
    AdamTensor& t = list[i];
    // what is right is not named: the names are built for an error alone
    const bool plain =
        plain_f32(p) && p->device == params[0].device && plain_moment(&m[i], p, eight) &&
        plain_moment(&v[i], p, eight) && plain_grad(&grads[i], p) &&
        (!eight || (plain_scales(&m_scales[i], p) && plain_scales(&v_scales[i], p))) &&
        (!copies || plain_copy(&copies[i], p));
    if (!plain) TRY(check_listed(params, grads, m, v, m_scales, v_scales, copies, i));
    store_type(grads[i].dtype, &t.gtype);
    t.ms = eight ? f(&m_scales[i]) : nullptr;
    t.vs = eight ? f(&v_scales[i]) : nullptr;
    t.copy = nullptr;
    t.ctype = kBF16;
    if (copies) {
      store_type(copies[i].dtype, &t.ctype);
      t.copy = copies[i].data;
    }
    t.p = f(p);
    t.g = grads[i].data;
    t.m = m[i].data;
    t.v = v[i].data;
    t.n = p->numel;
    ranges.add(0, p, i, "params");
    ranges.add(1, &grads[i], i, nullptr);
    ranges.add(2, &m[i], i, "m");
    ranges.add(3, &v[i], i, "v");
    if (eight) {
      ranges.add(4, &m_scales[i], i, "m_scales");
      ranges.add(5, &v_scales[i], i, "v_scales");
    }
    if (copies) ranges.add(6, &copies[i], i, "copies");
  }
  TRY(no_shared_writes(ranges));
  TRY(adam_hyper_checks(learning_rate, beta1, beta2, epsilon, timestep));
  return on_device(params[0].device, 0, "adamw_update_multi", [&](void*, int*) {
    const AdamCoeffs c =
        adam_coeffs(learning_rate, beta1, beta2, epsilon, weight_decay, timestep, true);
    if (!eight) return launch_adam_multi(list.data(), n, c, thread_stream());
    Adam8Coeffs c8;
    c8.b1 = c.b1;
    c8.one_minus_b1 = c.one_minus_b1;
    c8.b2 = c.b2;
    c8.one_minus_b2 = c.one_minus_b2;
    c8.c2 = (float)(1.0 / std::sqrt(1.0 - std::pow(beta2, (double)timestep)));
    c8.eps = std::max(c.eps, 0x1p-126f);   // a normal number, for the reciprocal
    c8.step = (float)(learning_rate / (1.0 - std::pow(beta1, (double)timestep)));
    c8.lr_wd = c.decay ? c.lr_wd : 0.0f;
    c8.one = 1.0f;
    return launch_adam8_multi(list.data(), n, c8, seed, wait_timeout_flag(params[0].device),
                              thread_stream());
  });
} catch (const std::bad_alloc&) {   // the lists' copies
  return backend_error("adamw_update_multi", cudaErrorMemoryAllocation);
}

namespace {
rtc_result check_packed(const rtc_tensor* m, const rtc_tensor* v, const rtc_tensor* mc,
                        const rtc_tensor* ms, const rtc_tensor* vc, const rtc_tensor* vs) {
  TRY(check_token_desc(m, "m"));
  TRY(check_token_desc(v, "v"));
  TRY(check_token_desc(mc, "m_codes"));
  TRY(check_token_desc(vc, "v_codes"));
  TRY(need_dtype(m, RTC_F32, What("m")));
  TRY(need_dtype(v, RTC_F32, What("v")));
  if (!same_shape(m, v)) return shape_mismatch("v", m, v);
  if (!same_shape(m, mc)) return shape_mismatch("m_codes", m, mc);
  if (!same_shape(m, vc)) return shape_mismatch("v_codes", m, vc);
  TRY(one_device(m, v));
  TRY(one_device(m, mc));
  TRY(one_device(m, vc));
  TRY(check_moments(m, mc, ms, "m_codes", "m_scales"));
  TRY(check_moments(m, vc, vs, "v_codes", "v_scales"));
  const rtc_tensor* all[6] = {m, v, mc, ms, vc, vs};
  for (int i = 0; i < 6; i++)
    for (int j = 0; j < i; j++) TRY(apart(all[i], all[j], "tensors"));
  return ok();
}
}  // namespace

extern "C" rtc_result rtc_adamw8_pack(const rtc_tensor* m, const rtc_tensor* v,
                                      const rtc_tensor* m_codes, const rtc_tensor* m_scales,
                                      const rtc_tensor* v_codes, const rtc_tensor* v_scales) {
  RTC_OP_RANGE();
  TRY(check_packed(m, v, m_codes, m_scales, v_codes, v_scales));
  if (m->numel == 0) return ok();
  return on_device(m->device, 0, "adamw8_pack", [&](void*, int*) {
    return launch_adam8_pack(cf(m), cf(v), m_codes->data, f(m_scales), v_codes->data, f(v_scales),
                             m->numel, thread_stream());
  });
}

extern "C" rtc_result rtc_adamw8_unpack(const rtc_tensor* m_codes, const rtc_tensor* m_scales,
                                        const rtc_tensor* v_codes, const rtc_tensor* v_scales,
                                        const rtc_tensor* m, const rtc_tensor* v) {
  RTC_OP_RANGE();
  TRY(check_packed(m, v, m_codes, m_scales, v_codes, v_scales));
  if (m->numel == 0) return ok();
  return on_device(m->device, 0, "adamw8_unpack", [&](void*, int*) {
    return launch_adam8_unpack(m_codes->data, cf(m_scales), v_codes->data, cf(v_scales), f(m),
                               f(v), m->numel, thread_stream());
  });
}
