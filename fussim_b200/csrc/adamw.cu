// C entry point of the AdamW step: argument checks, the tables of tensors and the launches. The
// kernel is in adamw.cuh.
#include "adamw.cuh"

#include <cmath>
#include <cstdint>
#include <memory>
#include <string>

#include "engine_host.h"
#include "launch_host.h"

namespace {

using fssim::AdamwTable;
using fssim::kAdamwBlock;
using fssim::kAdamwThreads;
using fssim::kRunUnit;
using fssim_host::aligned;
using fssim_host::fail;
using fssim_host::guarded;
using fssim_host::launch;
using fssim_host::NvtxRange;

// Runs per launch: a small table (4 KB of parameters) or a large one (31 KB, of the 32 KB that a
// launch may carry).
constexpr int kFew = 64;
constexpr int kMany = 448;
static_assert(sizeof(AdamwTable<kMany>) <= 32764, "kernel parameters are limited to 32764 bytes");

size_t elem_size(int dtype) { return dtype == FSSIM_F32 ? 4 : 2; }
bool known_dtype(int d) { return d == FSSIM_F32 || d == FSSIM_F16 || d == FSSIM_BF16; }
bool within(double v, double least, double below) { return v >= least && v < below; }

int check(const fssim_adamw_args* a) {
  if (!a) return fail(FSSIM_ERR_NULLPTR, "args is NULL");
  if (a->count < 0) return fail(FSSIM_ERR_SHAPE, "negative number of tensors");
  if (a->state_bits != 32 && a->state_bits != 8) return fail(FSSIM_ERR_ARGUMENT, "state_bits must be 32 or 8");
  if (!within(a->beta1, 0.0, 1.0) || !within(a->beta2, 0.0, 1.0))
    return fail(FSSIM_ERR_ARGUMENT, "beta1 and beta2 must be at least 0 and below 1");
  if (!within(a->eps, 0.0, HUGE_VAL) || !within(a->weight_decay, 0.0, HUGE_VAL))
    return fail(FSSIM_ERR_ARGUMENT, "eps and weight_decay must be finite and not negative");
  if (!a->lr_at && !within(a->lr, 0.0, HUGE_VAL)) return fail(FSSIM_ERR_ARGUMENT, "lr must be finite and not negative");
  if (!a->step_at && a->step < 1) return fail(FSSIM_ERR_ARGUMENT, "steps are counted from 1");
  if (a->norm && !(a->max_norm >= 0.0)) return fail(FSSIM_ERR_ARGUMENT, "max_norm must not be negative");
  for (const void* p : {static_cast<const void*>(a->step_at), static_cast<const void*>(a->lr_at),
                        static_cast<const void*>(a->norm)})
    if (!aligned(p, 4)) return fail(FSSIM_ERR_ARGUMENT, "step_at, lr_at and norm must be aligned to 4 bytes");
  const bool coded = a->state_bits == 8;
  if (a->count > 0 && (!a->params || !a->grads || !a->exp_avgs || !a->exp_avg_sqs || !a->sizes || !a->dtypes ||
                       !a->grad_dtypes || (coded && !a->scales) || (a->copies && !a->copy_dtypes)))
    return fail(FSSIM_ERR_NULLPTR, "an array of the tensors' is NULL");
  for (int64_t i = 0; i < a->count; ++i) {
    if (a->sizes[i] < 0 || a->sizes[i] > (int64_t{1} << 60))
      return fail(FSSIM_ERR_SHAPE, "a tensor's size is negative or too large");
    const int p = a->dtypes[i], g = a->grad_dtypes[i];
    if (!known_dtype(p) || !known_dtype(g) || (p != FSSIM_F32 && g != p && g != FSSIM_F32))
      return fail(FSSIM_ERR_DTYPE, "parameters must be F32, F16 or BF16, gradients of their type or F32 (of any "
                                   "of the three beside F32 parameters)");
    if (a->copies && (p != FSSIM_F32 || (a->copy_dtypes[i] != FSSIM_F16 && a->copy_dtypes[i] != FSSIM_BF16)))
      return fail(FSSIM_ERR_DTYPE, "copies are F16 or BF16, of F32 parameters");
    if (a->sizes[i] == 0) continue;
    const struct {
      const void* p;
      size_t align;
    } all[] = {{a->params[i], elem_size(p)},
               {a->grads[i], elem_size(g)},
               {a->exp_avgs[i], coded ? 1u : 4u},
               {a->exp_avg_sqs[i], coded ? 1u : 4u},
               {coded ? a->scales[i] : a->params[i], coded ? 4u : 1u},
               {a->copies ? a->copies[i] : a->params[i], a->copies ? 2u : 1u}};
    for (const auto& t : all) {
      if (!t.p) return fail(FSSIM_ERR_NULLPTR, "a tensor's pointer is NULL");
      if (!aligned(t.p, t.align)) return fail(FSSIM_ERR_ARGUMENT, "a tensor is not aligned to its element size");
    }
  }
  return FSSIM_OK;
}

int64_t units_of(int64_t size) { return (size + kRunUnit - 1) / kRunUnit; }

// The next tensors from `begin` on that are not empty, K of them at most; returns where they end.
template <int K>
int64_t fill(const fssim_adamw_args& a, int64_t begin, AdamwTable<K>* t) {
  int r = 0;
  int64_t unit = 0, i = begin;
  for (; i < a.count && r < K; ++i) {
    if (a.sizes[i] == 0) continue;
    t->param[r] = a.params[i];
    t->grad[r] = a.grads[i];
    t->first[r] = a.exp_avgs[i];
    t->second[r] = a.exp_avg_sqs[i];
    t->scales[r] = a.state_bits == 8 ? a.scales[i] : nullptr;
    t->copy[r] = a.copies ? a.copies[i] : nullptr;
    t->copy_dtype[r] = static_cast<unsigned char>(a.copies ? a.copy_dtypes[i] : 0);
    t->kind[r] = static_cast<unsigned char>(fssim::adamw_kind(a.dtypes[i], a.grad_dtypes[i]));
    t->size[r] = a.sizes[i];
    t->index[r] = static_cast<uint32_t>(i);
    t->unit0[r] = unit;
    unit += units_of(a.sizes[i]);
    ++r;
  }
  t->unit0[r] = unit;
  t->count = r;
  t->step = {a.beta1, a.beta2, a.eps,   a.lr,   a.weight_decay, a.max_norm, a.step,
             a.step_at, a.lr_at, a.norm, a.seed, a.maximize};
  return i;
}

template <int K>
int launch_from(const fssim_adamw_args& a, int64_t* begin, cudaStream_t stream) {
  const std::unique_ptr<AdamwTable<K>> t(new AdamwTable<K>);
  *begin = fill(a, *begin, t.get());
  if (t->count == 0) return FSSIM_OK;
  const int64_t units = t->unit0[t->count];
  const int64_t most = 148 * fssim::adamw_resident(a.state_bits);
  const unsigned grid = static_cast<unsigned>(units < most ? units : most);
  return a.state_bits == 32
             ? launch(fssim::adamw_kernel<32, K>, grid, kAdamwThreads, 0, stream, "AdamW launch", *t)
             : launch(fssim::adamw_kernel<8, K>, grid, kAdamwThreads, 0, stream, "AdamW launch", *t);
}

int run(const fssim_adamw_args* a, cudaStream_t stream) {
  int st = check(a);
  for (int64_t i = 0; !st && i < a->count;)
    st = a->count - i <= kFew ? launch_from<kFew>(*a, &i, stream) : launch_from<kMany>(*a, &i, stream);
  return st;
}

}  // namespace

extern "C" {

int fssim_adamw_step(const fssim_adamw_args* a, fssim_stream_t stream) {
  NvtxRange range("fssim_adamw_step");
  return guarded([&] { return run(a, stream); });
}

}  // extern "C"
