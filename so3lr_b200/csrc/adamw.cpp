// extern "C" boundary of the AdamW step: argument checks, then the launchers of
// adamw.cu. Every refusal happens before a launch.
#include "adamw.hpp"

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

#include "checks.hpp"

using so3lr_b200::Error;
using namespace so3lr_b200::checks;

namespace {

void check_count(const so3lr_adamw_args *a) {
  const char *call = "so3lr_adamw";
  require(a != nullptr, "so3lr_adamw: args is NULL");
  length(call, "count", a->count, 0, 1 << 24);
  require(a->count == 0 || a->tensors, "so3lr_adamw: tensors is NULL");
}
// Two updates of the same memory in one call would race.
void distinct(std::vector<std::pair<const char *, const char *>> &parts, const char *what) {
  if (!std::is_sorted(parts.begin(), parts.end())) std::sort(parts.begin(), parts.end());
  for (std::size_t i = 1; i < parts.size(); ++i)
    if (parts[i].first < parts[i - 1].second) throw Error(std::string("so3lr_adamw: the call's ") + what + " overlap");
}
void check(const so3lr_adamw_args *a) {
  const char *call = "so3lr_adamw";
  check_count(a);
  require(a->lr_device || (a->lr >= 0 && a->lr <= 1e30), "so3lr_adamw: lr must be finite and not negative");
  if (a->lr_device) pointer(call, "lr_device", a->lr_device, 4);
  require(a->beta1 >= 0 && a->beta1 < 1 && a->beta2 >= 0 && a->beta2 < 1, "so3lr_adamw: beta1 and beta2 must be in 0..1");
  require(a->eps >= 1e-30 && a->eps <= 1e30, "so3lr_adamw: eps must be in 1e-30..1e30");
  require(a->weight_decay >= 0 && a->weight_decay <= 1e30, "so3lr_adamw: weight_decay must be finite and not negative");
  std::vector<std::pair<const char *, const char *>> params, steps;
  params.reserve(a->count);
  steps.reserve(a->count);
  for (long long i = 0; i < a->count; ++i) {
    const so3lr_adamw_tensor &t = a->tensors[i];
    length(call, "n", t.n, 0, 1LL << 40);
    type(call, "dtype", t.dtype);
    if (t.grad_dtype != t.dtype && t.grad_dtype != SO3LR_FLOAT32)
      throw Error("so3lr_adamw: grad_dtype must be dtype or SO3LR_FLOAT32");
    require((t.exp_avg_scale != nullptr) == (t.exp_avg_sq_scale != nullptr),
            "so3lr_adamw: exp_avg_scale and exp_avg_sq_scale must be given together");
    pointer(call, "step", t.step, 8);
    const char *step = reinterpret_cast<const char *>(t.step);
    steps.emplace_back(step, step + 8);
    if (t.n == 0) continue;
    pointer(call, "param", t.param, bytes_of(t.dtype));
    pointer(call, "grad", t.grad, bytes_of(t.grad_dtype));
    if (t.master) {
      require(t.dtype != SO3LR_FLOAT32, "so3lr_adamw: master is for 16-bit parameters");
      pointer(call, "master", t.master, 4);
    }
    pointer(call, "exp_avg", t.exp_avg, t.exp_avg_scale ? 1 : 4);
    pointer(call, "exp_avg_sq", t.exp_avg_sq, t.exp_avg_scale ? 1 : 4);
    if (t.exp_avg_scale) {
      pointer(call, "exp_avg_scale", t.exp_avg_scale, 4);
      pointer(call, "exp_avg_sq_scale", t.exp_avg_sq_scale, 4);
    }
    const char *p = static_cast<const char *>(t.param);
    params.emplace_back(p, p + t.n * bytes_of(t.dtype));
  }
  distinct(params, "parameters");
  distinct(steps, "step counters");
}
void check(const so3lr_moment_values_args *a) {
  const char *call = "so3lr_moment_values";
  require(a != nullptr, "so3lr_moment_values: args is NULL");
  length(call, "n", a->n, 0, 1LL << 40);
  type(call, "dtype", a->dtype);
  if (a->n == 0) return;
  pointer(call, "codes", a->codes, 1);
  pointer(call, "scales", a->scales, 4);
  pointer(call, "values", a->values, bytes_of(a->dtype));
}

}  // namespace

extern "C" {

long long so3lr_adamw_workspace(const so3lr_adamw_args *args) {
  return sized([&] {
    check_count(args);
    return so3lr_b200::adamw_bytes(*args);
  });
}
int so3lr_adamw_check(const so3lr_adamw_args *args, char *err, size_t errlen) {
  return guarded(err, errlen, [&] { check(args); });
}
int so3lr_adamw(const so3lr_adamw_args *args, void *workspace, long long workspace_bytes, void *stream, char *err,
                size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    workspace_is("so3lr_adamw", workspace, workspace_bytes, so3lr_b200::adamw_bytes(*args));
    if (args->count == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_adamw(*args, workspace, static_cast<cudaStream_t>(stream));
  });
}

int so3lr_moment_values(const so3lr_moment_values_args *args, void *stream, char *err, size_t errlen) {
  return guarded(err, errlen, [&] {
    check(args);
    if (args->n == 0) return;
    so3lr_b200::check_gave_up();
    so3lr_b200::launch_moment_values(*args, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
