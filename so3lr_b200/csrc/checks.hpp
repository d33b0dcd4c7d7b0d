// Argument checks of the layers' C entry points (layers.cpp, block.cpp, adamw.cpp): every
// refusal is an Error with the call's and the argument's name, thrown before a launch;
// `guarded` and `sized` end it at the boundary.
#pragma once

#include <cstdio>
#include <cstring>
#include <exception>
#include <string>

#include "../../include/so3lr_b200.h"
#include "model_host.hpp"

namespace so3lr_b200 {
namespace checks {

constexpr long long kMaxLength = 1LL << 30;  // rows, widths: kernels index rows and columns with 32 bits
constexpr long long kMaxStride = 1LL << 40;

inline void require(bool ok, const char *what) {
  if (!ok) throw Error(what);
}
inline std::string name(const char *call, const char *arg, const char *what) {
  return std::string(call) + ": " + arg + " " + what;
}
inline bool float_type(int t) { return t == SO3LR_FLOAT32 || t == SO3LR_BFLOAT16 || t == SO3LR_FLOAT16; }
inline std::size_t bytes_of(int t) { return t == SO3LR_FLOAT32 ? 4 : 2; }

inline void length(const char *call, const char *arg, long long v, long long lo, long long hi) {
  if (v < lo || v > hi)
    throw Error(name(call, arg, "must be in ") + std::to_string(lo) + ".." + std::to_string(hi) + ", got " +
                std::to_string(v));
}
inline void pointer(const char *call, const char *arg, const void *p, std::size_t align) {
  if (!p) throw Error(name(call, arg, "is NULL"));
  if (reinterpret_cast<std::size_t>(p) % align) throw Error(name(call, arg, "is not aligned to its element type"));
}
// an input (any row stride >= 0) or an output (rows must not overlap)
inline void matrix(const char *call, const char *arg, const void *p, long long stride, long long rows, long long width,
            std::size_t size, bool output) {
  if (rows == 0) return;
  pointer(call, arg, p, size);
  if (stride < 0 || stride > kMaxStride || (output && rows > 1 && stride < width))
    throw Error(name(call, arg, output ? "needs a row stride of at least its row length"
                                       : "needs a row stride that is not negative"));
}
inline void type(const char *call, const char *arg, int t, bool half_only = false) {
  if (!float_type(t) || (half_only && t == SO3LR_FLOAT32))
    throw Error(name(call, arg, half_only ? "must be SO3LR_BFLOAT16 or SO3LR_FLOAT16"
                                          : "must be SO3LR_FLOAT32, SO3LR_BFLOAT16 or SO3LR_FLOAT16"));
}
inline void workspace_is(const char *call, const void *ws, long long have, long long need) {
  if (need < 0) throw Error(std::string(call) + ": invalid sizes");
  if (need == 0) return;
  if (have < need)
    throw Error(std::string(call) + ": the workspace has " + std::to_string(have) + " bytes, " +
                std::to_string(need) + " are needed");
  pointer(call, "workspace", ws, 256);
}

template <class F>
int guarded(char *err, std::size_t errlen, F &&f) {
  try {
    f();
    return 0;
  } catch (const std::exception &e) {
    if (err && errlen > 0) {
      std::strncpy(err, e.what(), errlen - 1);
      err[errlen - 1] = '\0';
    }
    return 1;
  } catch (...) {
    if (err && errlen > 0) std::snprintf(err, errlen, "unknown exception");
    return 1;
  }
}
template <class F>
long long sized(F &&f) {
  try {
    return f();
  } catch (...) {
    return -1;
  }
}

}  // namespace checks
}  // namespace so3lr_b200
