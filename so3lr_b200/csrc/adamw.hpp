// AdamW steps (include/so3lr_b200.h): launchers behind the C entry points of
// adamw.cpp. Arguments have been checked there.
#pragma once

#include "layers.hpp"

namespace so3lr_b200 {

long long adamw_bytes(const so3lr_adamw_args &a);
void launch_adamw(const so3lr_adamw_args &a, void *workspace, cudaStream_t s);
void launch_moment_values(const so3lr_moment_values_args &a, cudaStream_t s);

}  // namespace so3lr_b200
