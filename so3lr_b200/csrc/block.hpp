// What a block is made of besides its feed-forward layer (include/so3lr_b200.h): the norms
// on both sides of its boundary and the dense layer. Launchers behind the C entry points of
// block.cpp. Arguments have been checked there.
#pragma once

#include "layers.hpp"

namespace so3lr_b200 {

// sandwich.cu
void launch_sandwich_norm(const so3lr_sandwich_norm_args &a, cudaStream_t s);
long long sandwich_norm_backward_bytes(const so3lr_sandwich_norm_backward_args &a);
void launch_sandwich_norm_backward(const so3lr_sandwich_norm_backward_args &a, void *workspace, cudaStream_t s);

}  // namespace so3lr_b200
