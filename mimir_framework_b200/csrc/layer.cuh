// layer.cuh — the launches of a layer's norms and products in the serving group (serve.cu checks their arguments).
#pragma once

#include <cuda_runtime.h>

#include "mimir_b200.h"

namespace mb {

int launch_norm_rows(const MimirNormRows& a, cudaStream_t st);
// gated: a.up is there
int launch_linear(const MimirLinear& a, bool gated, cudaStream_t st);

}  // namespace mb
