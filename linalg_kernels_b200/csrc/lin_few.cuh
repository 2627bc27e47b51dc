// lin_few.cuh — grouped products with few rows per group.
#pragma once

#include "lin_common.cuh"

namespace lin {

bool few_better(const Product& p);
int launch_few(const Product& p, cudaStream_t q);
cudaError_t prepare_few();

}  // namespace lin
