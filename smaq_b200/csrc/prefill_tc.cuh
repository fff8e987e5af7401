// The tcgen05 prefill kernel (prefill_tc.cu) as paged_prefill.cu dispatches to it.
#pragma once
#include "paged.cuh"

namespace smaq {
bool prefill_tc_eligible(const smaq_paged_args& a);
int launch_prefill_tc(const PagedParams& p, cudaStream_t st);
}  // namespace smaq
