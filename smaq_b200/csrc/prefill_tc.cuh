// The tcgen05 prefill kernel (prefill_tc.cu) as paged_prefill.cu dispatches to it.
#pragma once
#include "paged.cuh"

namespace smaq {
bool prefill_tc_eligible(const smaq_paged_args& a);
size_t prefill_tc_workspace(int64_t n_rows, int batch, int n_q_heads, int n_kv_heads, int head_dim, int64_t max_tokens);
int launch_prefill_tc(const PagedParams& p, cudaStream_t st);
}  // namespace smaq
