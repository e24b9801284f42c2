// operators.h -- what plan.cu calls of operators.cu: the kernels behind b200_kv4_* and b200_log_probs on a plan's own stream.
#pragma once
#include "../../include/b200llama.h"

#include <cuda_runtime.h>

// How a step attention leaves its rows: as the public entry point does (B200_GGML_F32, _F16, _BF16), or as blocks of 32 quants with their scales (Q8_0 plans).
#define KV4_OUT_Q8 8

cudaError_t kv4_append_launch(const b200_kv4 *kv, const b200_kv4_append_args &a, cudaStream_t stream, bool pdl);
cudaError_t kv4_attention_launch(const b200_kv4 *kv, const b200_kv4_attention_args &a, int8_t *quants, float *scales, cudaStream_t stream, bool pdl, int *launches = nullptr);
bool kv4_gave_up(const b200_kv4 *kv); // a wait of a chunk's attention ran out (after a synchronisation)
cudaError_t log_probs_launch(const b200_log_probs_args &a, cudaStream_t stream);
