// Host-side launcher of the verification of drafted tokens (verify.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fp8lin {

size_t verify_ws_bytes(int64_t T, int64_t B, int64_t V);
hipError_t launch_verify(const void* logits, bool bf16, int64_t ld, const float* probs, int64_t ldp, int64_t prob_rows,
                         const int64_t* tokens, const float* u, const int32_t* offsets, const float* temperature, int64_t T,
                         int B, int V, int32_t* accepted, int64_t* out, void* ws, hipStream_t stream);

}  // namespace fp8lin
