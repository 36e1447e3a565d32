// Arguments and device helpers shared by the batched gated delta rule kernels
// (deltanet_batch.cu, deltanet_chunk.cu).
#pragma once

#include <cuda_bf16.h>
#include <math_constants.h>

#include "common.cuh"
#include "host.cuh"

namespace qfn {

// Rows are tokens; strides in elements.  Value head h uses key head h / ratio.
struct DnRows {
  const uint16_t *q, *k, *v, *beta;
  const float* g;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, g_row, g_head, b_row, b_head;
  uint16_t* out;        // [rows][heads][dv], contiguous
  const float* s_in;    // [slots][heads][dk][dv] or null (zeros)
  float* s_out;
  int heads, ratio, dv;
  float q_scale;        // sqrt(dk): the engine divides q by it
};

__device__ __forceinline__ uint16_t dn_bf16_bits(float v) {
  const __nv_bfloat16 b = __float2bfloat16_rn(v);
  return *reinterpret_cast<const uint16_t*>(&b);
}

// Whether cu[0 .. n] rises within [0, tokens] (read by the whole block).
__device__ __forceinline__ bool dn_plan_ok(const int32_t* cu, int64_t n, int64_t tokens) {
  int bad = 0;
  for (int64_t i = threadIdx.x; i <= n; i += blockDim.x) {
    const int64_t a = cu[i];
    bad |= i == 0 ? a < 0 : a < cu[i - 1];
    bad |= a > tokens;
  }
  return __syncthreads_or(bad) == 0;
}

// Fills DnRows and checks what the batched entry points share.  No row, no
// state: their pointers may be null.
int dn_rows_check(const char* what, const uint16_t* q, const uint16_t* k, const uint16_t* v, const float* g,
                  const uint16_t* beta, const int64_t* strides, const float* s_in, float* s_out, uint16_t* out,
                  int64_t rows, int64_t states, int n_heads, int n_key_heads, int dk, int dv, DnRows* r);

}  // namespace qfn
