// Block-scaled 8-bit float linear, first form: one thread per output, the
// sum of each 128-column block in f32, scaled and added to the total.
#include "fp8_rows.cuh"
#include <cuda_fp8.h>

namespace g4m {

__device__ __forceinline__ float e4m3_f32(uint8_t c) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

__global__ void __launch_bounds__(128) fp8_gemm_simple_kernel(Fp8GemmArgs a) {
  const int o = blockIdx.x * 128 + threadIdx.x;
  if (o >= a.out) return;
  const int blocks = (a.in + kFp8Block - 1) / kFp8Block;
  for (long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    float total = 0.0f;
    for (int k = 0; k < blocks; ++k) {
      float s = 0.0f;
      const int end = min(a.in, (k + 1) * kFp8Block);
      for (int c = k * kFp8Block; c < end; ++c) s = fmaf(e4m3_f32(a.x[r * a.ldx + c]), e4m3_f32(a.w[(long)o * a.in + c]), s);
      total = fmaf(s, a.sx[k * a.lds + r] * a.sw[(long)(o / kFp8Block) * blocks + k], total);
    }
    if (a.bias) total += a.bias[o];
    with_type(a.y_dtype, [&](auto* tp) { from_f32(total, static_cast<decltype(tp)>(a.y) + r * a.ldy + o); });
  }
}

cudaError_t fp8_gemm(const Fp8GemmArgs& a, cudaStream_t st) {
  const dim3 grid((a.out + 127) / 128, (unsigned)(a.rows < 32768 ? a.rows : 32768));
  fp8_gemm_simple_kernel<<<grid, 128, 0, st>>>(a);
  return cudaGetLastError();
}

}  // namespace g4m
