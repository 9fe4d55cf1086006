// Sums over rows that many CTAs take part in: each writes the sums of its rows to a line of its own, and
// col_finish adds the lines up, always in the same order.  No atomics: the result does not depend on timing.
#pragma once
#include "ff_math.cuh"
#include "launch.cuh"

namespace gtk {

// partial[lines][cols] -> up to three vectors of `each` sums, one after the other in a line (a null one is left out).  A CTA
// of 32 x 8 threads takes 32 columns; 8 threads share a column's lines.
template <typename T>
__global__ void __launch_bounds__(256) col_finish(const float* partial, int lines, long long cols, long long each, T* out0, T* out1, T* out2) {
  __shared__ float s[8][33];
  pdl_begin(partial);
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x;
  float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
  if (c < cols) {
    int l = (int)threadIdx.y;
    for (; l + 24 < lines; l += 32) {
      a0 += partial[(long long)l * cols + c];
      a1 += partial[(long long)(l + 8) * cols + c];
      a2 += partial[(long long)(l + 16) * cols + c];
      a3 += partial[(long long)(l + 24) * cols + c];
    }
    for (; l < lines; l += 8) a0 += partial[(long long)l * cols + c];
  }
  s[threadIdx.y][threadIdx.x] = (a0 + a1) + (a2 + a3);
  __syncthreads();
  if (threadIdx.y == 0 && c < cols) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += s[i][threadIdx.x];
    T* out = c < each ? out0 : c < 2 * each ? out1 : out2;
    if (out) out[c % each] = from_f32<T>(sum);
  }
}

template <typename T>
inline cudaError_t launch_col_finish(const float* partial, int lines, long long cols, long long each, T* out0, T* out1, T* out2, cudaStream_t stream) {
  return launch_pdl(col_finish<T>, dim3((unsigned)((cols + 31) / 32)), dim3(32, 8), stream, partial, lines, cols, each, out0, out1, out2);
}

}  // namespace gtk
