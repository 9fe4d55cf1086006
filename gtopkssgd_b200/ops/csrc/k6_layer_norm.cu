// K6: layer norm over the last axis, forward and backward.
//
//   mean = sum x / D, rstd = (sum (x - mean)^2 / D + eps)^-1/2, xh = (x - mean) rstd, y = xh w + b
//   t = dy w, dx = rstd (t - mean_D(t) - xh mean_D(t xh)) + add, dw = sum_R dy xh, db = sum_R dy
//
// Bound by memory: the forward pass reads x and writes y, the backward pass reads dy and x and writes dx.  A row is
// read once and stays in registers (the variance is summed over the centred values, not from sums of squares).  A
// group of warps takes a row.  In the backward pass the groups go through rows in turn, the column sums of a
// thread's own columns stay in its registers all along, the groups of a CTA join theirs in shared memory, and
// col_finish adds up one line per CTA.
#include "colsum.cuh"
#include "common.cuh"
#include "host_api.h"
#include "launch.cuh"

namespace gtk {

constexpr int kNormMaxWarps = 32;

// Sum of N values over the threads of a group of `warps` warps (named barrier `bar`; scratch: 2 x N x 32 floats per
// group, used in turn so that one barrier per sum is enough).
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int warps, int warp, int bar, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (warps == 1) return;
  if (lane_id() == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) scratch[i * kNormMaxWarps + warp] = v[i];
  asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(warps * 32) : "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = (int)lane_id() < warps ? scratch[i * kNormMaxWarps + lane_id()] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    v[i] = s;
  }
}

struct NormShape {
  long long rows, x_ld, dy_ld, add_ld;   // leading dimensions in elements
  int cols;
  int warps;                             // of a group
  float eps;
};

// blockDim = (32 * warps, groups).  NV vectors of VEC elements per thread cover the row.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(1024) k6_norm_forward(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, NormShape s) {
  __shared__ float scratch[8][2][kNormMaxWarps];
  pdl_begin(x, w, b);
  const int threads = s.warps * 32, at = (int)threadIdx.x, group = (int)threadIdx.y;
  const long long row = (long long)blockIdx.x * blockDim.y + group;
  if (row >= s.rows) return;   // the whole group
  const T* xr = x + row * s.x_ld;
  float v[NV][VEC];
  float sum[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (at + i * threads) * VEC;
    if (c < s.cols) {
      load_f32<T, VEC>(xr + c, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) sum[0] += v[i][j];
  group_sum<1>(sum, s.warps, at >> 5, 1 + group, scratch[group][0]);
  const float m = sum[0] / (float)s.cols;
  float sq[1] = {0.f};
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((at + i * threads) * VEC < s.cols)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] -= m;
        sq[0] += v[i][j] * v[i][j];
      }
  group_sum<1>(sq, s.warps, at >> 5, 1 + group, scratch[group][1]);
  const float r = 1.f / sqrtf(sq[0] / (float)s.cols + s.eps);
  if (at == 0) {
    mean[row] = m;
    rstd[row] = r;
  }
  T* yr = y + row * s.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (at + i * threads) * VEC;
    if (c < s.cols) {
      float wv[VEC], bv[VEC];
      if (w) load_f32<T, VEC>(w + c, wv);
      if (b) load_f32<T, VEC>(b + c, bv);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float o = v[i][j] * r;
        if (w) o *= wv[j];
        if (b) o += bv[j];
        v[i][j] = o;
      }
      store_f32<T, VEC>(yr + c, v[i]);
    }
  }
}

// Rows longer than the registers hold: three passes over the row, the later two from the caches.
template <typename T>
__global__ void __launch_bounds__(1024) k6_norm_forward_long(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, NormShape s) {
  __shared__ float scratch[2][kNormMaxWarps];
  pdl_begin(x, w, b);
  for (long long row = blockIdx.x; row < s.rows; row += gridDim.x) {
    const T* xr = x + row * s.x_ld;
    float sum[1] = {0.f};
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) sum[0] += to_f32(xr[c]);
    group_sum<1>(sum, 32, (int)threadIdx.x >> 5, 1, scratch[0]);
    const float m = sum[0] / (float)s.cols;
    float sq[1] = {0.f};
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) {
      const float d = to_f32(xr[c]) - m;
      sq[0] += d * d;
    }
    group_sum<1>(sq, 32, (int)threadIdx.x >> 5, 1, scratch[1]);
    const float r = 1.f / sqrtf(sq[0] / (float)s.cols + s.eps);
    if (threadIdx.x == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) {
      float o = (to_f32(xr[c]) - m) * r;
      if (w) o *= to_f32(w[c]);
      if (b) o += to_f32(b[c]);
      y[row * s.cols + c] = from_f32<T>(o);
    }
  }
}

// partial: [gridDim.x][2 * cols], sums of dy xh, then of dy.  blockDim = (32 * warps, groups).  THREADS: the most that it
// is launched with; with 1024 (rows over 8192 elements) the column sums do not fit the registers and lie in shared memory.
template <typename T, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS)
k6_norm_backward(const T* dy, const T* x, const float* mean, const float* rstd, const T* w, const T* add, T* dx, float* partial, NormShape s) {
  constexpr bool kShared = THREADS > 512;
  extern __shared__ float joined[];   // [groups - 1][2 * cols], or [2 * cols]
  __shared__ float scratch[8][2][2][kNormMaxWarps];
  pdl_begin(dy, x, mean, rstd, w, add);
  const int threads = s.warps * 32, at = (int)threadIdx.x, group = (int)threadIdx.y, groups = (int)blockDim.y;
  float dw[kShared ? 1 : NV][VEC], db[kShared ? 1 : NV][VEC];
  if constexpr (kShared) {
    if (partial)
      for (int c = at; c < 2 * s.cols; c += threads) joined[c] = 0.f;
    __syncthreads();
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  const float inv = 1.f / (float)s.cols;
  int turn = 0;
  for (long long row = (long long)blockIdx.x * groups + group; row < s.rows; row += (long long)gridDim.x * groups) {
    const T* xr = x + row * s.x_ld;
    const T* gr = dy + row * s.dy_ld;
    const float m = mean[row], r = rstd[row];
    float xh[NV][VEC], t[NV][VEC];
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (at + i * threads) * VEC;
      if (c < s.cols) {
        load_f32<T, VEC>(xr + c, xh[i]);
        load_f32<T, VEC>(gr + c, t[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (at + i * threads) * VEC;
      if (c < s.cols) {
        float wv[VEC];
        if (w) load_f32<T, VEC>(w + c, wv);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          xh[i][j] = (xh[i][j] - m) * r;
          if constexpr (kShared) {
            if (partial) {   // this thread's own columns
              joined[c + j] += t[i][j] * xh[i][j];
              joined[s.cols + c + j] += t[i][j];
            }
          } else {
            dw[i][j] += t[i][j] * xh[i][j];
            db[i][j] += t[i][j];
          }
          if (w) t[i][j] *= wv[j];
          sums[0] += t[i][j];
          sums[1] += t[i][j] * xh[i][j];
        }
      }
    }
    group_sum<2>(sums, s.warps, at >> 5, 1 + group, scratch[group][turn][0]);
    turn ^= 1;
    const float c1 = sums[0] * inv, c2 = sums[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (at + i * threads) * VEC;
      if (c < s.cols) {
        float o[VEC];
        if (add) load_f32<T, VEC>(add + row * s.add_ld + c, o);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float g = r * (t[i][j] - c1 - xh[i][j] * c2);
          o[j] = add ? g + o[j] : g;
        }
        store_f32<T, VEC>(dx + row * s.cols + c, o);
      }
    }
  }
  if (!partial) return;
  float* line = partial + (size_t)blockIdx.x * 2 * s.cols;
  if constexpr (kShared) {
    __syncthreads();
    for (int c = at; c < 2 * s.cols; c += threads) line[c] = joined[c];
  } else {
    if (group) {
      float* mine = joined + (size_t)(group - 1) * 2 * s.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            mine[c + j] = dw[i][j];
            mine[s.cols + c + j] = db[i][j];
          }
      }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols)
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            float a = dw[i][j], d = db[i][j];
            for (int g = 1; g < groups; ++g) {
              a += joined[(size_t)(g - 1) * 2 * s.cols + c + j];
              d += joined[(size_t)(g - 1) * 2 * s.cols + s.cols + c + j];
            }
            line[c + j] = a;
            line[s.cols + c + j] = d;
          }
      }
    }
  }
}

// Long rows: dx by one CTA per row in two passes; the column sums by k6_norm_columns_long.
template <typename T>
__global__ void __launch_bounds__(1024) k6_norm_backward_long(const T* dy, const T* x, const float* mean, const float* rstd, const T* w,
                                                              const T* add, T* dx, NormShape s) {
  __shared__ float scratch[2][2][kNormMaxWarps];
  pdl_begin(dy, x, mean, rstd, w, add);
  int turn = 0;
  for (long long row = blockIdx.x; row < s.rows; row += gridDim.x) {
    const T* xr = x + row * s.x_ld;
    const T* gr = dy + row * s.dy_ld;
    const float m = mean[row], r = rstd[row];
    float sums[2] = {0.f, 0.f};
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) {
      const float t = to_f32(gr[c]) * (w ? to_f32(w[c]) : 1.f);
      sums[0] += t;
      sums[1] += t * ((to_f32(xr[c]) - m) * r);
    }
    group_sum<2>(sums, 32, (int)threadIdx.x >> 5, 1, scratch[turn][0]);
    turn ^= 1;
    const float c1 = sums[0] / (float)s.cols, c2 = sums[1] / (float)s.cols;
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) {
      const float t = to_f32(gr[c]) * (w ? to_f32(w[c]) : 1.f);
      float o = r * (t - c1 - ((to_f32(xr[c]) - m) * r) * c2);
      if (add) o += to_f32(add[row * s.add_ld + c]);
      dx[row * s.cols + c] = from_f32<T>(o);
    }
  }
}
template <typename T>
__global__ void __launch_bounds__(256) k6_norm_columns_long(const T* dy, const T* x, const float* mean, const float* rstd, float* partial, NormShape s) {
  pdl_begin(dy, x, mean, rstd);
  const int c = (int)(blockIdx.x * 256 + threadIdx.x);
  if (c >= s.cols) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < s.rows; row += gridDim.y) {
    const float g = to_f32(dy[row * s.dy_ld + c]);
    db += g;
    dw += g * ((to_f32(x[row * s.x_ld + c]) - mean[row]) * rstd[row]);
  }
  partial[(size_t)blockIdx.y * 2 * s.cols + c] = dw;
  partial[(size_t)blockIdx.y * 2 * s.cols + s.cols + c] = db;
}

// ---- host -------------------------------------------------------------------------------------------------------
// How a row is spread over a group: `nv` vectors of `vec` elements per thread.  About 8 elements a thread where that
// needs no more than 8 warps; longer rows take more warps, then more vectors.
struct NormPlan {
  int vec, nv, warps, groups;   // nv 0: the form for long rows
};

inline bool divides(long long bytes, const void* p, long long ld_bytes) {
  return p == nullptr || ((uintptr_t)p % bytes == 0 && ld_bytes % bytes == 0);
}

inline NormPlan norm_plan(int cols, int vec) {
  NormPlan p{vec, 1, 1, 1};
  const int vectors = (cols + vec - 1) / vec;
  const int per = 8 / vec > 0 ? 8 / vec : 1;
  int warps = (vectors + 32 * per - 1) / (32 * per);
  if (warps > 8) warps = 8;
  for (;;) {
    const int need = (vectors + 32 * warps - 1) / (32 * warps);
    const int cap = 16 / vec;   // vectors per thread: 16 elements at most
    if (need <= (cap > 1 ? cap : 1)) {
      p.nv = need;
      break;
    }
    if (warps == 32) {
      p.nv = 0;
      break;
    }
    warps = warps <= 8 ? 16 : 32;
  }
  p.warps = warps;
  int groups = 8 / warps;
  p.groups = groups < 1 ? 1 : groups;
  int nv = 1;
  while (p.nv > nv) nv *= 2;
  p.nv = p.nv ? nv : 0;
  return p;
}

template <typename T, typename F>
bool with_plan(const NormPlan& p, F&& f) {
  constexpr int wide = 16 / sizeof(T);
  auto nv = [&](auto vec) {
    constexpr int V = decltype(vec)::value;
    switch (p.nv) {
      case 1: f(vec, std::integral_constant<int, 1>{}); return true;
      case 2: if constexpr (V * 2 <= 16) { f(vec, std::integral_constant<int, 2>{}); return true; } break;
      case 4: if constexpr (V * 4 <= 16) { f(vec, std::integral_constant<int, 4>{}); return true; } break;
      case 8: if constexpr (V * 8 <= 16) { f(vec, std::integral_constant<int, 8>{}); return true; } break;
      case 16: if constexpr (V * 16 <= 16) { f(vec, std::integral_constant<int, 16>{}); return true; } break;
    }
    return false;
  };
  if (p.vec == wide) return nv(std::integral_constant<int, wide>{});
  if (sizeof(T) == 2 && p.vec == 4) return nv(std::integral_constant<int, 4>{});
  return nv(std::integral_constant<int, 1>{});
}

template <typename T>
int pick_vec(long long cols, std::initializer_list<std::pair<const void*, long long>> bases) {
  for (int vec : {(int)(16 / sizeof(T)), 4, 1}) {
    bool ok = cols % vec == 0;
    for (const auto& b : bases) ok = ok && divides((long long)vec * (long long)sizeof(T), b.first, b.second * (long long)sizeof(T));
    if (ok) return vec;
  }
  return 1;
}

template <typename T>
int norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, NormShape s, cudaStream_t stream) {
  const int vec = pick_vec<T>(s.cols, {{x, s.x_ld}, {w, 0}, {b, 0}, {y, s.cols}});
  NormPlan p = norm_plan(s.cols, vec);
  s.warps = p.warps;
  cudaError_t e = cudaSuccess;
  if (p.nv == 0) {
    const long long grid = s.rows < 65535 ? s.rows : 65535;
    e = launch_pdl(k6_norm_forward_long<T>, dim3((unsigned)grid), dim3(1024), stream, (const T*)x, (const T*)w, (const T*)b, (T*)y, mean, rstd, s);
  } else {
    while (p.groups > 1 && s.rows < 148 * p.groups) p.groups /= 2;   // few rows: one row a CTA spreads them over the SMs
    const long long grid = (s.rows + p.groups - 1) / p.groups;
    if (grid > 0x7fffffffLL) return GTK_ERR_UNSUPPORTED;
    if (!with_plan<T>(p, [&](auto V, auto N) {
          e = launch_pdl(k6_norm_forward<T, decltype(V)::value, decltype(N)::value>, dim3((unsigned)grid), dim3(32 * p.warps, p.groups), stream,
                         (const T*)x, (const T*)w, (const T*)b, (T*)y, mean, rstd, s);
        }))
      return GTK_ERR_UNSUPPORTED;
  }
  gtk_count_launch(1);
  return e == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

constexpr int kNormLines = 148;   // lines of column sums at most

template <typename T>
int norm_backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, const void* add, void* dx, void* dw, void* db,
                  float* partial, NormShape s, cudaStream_t stream) {
  const int vec = pick_vec<T>(s.cols, {{x, s.x_ld}, {dy, s.dy_ld}, {w, 0}, {add, s.add_ld}, {dx, s.cols}});
  NormPlan p = norm_plan(s.cols, vec);
  s.warps = p.warps;
  cudaError_t e = cudaSuccess;
  int lines;
  float* sums = dw || db ? partial : nullptr;
  if (p.nv == 0) {
    const long long grid = s.rows < 65535 ? s.rows : 65535;
    e = launch_pdl(k6_norm_backward_long<T>, dim3((unsigned)grid), dim3(1024), stream, (const T*)dy, (const T*)x, mean, rstd, (const T*)w,
                   (const T*)add, (T*)dx, s);
    gtk_count_launch(1);
    if (e != cudaSuccess) return GTK_ERR_CUDA;
    if (!sums) return GTK_OK;
    lines = s.rows < 16 ? (int)s.rows : 16;
    e = launch_pdl(k6_norm_columns_long<T>, dim3((unsigned)((s.cols + 255) / 256), (unsigned)lines), dim3(256), stream, (const T*)dy, (const T*)x, mean,
                   rstd, sums, s);
  } else {
    const size_t line_bytes = 2 * (size_t)s.cols * 4;
    while (p.groups > 1 && (p.groups - 1) * line_bytes > 32768) p.groups /= 2;
    const bool shared = p.warps > 16;
    const size_t dynamic = !sums ? 0 : shared ? line_bytes : (p.groups - 1) * line_bytes;
    const long long need = (s.rows + p.groups - 1) / p.groups;
    lines = need < kNormLines ? (int)need : kNormLines;
    if (!with_plan<T>(p, [&](auto V, auto N) {
          cudaLaunchConfig_t cfg = {};
          cfg.gridDim = dim3((unsigned)lines);
          cfg.blockDim = dim3(32 * p.warps, p.groups);
          cfg.dynamicSmemBytes = dynamic;
          cfg.stream = stream;
          cudaLaunchAttribute attr[1];
          attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
          attr[0].val.programmaticStreamSerializationAllowed = 1;
          cfg.attrs = attr;
          cfg.numAttrs = 1;
          constexpr int kV = decltype(V)::value, kN = decltype(N)::value;
          auto go = [&](auto kernel) {
            e = cudaLaunchKernelEx(&cfg, kernel, (const T*)dy, (const T*)x, mean, rstd, (const T*)w, (const T*)add, (T*)dx, sums, s);
          };
          if (!shared) {
            go(k6_norm_backward<T, kV, kN, 512>);
          } else if constexpr (kV * kN > 8) {
            e = cudaFuncSetAttribute(k6_norm_backward<T, kV, kN, 1024>, cudaFuncAttributeMaxDynamicSharedMemorySize, 16384 * 8);
            if (e == cudaSuccess) go(k6_norm_backward<T, kV, kN, 1024>);
          } else {
            e = cudaErrorInvalidConfiguration;   // rows for which 17 warps and more are taken give a thread over 8 elements
          }
        }))
      return GTK_ERR_UNSUPPORTED;
    if (!sums) {
      gtk_count_launch(1);
      return e == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
    }
  }
  gtk_count_launch(1);
  if (e != cudaSuccess) return GTK_ERR_CUDA;
  e = launch_col_finish<T>(partial, lines, 2LL * s.cols, s.cols, (T*)dw, (T*)db, stream);
  gtk_count_launch(1);
  return e == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

}  // namespace gtk

using namespace gtk;

// x: rows of `cols` elements, x_ld apart; y dense; w and b may be null.
extern "C" int gtk_k6_norm_forward(int type, const void* x, long long x_ld, const void* w, const void* b, void* y, float* mean, float* rstd, long long rows,
                                   long long cols, float eps, void* stream) {
  if (rows <= 0 || cols <= 0 || cols > 0x3fffffff || x_ld < 0) return GTK_ERR_ARG;
  const NormShape s{rows, x_ld, 0, 0, (int)cols, 1, eps};
  switch (type) {
    case kF32: return norm_forward<float>(x, w, b, y, mean, rstd, s, (cudaStream_t)stream);
    case kF16: return norm_forward<__half>(x, w, b, y, mean, rstd, s, (cudaStream_t)stream);
    case kBF16: return norm_forward<__nv_bfloat16>(x, w, b, y, mean, rstd, s, (cudaStream_t)stream);
  }
  return GTK_ERR_ARG;
}

// Lines of 2 * cols floats that `partial` has to hold.
extern "C" int gtk_k6_norm_lines(void) { return kNormLines; }

// dx dense; add (may be null): a gradient that is added to dx; dw, db may be null.
extern "C" int gtk_k6_norm_backward(int type, const void* dy, long long dy_ld, const void* x, long long x_ld, const float* mean, const float* rstd,
                                    const void* w, const void* add, long long add_ld, void* dx, void* dw, void* db, float* partial, long long rows,
                                    long long cols, void* stream) {
  if (rows <= 0 || cols <= 0 || cols > 0x3fffffff || x_ld < 0 || dy_ld < 0 || add_ld < 0) return GTK_ERR_ARG;
  const NormShape s{rows, x_ld, dy_ld, add_ld, (int)cols, 1, 0.f};
  switch (type) {
    case kF32: return norm_backward<float>(dy, x, mean, rstd, w, add, dx, dw, db, partial, s, (cudaStream_t)stream);
    case kF16: return norm_backward<__half>(dy, x, mean, rstd, w, add, dx, dw, db, partial, s, (cudaStream_t)stream);
    case kBF16: return norm_backward<__nv_bfloat16>(dy, x, mean, rstd, w, add, dx, dw, db, partial, s, (cudaStream_t)stream);
  }
  return GTK_ERR_ARG;
}
