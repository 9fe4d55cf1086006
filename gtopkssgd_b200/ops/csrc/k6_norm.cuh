#pragma once
// K6: layer norm over the last axis, forward and backward.
//
//   mean = sum x / D, rstd = (sum (x - mean)^2 / D + eps)^-1/2, xh = (x - mean) rstd, y = xh w + b
//   t = dy w, dx = rstd (t - mean_D(t) - xh mean_D(t xh)) + add, dw = sum_R dy xh, db = sum_R dy
//
// Bound by memory: the forward pass reads x and writes y, the backward pass reads dy and x and writes dx.  A row is
// read once and stays in registers (the variance is summed over the centred values, not from sums of squares).  A
// group of warps takes a row, 16 elements a thread (8 where rows are few), and goes through rows in turn; the rows to
// come are copied to shared memory meanwhile, every thread its own elements (no thread waits for another's copies).
// With 8 elements a thread the work per thread and row - sums across lanes and warps, addresses - took 37
// instructions an element forward and 70 backward, and their issue, not memory, set the time.  In the backward pass the column sums of
// a thread's own columns stay in its registers all along, the groups of a CTA join theirs in shared memory, and
// col_finish adds up one line per CTA.  16384 x 4096 bf16: forward 72 us (3.7 TB/s, 64 % of the issue slots), backward 122
// (3.3 TB/s, 59 %): instructions for unpacking and addresses still weigh as much as memory.  700 x 1500 f32: 4.6 and 12 us
// with col_finish.
#include <atomic>

#include "colsum.cuh"
#include "common.cuh"
#include "host_api.h"
#include "launch.cuh"

namespace gtk {

constexpr int kNormMaxWarps = 32;

// Sums of N values over the threads of a group of warps.  All groups of the CTA take part at the same time: a barrier
// whose number is known only at run time makes the compiler reserve all 16, and four such CTAs fill an SM.  Scratch:
// N floats a warp on a boundary of 16 bytes, zeros past the last warp up to a multiple of 4; used in turn, so that one
// barrier a sum is enough.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int warps, int warp, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (warps == 1) return;
  if (lane_id() == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) scratch[warp * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  for (int k = 0; k < warps * N; k += 4) {
    const float4 x = *reinterpret_cast<const float4*>(scratch + k);
    v[0] += N == 1 ? (x.x + x.y) + (x.z + x.w) : x.x + x.z;
    if constexpr (N == 2) v[1] += x.y + x.w;
  }
}

struct NormShape {
  long long rows, x_ld, dy_ld, add_ld, y_ld;   // leading dimensions in elements; y_ld: of y, or of the norm's output made again
  int cols;
  int warps;                             // of a group
  int depth;                             // rows of a group under way
  float eps;
};

// A thread's part of a row, as it lies in memory: NV vectors of VEC elements.
template <typename T, int VEC, int NV>
struct RowRaw {
  Vec<T, VEC> v[NV];
};

// The rows to come.  Vectors of less than 4 elements are not copied asynchronously, which costs an instruction each: of
// those rows the next one waits in registers (depth 1).  7553 rows of 893 and 894 f32, forward and backward: 20 and 43, 16
// and 30 us; with asynchronous copies 36 and 99, 20 and 47.
constexpr bool ring_async(int vec) { return vec >= 4; }

template <typename T, int VEC, int NV>
struct RowRing {
  static constexpr int kBytes = VEC * (int)sizeof(T);
  static constexpr bool kAsync = ring_async(VEC);
  uint8_t* mine;      // [depth][NV][threads of the CTA] vectors
  uint32_t stride;    // bytes between the vectors of a thread
  uint32_t slot;      // bytes of a row of all groups
  RowRaw<T, VEC, kAsync ? 1 : NV> held;

  __device__ __forceinline__ RowRing(uint8_t* base, int cta_threads, int thread)
      : mine(base + thread * kBytes), stride((uint32_t)(cta_threads * kBytes)), slot((uint32_t)(NV * cta_threads * kBytes)) {}
  __device__ __forceinline__ void copy(int at, const T* row, int first, int threads, int cols) {
    if constexpr (kAsync) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (first + i * threads) * VEC;
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(mine) + (uint32_t)at * slot + (uint32_t)i * stride;
        if (c < cols) {
          if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(row + c) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(row + c), "n"(kBytes) : "memory");
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (first + i * threads) * VEC;
        if (c < cols) held.v[i] = *reinterpret_cast<const Vec<T, VEC>*>(row + c);
      }
    }
  }
  __device__ __forceinline__ void take(int at, int first, int threads, int cols, RowRaw<T, VEC, NV>* out) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (first + i * threads) * VEC;
      if (c < cols) {
        if constexpr (kAsync) out->v[i] = *reinterpret_cast<const Vec<T, VEC>*>(mine + (size_t)at * slot + (size_t)i * stride);
        else out->v[i] = held.v[i];
      }
    }
  }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void ring_wait(int newer) {   // all but the `newer` last groups have arrived
  switch (newer) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
  }
}
constexpr int kRingDepth = 4;   // at most; ring_wait knows these

// blockDim = (32 * warps, groups).  Dynamic shared memory: `depth` rows of every group.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(1024) k6_norm_forward(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, NormShape s) {
  using V = Wide<VEC>;
  constexpr int kV = VEC * 4 / (int)sizeof(V);   // of V in a vector
  extern __shared__ uint4 dynamic[];
  __shared__ alignas(16) float scratch[8][2][kNormMaxWarps];
  pdl_begin(x, w, b);
  const int threads = s.warps * 32, at = (int)threadIdx.x, group = (int)threadIdx.y;
  for (int i = group * threads + at; i < 8 * 2 * kNormMaxWarps; i += threads * (int)blockDim.y) (&scratch[0][0][0])[i] = 0.f;
  __syncthreads();
  const long long step = (long long)gridDim.x * blockDim.y;
  RowRing<T, VEC, NV> ring(reinterpret_cast<uint8_t*>(dynamic), threads * (int)blockDim.y, group * threads + at);
  long long row = (long long)blockIdx.x * blockDim.y + group;
  const T* coming = x + row * s.x_ld;   // the row to be copied next, and its number
  long long coming_row = row;
  for (int i = 0; i < s.depth; ++i) {
    if (coming_row < s.rows) ring.copy(i, coming, at, threads, s.cols);
    ring_commit();
    coming += step * s.x_ld;
    coming_row += step;
  }
  const float inv = 1.f / (float)s.cols;
  T* yr = y + row * s.y_ld;
  int slot = 0;
  for (long long left = s.rows - (long long)blockIdx.x * blockDim.y; left > 0; left -= step) {   // the whole CTA
    const bool mine = row < s.rows;
    RowRaw<T, VEC, NV> raw;
    ring_wait(s.depth - 1);
    if (mine) ring.take(slot, at, threads, s.cols, &raw);
    float v[NV][VEC];
    V total = vset<V>(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((at + i * threads) * VEC < s.cols) {
        to_f32<T, VEC>(raw.v[i], v[i]);
#pragma unroll
        for (int j = 0; j < kV; ++j) total = vadd(total, vget<V>(v[i], j));
      }
    float sum[1] = {vtotal(total)};
    group_sum<1>(sum, s.warps, at >> 5, scratch[group][0]);
    if (coming_row < s.rows) ring.copy(slot, coming, at, threads, s.cols);
    ring_commit();
    coming += step * s.x_ld;
    coming_row += step;
    slot = slot + 1 == s.depth ? 0 : slot + 1;
    const float m = sum[0] * inv;
    const V minus = vset<V>(-m);
    total = vset<V>(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((at + i * threads) * VEC < s.cols) {
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          const V d = vadd(vget<V>(v[i], j), minus);
          vput(v[i], j, d);
          total = vfma(d, d, total);
        }
      }
    float sq[1] = {vtotal(total)};
    group_sum<1>(sq, s.warps, at >> 5, scratch[group][1]);
    const float r = rsqrtf(fmaf(sq[0], inv, s.eps));
    if (mine) {
      if (at == 0) {
        mean[row] = m;
        rstd[row] = r;
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols) {
          float wv[VEC], bv[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            wv[j] = 1.f;
            bv[j] = 0.f;
          }
          if (w) load_f32<T, VEC>(w + c, wv);
          if (b) load_f32<T, VEC>(b + c, bv);
#pragma unroll
          for (int j = 0; j < kV; ++j) vput(v[i], j, vfma(vmul(vget<V>(v[i], j), vset<V>(r)), vget<V>(wv, j), vget<V>(bv, j)));
          store_f32<T, VEC>(yr + c, v[i]);
        }
      }
    }
    row += step;
    yr += step * s.y_ld;
  }
}

// Rows longer than the registers hold: three passes over the row, the later two from the caches.
template <typename T>
__global__ void __launch_bounds__(1024) k6_norm_forward_long(const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, NormShape s) {
  __shared__ alignas(16) float scratch[2][kNormMaxWarps];
  pdl_begin(x, w, b);
  for (long long row = blockIdx.x; row < s.rows; row += gridDim.x) {
    const T* xr = x + row * s.x_ld;
    float sum[1] = {0.f};
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) sum[0] += to_f32(xr[c]);
    group_sum<1>(sum, 32, (int)threadIdx.x >> 5, scratch[0]);
    const float m = sum[0] / (float)s.cols;
    float sq[1] = {0.f};
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) {
      const float d = to_f32(xr[c]) - m;
      sq[0] += d * d;
    }
    group_sum<1>(sq, 32, (int)threadIdx.x >> 5, scratch[1]);
    const float r = 1.f / sqrtf(sq[0] / (float)s.cols + s.eps);
    if (threadIdx.x == 0) {
      mean[row] = m;
      rstd[row] = r;
    }
    for (int c = (int)threadIdx.x; c < s.cols; c += 1024) {
      float o = (to_f32(xr[c]) - m) * r;
      if (w) o *= to_f32(w[c]);
      if (b) o += to_f32(b[c]);
      y[row * s.y_ld + c] = from_f32<T>(o);
    }
  }
}

// What a backward pass inside a block takes and gives besides: x may come as codes, the norm's output is made again
// from it, and what is added to dx (the gradient of the block's output) is summed over the rows.
template <typename T>
struct NormMore {
  const unsigned char* e;   // exponents of x's codes
  long long e_ld;
  const T* b;
  T* y;
  T* dadd;
};

// partial: [gridDim.x][2 * cols], sums of dy xh, then of dy (MORE: 3 * cols, then of add).  blockDim = (32 * warps, groups).
// Dynamic shared memory: `depth` rows of x, as many of dy, of every group; afterwards the groups' column sums.
// THREADS: the most that it is launched with; with 1024 (rows over 8192 elements) the column sums lie in shared memory
// all along, and rows are loaded when they are used.  A single CTA stores the sums itself.  S: type of x (signed char:
// codes).
template <typename T, typename S, bool MORE, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS)
k6_norm_backward(const T* dy, const S* x, const float* mean, const float* rstd, const T* w, const T* add, T* dx, T* dw_out, T* db_out, float* partial,
                 NormShape s, NormMore<T> more) {
  constexpr bool kShared = THREADS > 512;
  constexpr int kSums = MORE ? 3 : 2;
  using V = Wide<VEC>;
  constexpr int kV = VEC * 4 / (int)sizeof(V);   // of V in a vector
  extern __shared__ uint4 dynamic[];   // then [groups - 1][kSums * cols], or [kSums * cols], of floats
  __shared__ alignas(16) float scratch[8][2][2 * kNormMaxWarps];
  pdl_begin(dy, x, mean, rstd, w, add, more.e, more.b);
  float* joined = reinterpret_cast<float*>(dynamic);
  const int threads = s.warps * 32, at = (int)threadIdx.x, group = (int)threadIdx.y, groups = (int)blockDim.y;
  for (int i = group * threads + at; i < 8 * 2 * 2 * kNormMaxWarps; i += threads * groups) (&scratch[0][0][0])[i] = 0.f;
  RowRing<S, VEC, NV> xs(reinterpret_cast<uint8_t*>(dynamic), threads * groups, group * threads + at);
  RowRing<T, VEC, NV> gs(reinterpret_cast<uint8_t*>(dynamic) + (size_t)s.depth * xs.slot, threads * groups, group * threads + at);
  float sum[kSums][kShared ? 1 : NV][VEC];
  if constexpr (kShared) {
    if (partial)
      for (int c = at; c < kSums * s.cols; c += threads) joined[c] = 0.f;
  } else {
#pragma unroll
    for (int k = 0; k < kSums; ++k)
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum[k][i][j] = 0.f;
  }
  __syncthreads();
  const float inv = 1.f / (float)s.cols;
  const long long step = (long long)gridDim.x * groups;
  long long row = (long long)blockIdx.x * groups + group;
  long long coming = row;   // the row to be copied next
  if constexpr (!kShared)
    for (int i = 0; i < s.depth; ++i) {
      if (coming < s.rows) {
        xs.copy(i, x + coming * s.x_ld, at, threads, s.cols);
        gs.copy(i, dy + coming * s.dy_ld, at, threads, s.cols);
      }
      ring_commit();
      coming += step;
    }
  float nm = 0.f, nr = 0.f;
  unsigned char ne[NV];        // of the row after this one, too
  auto fetch = [&](long long from) {
    nm = mean[from];
    nr = rstd[from];
    if constexpr (sizeof(S) == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols) ne[i] = more.e[from * more.e_ld + c / kBlock8];
      }
    }
  };
  if (row < s.rows) fetch(row);
  int turn = 0, slot = 0;
  for (long long left = s.rows - (long long)blockIdx.x * groups; left > 0; left -= step) {   // the whole CTA
    const bool mine = row < s.rows;
    const float r = nr, minus = -0.5f * nm, twice = 2.f * nr;
    float xh[NV][VEC], t[NV][VEC];
    V sum_t = vset<V>(0.f), sum_th = vset<V>(0.f);
    {
      RowRaw<S, VEC, NV> rx;
      RowRaw<T, VEC, NV> rg;
      if constexpr (kShared) {
        const S* xr = x + row * s.x_ld;
        const T* gr = dy + row * s.dy_ld;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (at + i * threads) * VEC;
          if (c < s.cols && mine) {
            rx.v[i] = *reinterpret_cast<const Vec<S, VEC>*>(xr + c);
            rg.v[i] = *reinterpret_cast<const Vec<T, VEC>*>(gr + c);
          }
        }
      } else {
        ring_wait(s.depth - 1);
        if (mine) {
          xs.take(slot, at, threads, s.cols, &rx);
          gs.take(slot, at, threads, s.cols, &rg);
        }
      }
      if (mine) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int c = (at + i * threads) * VEC;
          if (c < s.cols) {
            float wv[VEC];
            if (w) load_f32<T, VEC>(w + c, wv);
            if constexpr (sizeof(S) == 1) {
              const float scale = block8_scale(ne[i]);
              if constexpr (VEC % 4 == 0) {
#pragma unroll
                for (int j = 0; j < VEC / 4; ++j) block8_values(reinterpret_cast<const uint32_t*>(&rx.v[i])[j], scale, xh[i] + 4 * j);
              } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) xh[i][j] = (float)rx.v[i].v[j] * scale;
              }
            } else {
              to_f32<S, VEC>(rx.v[i], xh[i]);
            }
            to_f32<T, VEC>(rg.v[i], t[i]);
#pragma unroll
            for (int j = 0; j < kV; ++j) {
              // (x - mean) rstd by halves, whose difference f32 always holds.  (One multiply-add of x rstd and mean rstd would
              // leave the rounding of the latter, many times xh where the mean is many deviations.)
              const V h = vmul(vfma(vget<V>(xh[i], j), vset<V>(0.5f), vset<V>(minus)), vset<V>(twice)), g = vget<V>(t[i], j);
              if constexpr (kShared) {
                if (partial) {   // this thread's own columns
                  float* own = joined + c;
                  vput(own, j, vfma(g, h, vget<V>(own, j)));
                  vput(own + s.cols, j, vadd(vget<V>(own + s.cols, j), g));
                }
              } else {
                vput(sum[0][i], j, vfma(g, h, vget<V>(sum[0][i], j)));
                vput(sum[1][i], j, vadd(vget<V>(sum[1][i], j), g));
              }
              const V gw = w ? vmul(g, vget<V>(wv, j)) : g;
              vput(xh[i], j, h);
              vput(t[i], j, gw);
              sum_t = vadd(sum_t, gw);
              sum_th = vfma(gw, h, sum_th);
            }
          }
        }
      }
    }
    float sums[2] = {vtotal(sum_t), vtotal(sum_th)};
    row += step;
    if (row < s.rows) fetch(row);
    group_sum<2>(sums, s.warps, at >> 5, scratch[group][turn]);
    turn ^= 1;
    if constexpr (!kShared) {
      if (coming < s.rows) {
        xs.copy(slot, x + coming * s.x_ld, at, threads, s.cols);
        gs.copy(slot, dy + coming * s.dy_ld, at, threads, s.cols);
      }
      ring_commit();
      coming += step;
      slot = slot + 1 == s.depth ? 0 : slot + 1;
    }
    if (mine) {
      const float c1 = -r * sums[0] * inv, c2 = -r * sums[1] * inv;   // dx = r t + c1 + c2 xh
      const long long now = row - step;
      T* out = dx + now * s.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols) {
          float o[VEC];
          if (add) load_f32<T, VEC>(add + now * s.add_ld + c, o);
          if constexpr (MORE) {
            float wv[VEC], bv[VEC], y[VEC];
            load_f32<T, VEC>(w + c, wv);
            load_f32<T, VEC>(more.b + c, bv);
#pragma unroll
            for (int j = 0; j < kV; ++j) {
              vput(y, j, vfma(vget<V>(xh[i], j), vget<V>(wv, j), vget<V>(bv, j)));
              if constexpr (kShared) {
                float* own = joined + 2 * s.cols + c;
                if (partial) vput(own, j, vadd(vget<V>(own, j), vget<V>(o, j)));
              } else {
                vput(sum[2][i], j, vadd(vget<V>(sum[2][i], j), vget<V>(o, j)));
              }
            }
            store_f32<T, VEC>(more.y + now * s.y_ld + c, y);
          }
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const V g = vfma(vget<V>(t[i], j), vset<V>(r), vfma(vget<V>(xh[i], j), vset<V>(c2), vset<V>(c1)));
            vput(o, j, add ? vadd(g, vget<V>(o, j)) : g);
          }
          store_f32<T, VEC>(out + c, o);
        }
      }
    }
  }
  if (!partial) return;
  float* line = partial + (size_t)blockIdx.x * kSums * s.cols;
  __syncthreads();
  if constexpr (kShared) {
    for (int c = at; c < kSums * s.cols; c += threads) line[c] = joined[c];   // (never a single CTA)
  } else {
    if (group) {
      float* own = joined + (size_t)(group - 1) * kSums * s.cols;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols)
#pragma unroll
          for (int k = 0; k < kSums; ++k) store_f32<float, VEC>(own + k * s.cols + c, sum[k][i]);
      }
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = (at + i * threads) * VEC;
        if (c < s.cols)
#pragma unroll
          for (int k = 0; k < kSums; ++k) {
            for (int g = 0; g + 1 < groups; ++g) {
              float a[VEC];
              load_f32<float, VEC>(joined + (size_t)(g * kSums + k) * s.cols + c, a);
#pragma unroll
              for (int j = 0; j < VEC; ++j) sum[k][i][j] += a[j];
            }
            if (gridDim.x == 1) {
              T* to = k == 0 ? dw_out : k == 1 ? db_out : more.dadd;
#pragma unroll
              for (int j = 0; j < VEC; ++j)   // (no vector: it may lie anywhere)
                if (to) to[c + j] = from_f32<T>(sum[k][i][j]);
            } else {
              store_f32<float, VEC>(line + k * s.cols + c, sum[k][i]);
            }
          }
      }
    }
  }
}

// Long rows: dx by one CTA per row in two passes; the column sums by k6_norm_columns_long.
template <typename T>
__global__ void __launch_bounds__(1024) k6_norm_backward_long(const T* dy, const T* x, const float* mean, const float* rstd, const T* w,
                                                              const T* add, T* dx, NormShape s) {
  __shared__ alignas(16) float scratch[2][2][kNormMaxWarps];
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
    group_sum<2>(sums, 32, (int)threadIdx.x >> 5, scratch[turn][0]);
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
// How a row is spread over a group of `most` warps at most: `nv` vectors of `vec` elements per thread, 8 elements or, where
// there are rows for two groups of every SM and those to come can be copied to shared memory, 16, so that the work per
// thread and row is shared by more elements (32 do not fit the registers: 82 us for 72).  Longer rows take another form
// (nv 0).
struct NormPlan {
  int vec, nv, warps;
};

inline bool divides(long long bytes, const void* p, long long ld_bytes) {
  return p == nullptr || ((uintptr_t)p % bytes == 0 && ld_bytes % bytes == 0);
}

inline NormPlan norm_plan(long long rows, int cols, int vec, bool async, int most) {
  const int vectors = (cols + vec - 1) / vec;
  for (int each = rows >= 296 && async ? 16 : 8; each <= 16; each *= 2) {
    const int warps = (vectors + 32 * (each / vec) - 1) / (32 * (each / vec));
    if (warps <= most) {
      int nv = 1;
      while (nv * 32 * warps < vectors) nv *= 2;
      return NormPlan{vec, nv, warps};
    }
  }
  return NormPlan{vec, 0, 32};
}

// Rows under way: as many as the rest of the shared memory holds.
inline int ring_depth(size_t bytes_a_row, size_t room) {
  const size_t d = room / bytes_a_row;
  return d < 1 ? 1 : d > (size_t)kRingDepth ? kRingDepth : (int)d;
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
  if (p.vec == 2) return nv(std::integral_constant<int, 2>{});
  return nv(std::integral_constant<int, 1>{});
}

template <typename T>
int pick_vec(long long cols, std::initializer_list<std::pair<const void*, long long>> bases) {
  for (int vec : {(int)(16 / sizeof(T)), 4, 2, 1}) {
    bool ok = cols % vec == 0;
    for (const auto& b : bases) ok = ok && divides((long long)vec * (long long)sizeof(T), b.first, b.second * (long long)sizeof(T));
    if (ok) return vec;
  }
  return 1;
}

constexpr int kNormShared = 200 * 1024;   // dynamic shared memory of an SM that the rows under way may take

template <auto Kernel, typename... A>
cudaError_t launch_norm(long long grid, int warps, int groups, size_t shared, cudaStream_t stream, A... args) {
  if (shared > 32 * 1024) {
    static std::atomic<unsigned long long> devices;   // that this kernel has been given its shared memory on
    const DeviceInfo* info = gtk_device_info();
    if (!info) return cudaErrorInvalidDevice;
    const unsigned long long bit = 1ull << info->device;
    if (!(devices.load(std::memory_order_relaxed) & bit)) {
      const cudaError_t err = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormShared);
      if (err != cudaSuccess) return err;
      devices.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(32 * warps, groups);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, Kernel, args...);
}

constexpr int kNormLines = 148;   // lines of column sums at most

// MORE and S: see k6_norm_backward; rows of up to 16384 elements.
template <typename T, typename S, bool MORE>
int norm_backward(const void* dy, const void* x, const float* mean, const float* rstd, const void* w, const void* add, void* dx, void* dw, void* db,
                  float* partial, NormShape s, NormMore<T> more, cudaStream_t stream) {
  int vec = pick_vec<T>(s.cols, {{w, 0}, {dy, s.dy_ld}, {add, s.add_ld}, {dx, s.cols}, {more.b, 0}, {more.y, s.y_ld}});
  while (vec > 1 && !divides((long long)vec * (long long)sizeof(S), x, s.x_ld * (long long)sizeof(S))) vec /= 2;
  const bool async = ring_async(vec);
  NormPlan p = norm_plan(s.rows, s.cols, vec, async, 16);   // 512 threads of 128 registers
  const bool shared = p.nv == 0;
  if (shared) p = norm_plan(296, s.cols, vec, true, 32);
  s.warps = p.warps;
  cudaError_t e = cudaSuccess;
  constexpr int kSums = MORE ? 3 : 2;
  int lines;
  float* sums = dw || db ? partial : nullptr;
  if (p.nv == 0) {
    if constexpr (MORE) {
      return GTK_ERR_UNSUPPORTED;
    } else {
      const long long grid = s.rows < 65535 ? s.rows : 65535;
      e = launch_pdl(k6_norm_backward_long<T>, dim3((unsigned)grid), dim3(1024), stream, (const T*)dy, (const T*)x, mean, rstd, (const T*)w,
                     (const T*)add, (T*)dx, s);
      gtk_count_launch(1);
      if (e != cudaSuccess) return GTK_ERR_CUDA;
      if (!sums) return GTK_OK;
      lines = s.rows < 16 ? (int)s.rows : 16;
      e = launch_pdl(k6_norm_columns_long<T>, dim3((unsigned)((s.cols + 255) / 256), (unsigned)lines), dim3(256), stream, (const T*)dy, (const T*)x,
                     mean, rstd, sums, s);
    }
  } else {
    const size_t line_bytes = kSums * (size_t)s.cols * 4;
    int groups = shared ? 1 : 16 / p.warps > 8 ? 8 : 16 / p.warps;
    // One CTA takes up to four rows a group: 1.4 us each, of which all but one are more than with a CTA a row, against a
    // launch less (2.5 us on the device, 2.6 of host time)
    const bool one = sums && !shared && s.rows <= 4LL * groups;
    while (!one && groups > 1 && s.rows < 148LL * groups) --groups;
    const size_t slot = (size_t)groups * p.warps * 32 * p.nv * p.vec * (sizeof(T) + sizeof(S));   // of x and dy
    const long long need = (s.rows + groups - 1) / groups;
    lines = one ? 1 : need < 2 ? 2 : need < kNormLines ? (int)need : kNormLines;
    s.depth = ring_depth(slot, kNormShared);
    while (s.depth > 1 && ((long long)(s.depth - 1) * lines >= need || !async)) --s.depth;
    size_t dynamic = shared ? 0 : slot * s.depth;
    const size_t join = !sums ? 0 : shared ? line_bytes : (groups - 1) * line_bytes;
    dynamic = dynamic > join ? dynamic : join;
    if (!with_plan<T>(p, [&](auto V, auto N) {
          constexpr int kV = decltype(V)::value, kN = decltype(N)::value;
          auto go = [&](auto threads) {
            e = launch_norm<k6_norm_backward<T, S, MORE, kV, kN, decltype(threads)::value>>(lines, p.warps, groups, dynamic, stream, (const T*)dy, (const S*)x,
                                                                                            mean, rstd, (const T*)w, (const T*)add, (T*)dx, (T*)dw, (T*)db,
                                                                                            sums, s, more);
          };
          if (!shared) go(std::integral_constant<int, 512>{});
          else if constexpr (kV * kN == 16) go(std::integral_constant<int, 1024>{});   // over 8192 elements of 32 warps
          else e = cudaErrorInvalidConfiguration;
        }))
      return GTK_ERR_UNSUPPORTED;
    if (!sums || lines == 1) {
      gtk_count_launch(1);
      return e == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
    }
  }
  gtk_count_launch(1);
  if (e != cudaSuccess) return GTK_ERR_CUDA;
  e = launch_col_finish<T>(partial, lines, (long long)kSums * s.cols, s.cols, (T*)dw, (T*)db, more.dadd, stream);
  gtk_count_launch(1);
  return e == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

// x and what else a block's backward pass needs: k6_norm_block.cu has it for the three types.
template <typename T>
int norm_backward_block(bool codes, const void* dy, const void* x, const float* mean, const float* rstd, const void* w, const void* add, void* dx, void* dw,
                        void* db, float* partial, NormShape s, NormMore<T> more, cudaStream_t stream);

}  // namespace gtk
