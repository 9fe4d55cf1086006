// K7: element-wise passes over a matrix of activations.
//
//   k7_keep          x -> 8-bit codes and one exponent byte per 32 columns of a row (the format is in ff_math.cuh)
//   k7_restore       a matrix, in 8 bits or in its own type, restored, or with the norm applied again
//   k7_pack          matrices -> operands of a matrix product
//   k7_act_backward  dz = dy act'(z) and the sums of dz over the rows (the bias's gradient)
//
// Bound by memory.  A warp takes 32 * VEC neighbouring columns of a row, so that a block of 32 lies in 32 / VEC
// neighbouring lanes and its maximum takes log2(32 / VEC) shuffles; eight warps of a CTA take rows in turn.  16384 x 8192
// bf16 (a copy: 6.5 TB/s): keep 69 us (5.8 TB/s), restore 79 (5.1), act_backward from 8 bits 139 (4.8; the activation's
// instructions, 61 % of the issue slots), from bf16 142 (5.7), the sums alone 45 (6.0).
#include "colsum.cuh"
#include "common.cuh"
#include "host_api.h"
#include "launch.cuh"

namespace gtk {

constexpr int kRowWarps = 8;   // warps of a CTA, each with rows of its own

template <typename T, int VEC>
__global__ void __launch_bounds__(256) k7_keep(const T* x, long long x_ld, signed char* q, long long q_ld, unsigned char* e, long long e_ld, long long rows,
                                               int cols, int rows_per_warp) {
  pdl_begin(x);
  const int c = (int)((blockIdx.x * 32 + threadIdx.x) * VEC);
  const int padded = (cols + kBlock8 - 1) / kBlock8 * kBlock8;
  const long long first = ((long long)blockIdx.y * kRowWarps + threadIdx.y) * rows_per_warp;
  for (int i = 0; i < rows_per_warp; ++i) {
    const long long row = first + i;
    if (row >= rows) break;   // the whole warp
    float v[VEC];
    if (c < cols) {
      load_f32<T, VEC>(x + row * x_ld + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    }
    float largest = fabsf(v[0]);
    if constexpr (VEC > 1) {
#pragma unroll
      for (int j = 0; j < VEC; j += 2) largest = max_abs(largest, v[j], v[j + 1]);
    }
    uint32_t most = __float_as_uint(largest);
#pragma unroll
    for (int o = kBlock8 / VEC / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const uint32_t byte = block8_byte(most);
    if (c < padded) {
      if constexpr (VEC % 4 == 0) {
        Vec<uint32_t, VEC / 4> codes;
        if (byte < kBlock8Last) {
          const float inverse = block8_inverse(byte);
#pragma unroll
          for (int j = 0; j < VEC / 4; ++j) codes.v[j] = block8_codes(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3], inverse);
        } else {
#pragma unroll
          for (int j = 0; j < VEC / 4; ++j) {
            codes.v[j] = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) codes.v[j] |= ((uint32_t)block8_code(v[4 * j + k], byte) & 255u) << (8 * k);
          }
        }
        *reinterpret_cast<Vec<uint32_t, VEC / 4>*>(q + row * q_ld + c) = codes;
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) q[row * q_ld + c + j] = (signed char)block8_code(v[j], byte);
      }
      if (c % kBlock8 == 0) e[row * e_ld + c / kBlock8] = (unsigned char)byte;
    }
  }
}

// Where an element comes from: a matrix of S, or codes with exponents (S = signed char).
struct Source {
  const void* p;
  long long ld;
  const unsigned char* e;
  long long e_ld;
};
template <typename S, int VEC>
__device__ __forceinline__ void load_source(const Source& s, long long row, int c, float (&v)[VEC]) {
  if constexpr (sizeof(S) == 1) {
    const float scale = block8_scale(s.e[row * s.e_ld + c / kBlock8]);
    const signed char* p = (const signed char*)s.p + row * s.ld + c;
    if constexpr (VEC % 4 == 0) {
      const Vec<uint32_t, VEC / 4> w = *reinterpret_cast<const Vec<uint32_t, VEC / 4>*>(p);
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) block8_values(w.v[j], scale, v + 4 * j);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = (float)p[j] * scale;
    }
  } else {
    load_f32<S, VEC>((const S*)s.p + row * s.ld + c, v);
  }
}

// Codes of f16 values may stand for 65536, up to half a step above what was kept.
template <int VEC>
__device__ __forceinline__ void hold_f16(float (&v)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j)
    if (fabsf(v[j]) > 65504.f) v[j] = copysignf(65504.f, v[j]);
}

// What is done to it: (v - mean) rstd g + b where mean is given.
template <typename T>
struct Apply {
  const float* mean;
  const float* rstd;
  const T* g;
  const T* b;
};

template <typename S, typename T, int VEC>
__global__ void __launch_bounds__(256) k7_restore(Source src, Apply<T> f, T* out, long long out_ld, long long rows, int cols, int rows_per_warp) {
  pdl_begin(src.p, src.e, f.mean, f.rstd, f.g, f.b);
  const int c = (int)((blockIdx.x * 32 + threadIdx.x) * VEC);
  if (c >= cols) return;
  const long long first = ((long long)blockIdx.y * kRowWarps + threadIdx.y) * rows_per_warp;
  for (int i = 0; i < rows_per_warp; ++i) {
    const long long row = first + i;
    if (row >= rows) return;
    float v[VEC];
    load_source<S, VEC>(src, row, c, v);
    if constexpr (sizeof(S) == 1 && std::is_same_v<T, __half>) hold_f16<VEC>(v);
    if (f.mean) {
      const float m = f.mean[row], r = f.rstd[row];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[j] = (v[j] - m) * r;
        if (f.g) v[j] *= to_f32(f.g[c + j]);
        if (f.b) v[j] += to_f32(f.b[c + j]);
      }
    }
    store_f32<T, VEC>(out + row * out_ld + c, v);
  }
}

// Matrices that are made operands of a matrix product by one launch: up to four, CTAs in the order of the matrices.
// Rows get a pitch of a multiple of 8 elements, zeros behind the columns.
enum PackKind : int { kPackPieces = 0, kPackCopy = 1, kPackCodesF16 = 2, kPackCodesBF16 = 3, kPackPairsOfRows = 4, kPackPairsOfColumns = 5 };
struct PackItem {
  Source src;
  void* out;
  long long rows;
  int cols, pitch, kind, step, per;   // step: elements of a load (8, 4 or 1)
  unsigned strips, first;      // strips of columns; the matrix's first CTA
  unsigned int* most;          // pairs: the largest magnitudes (bits) of the rows (written) or of the columns (read)
};
constexpr int kPackItems = 4;
struct PackList {
  PackItem item[kPackItems];
  int count;
};

// VEC elements of a row from column c on, zeros past its end, by loads of STEP: the row's columns are whole STEPs on their
// boundaries.  An odd row costs narrow loads, but its stores stay wide (515 x 1001 and 2047 x 1001 of f16: 6.4 us, 13.4
// with both element by element).
template <int STEP, typename T, int VEC>
__device__ __forceinline__ void load_row(const T* row, int c, int cols, Vec<T, VEC>* v) {
#pragma unroll
  for (int j = 0; j < VEC; j += STEP) {
    Vec<T, STEP> part = {};
    if (c + j < cols) part = *reinterpret_cast<const Vec<T, STEP>*>(row + c + j);
#pragma unroll
    for (int k = 0; k < STEP; ++k) v->v[j + k] = part.v[k];
  }
}

template <int KIND, int VEC, int STEP>
__device__ __forceinline__ void pack_rows(const PackItem& p, unsigned block) {
  const int c = (int)((block % p.strips * 32 + threadIdx.x) * VEC);
  if (c >= p.pitch) return;
  const long long first = ((long long)(block / p.strips) * kRowWarps + threadIdx.y) * p.per, stride = p.rows * p.pitch;
  for (int i = 0; i < p.per; ++i) {
    const long long row = first + i;
    if (row >= p.rows) return;
    const long long to = row * p.pitch + c;
    if constexpr (KIND == kPackCopy) {
      Vec<uint16_t, VEC> v;
      load_row<STEP>((const uint16_t*)p.src.p + row * p.src.ld, c, p.cols, &v);
      *reinterpret_cast<Vec<uint16_t, VEC>*>((uint16_t*)p.out + to) = v;
    } else if constexpr (KIND == kPackPieces) {
      Vec<float, VEC> v;
      load_row<STEP>((const float*)p.src.p + row * p.src.ld, c, p.cols, &v);
      float piece[3][VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        __nv_bfloat16 b[3];
        split3(v.v[j], b);
#pragma unroll
        for (int k = 0; k < 3; ++k) piece[k][j] = __bfloat162float(b[k]);
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) store_f32<__nv_bfloat16, VEC>((__nv_bfloat16*)p.out + k * stride + to, piece[k]);
    } else {
      Vec<signed char, VEC> q;
      load_row<STEP>((const signed char*)p.src.p + row * p.src.ld, c, p.cols, &q);
      const float scale = c < p.cols ? block8_scale(p.src.e[row * p.src.e_ld + c / kBlock8]) : 0.f;
      float v[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = c + j < p.cols ? (float)q.v[j] * scale : 0.f;   // (a NaN's scale stays inside)
      if constexpr (KIND == kPackCodesF16) {
        hold_f16<VEC>(v);
        store_f32<__half, VEC>((__half*)p.out + to, v);
      } else {
        store_f32<__nv_bfloat16, VEC>((__nv_bfloat16*)p.out + to, v);
      }
    }
  }
}

// Two f16 pieces of scaled f32 values.  A NaN or an infinity is all in the first, which has its value's sign and is zero only
// where it is (a scaled value too small for that is the smallest number in the first piece and less than nothing in the
// second).  Beside an infinity, where nothing is scaled, the others count by their signs alone and stop at f16's largest.
template <int VEC>
__device__ __forceinline__ void store_pairs(__half* out, long long stride, const Vec<float, VEC>& v, const float (&scale)[VEC]) {
  float high[VEC], low[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const float f = v.v[j], x = f * scale[j];
    float first = __half2float(__float2half_rn(x));
    if (isinf(first) && !isinf(f)) first = copysignf(65504.f, f);
    if (first == 0.f && f != 0.f) first = copysignf(5.9604644775390625e-8f, f);   // 2^-24
    high[j] = first;
    low[j] = fabsf(x) <= 65504.f ? x - first : 0.f;
  }
  store_f32<__half, VEC>(out, high);
  store_f32<__half, VEC>(out + stride, low);
}

// Loads of a thread in flight: one of 16 bytes does not cover the memory's latency.
constexpr int kLoads = 4;
constexpr int kWarpRow = 2048;

// Rows scaled by their own largest magnitude: a warp takes a row of up to kWarpRow columns (strips 1: eight rows a CTA),
// the CTA's eight warps one of more; the row's second reading comes from the caches.  10000 + 700 rows of 1500: 23 us
// (64 MB read and as many written, 5.5 TB/s); with a load at a time and a CTA to each row 38 us.
template <int STEP>
__device__ __forceinline__ void pack_pairs_of_rows(const PackItem& p, unsigned block, unsigned int* room) {
  constexpr int VEC = 4;
  const bool shared = p.strips != 1;
  const long long row = shared ? block : (long long)block * kRowWarps + threadIdx.y, stride = p.rows * p.pitch;
  const int first = (int)((shared ? threadIdx.y * 32 + threadIdx.x : threadIdx.x) * VEC), step = (shared ? 256 : 32) * VEC;
  if (row >= p.rows) return;   // the whole warp, or the whole CTA
  const float* x = (const float*)p.src.p + row * p.src.ld;
  unsigned int most = 0;
  for (int c = first; c < p.cols; c += step * kLoads) {
    Vec<float, VEC> v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) load_row<STEP>(x, c + k * step, p.cols, &v[k]);
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) most = max(most, __float_as_uint(v[k].v[j]) & 0x7fffffffu);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (shared) {
    if (threadIdx.x == 0) room[threadIdx.y] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kRowWarps; ++k) most = max(most, room[k]);
  }
  if (first == 0) p.most[row] = most;
  float scale[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) scale[j] = __uint_as_float((uint32_t)(pair_shift(most) + 127) << 23);
  __half* out = (__half*)p.out + row * p.pitch;
  for (int c = first; c < p.pitch; c += step * kLoads) {
    Vec<float, VEC> v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) load_row<STEP>(x, c + k * step, p.cols, &v[k]);
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (c + k * step < p.pitch) store_pairs<VEC>(out + c + k * step, stride, v[k], scale);
  }
}

template <int STEP>
__device__ __forceinline__ void pack_pairs_of_columns(const PackItem& p, unsigned block) {
  constexpr int VEC = 4;
  const int c = (int)((block % p.strips * 32 + threadIdx.x) * VEC);
  if (c >= p.pitch) return;
  const long long first = ((long long)(block / p.strips) * kRowWarps + threadIdx.y) * p.per, stride = p.rows * p.pitch;
  float scale[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) scale[j] = c + j < p.cols ? __uint_as_float((uint32_t)(pair_shift(p.most[c + j]) + 127) << 23) : 0.f;
  const int rows = (int)max(min(p.rows - first, (long long)p.per), 0ll);
  const float* x = (const float*)p.src.p + first * p.src.ld;
  __half* out = (__half*)p.out + first * p.pitch + c;
  int i = 0;
  for (; i + kLoads <= rows; i += kLoads) {
    Vec<float, VEC> v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) load_row<STEP>(x + (i + k) * p.src.ld, c, p.cols, &v[k]);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) store_pairs<VEC>(out + (i + k) * (long long)p.pitch, stride, v[k], scale);
  }
  for (; i < rows; ++i) {
    Vec<float, VEC> v;
    load_row<STEP>(x + i * p.src.ld, c, p.cols, &v);
    store_pairs<VEC>(out + i * (long long)p.pitch, stride, v, scale);
  }
}

// The largest magnitudes of the columns of the list's kPackPairsOfColumns matrices, by atomic maxima over zeros: whatever
// their order, the result is the same.
template <int STEP>
__device__ __forceinline__ void column_most(const PackItem& p, unsigned block, unsigned int (*room)[32 * 4]) {
  constexpr int VEC = 4;
  const int c = (int)((block % p.strips * 32 + threadIdx.x) * VEC);
  const long long first = ((long long)(block / p.strips) * kRowWarps + threadIdx.y) * p.per;
  unsigned int most[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) most[j] = 0;
  const int rows = c < p.cols ? (int)max(min(p.rows - first, (long long)p.per), 0ll) : 0;
  const float* x = (const float*)p.src.p + first * p.src.ld;
  auto look = [&](const Vec<float, VEC>& v) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) most[j] = max(most[j], __float_as_uint(v.v[j]) & 0x7fffffffu);
  };
  int i = 0;
  for (; i + kLoads <= rows; i += kLoads) {
    Vec<float, VEC> v[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) load_row<STEP>(x + (i + k) * p.src.ld, c, p.cols, &v[k]);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) look(v[k]);
  }
  for (; i < rows; ++i) {
    Vec<float, VEC> v;
    load_row<STEP>(x + i * p.src.ld, c, p.cols, &v);
    look(v);
  }
#pragma unroll
  for (int j = 0; j < VEC; ++j) room[threadIdx.y][threadIdx.x * VEC + j] = most[j];
  __syncthreads();
  for (int i = (int)(threadIdx.y * 32 + threadIdx.x); i < 32 * VEC; i += 256) {
    const int col = (int)(block % p.strips * 32 * VEC) + i;
    if (col >= p.cols) break;
    unsigned int m = 0;
#pragma unroll
    for (int k = 0; k < kRowWarps; ++k) m = max(m, room[k][i]);
    if (m) atomicMax(p.most + col, m);
  }
}
__global__ void __launch_bounds__(256) k7_column_most(const __grid_constant__ PackList list) {
  __shared__ unsigned int room[kRowWarps][32 * 4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int k = 0;
  while (k + 1 < list.count && blockIdx.x >= list.item[k + 1].first) ++k;
  const PackItem& p = list.item[k];
  if (p.step == 4) column_most<4>(p, blockIdx.x - p.first, room);
  else column_most<1>(p, blockIdx.x - p.first, room);
}

template <int KIND>
__device__ __forceinline__ void pack_of(const PackItem& p, unsigned block) {
  constexpr int VEC = KIND == kPackPieces ? 4 : 8;   // of the pitch, a multiple of 8
  if (p.step == VEC) pack_rows<KIND, VEC, VEC>(p, block);
  else if (p.step == 4) pack_rows<KIND, VEC, 4>(p, block);
  else pack_rows<KIND, VEC, 1>(p, block);
}

__global__ void __launch_bounds__(256) k7_pack(const __grid_constant__ PackList list) {
  __shared__ unsigned int room[kRowWarps];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int k = 0;
  while (k + 1 < list.count && blockIdx.x >= list.item[k + 1].first) ++k;
  const PackItem& p = list.item[k];
  const unsigned block = blockIdx.x - p.first;
  switch (p.kind) {
    case kPackPieces: pack_of<kPackPieces>(p, block); break;
    case kPackCopy: pack_of<kPackCopy>(p, block); break;
    case kPackCodesF16: pack_of<kPackCodesF16>(p, block); break;
    case kPackPairsOfRows:
      if (p.step == 4) pack_pairs_of_rows<4>(p, block, room);
      else pack_pairs_of_rows<1>(p, block, room);
      break;
    case kPackPairsOfColumns:
      if (p.step == 4) pack_pairs_of_columns<4>(p, block);
      else pack_pairs_of_columns<1>(p, block);
      break;
    default: pack_of<kPackCodesBF16>(p, block); break;
  }
}

template <int BYTES>
__device__ __forceinline__ void async_copy(void* to, const void* from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES; i += 16)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i), "l"(reinterpret_cast<const uint8_t*>(from) + i) : "memory");
  } else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}

// Z: element type of z (signed char: codes).  dz may be null (sums only); partial and db may be null.  With one line of
// partial sums they are the sums, and are stored as such.
// One wave of CTAs, four an SM, whose threads each have four rows under way: with a row at a time, loaded to registers,
// 24 KB an SM were under way and a pass over 16384 x 8192 took 152 us instead of 140.
template <typename T, typename Z, int VEC>
__global__ void __launch_bounds__(256, 4) k7_act_backward(const T* dy, long long dy_ld, Source z, int act, T* dz, long long dz_ld, T* db, float* partial,
                                                       long long rows, int cols) {
  __shared__ float joined[kRowWarps][32 * VEC];
  pdl_begin(dy, z.p, z.e);
  const int c = (int)((blockIdx.x * 32 + threadIdx.x) * VEC);
  float sum[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sum[j] = 0.f;
  const long long step = (long long)gridDim.y * kRowWarps, row0 = (long long)blockIdx.y * kRowWarps + threadIdx.y;
  // Rows to come: each thread's own part in shared memory (vectors of less than 4 bytes, of which there are no
  // asynchronous copies, are loaded when they are used)
  constexpr int kBytes = VEC * (int)sizeof(T), kBytesZ = VEC * (int)sizeof(Z);
  constexpr bool kAsync = kBytes >= 4 && kBytesZ >= 4;
  constexpr int kActDepth = VEC == 16 ? 2 : 4;   // rows of a thread under way
  __shared__ alignas(16) uint8_t ring[kAsync ? kActDepth : 1][256][kBytes], ring_z[kAsync ? kActDepth : 1][256][kBytesZ];
  const int t = (int)(threadIdx.y * 32 + threadIdx.x);
  auto copy = [&](int slot, long long row) {
    if constexpr (kAsync) {
      if (c < cols && row < rows) {
        async_copy<kBytes>(ring[slot][t], dy + row * dy_ld + c);
        if (act != kActNone) {
          async_copy<kBytesZ>(ring_z[slot][t], (const Z*)z.p + row * z.ld + c);
          if (sizeof(Z) == 1) asm volatile("prefetch.global.L2 [%0];" ::"l"(z.e + row * z.e_ld + c / kBlock8) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  if constexpr (kAsync) {
#pragma unroll
    for (int i = 0; i < kActDepth; ++i) copy(i, row0 + i * step);
  }
  int slot = 0;
  for (long long row = row0; row < rows; row += step) {
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(kActDepth - 1) : "memory");
    if (c < cols) {
      float g[VEC];
      if constexpr (kAsync) to_f32<T, VEC>(*reinterpret_cast<const Vec<T, VEC>*>(ring[slot][t]), g);
      else load_f32<T, VEC>(dy + row * dy_ld + c, g);
      if (act != kActNone) {
        float zv[VEC];
        if constexpr (!kAsync) {
          load_source<Z, VEC>(z, row, c, zv);
        } else if constexpr (sizeof(Z) == 1) {
          const float scale = block8_scale(z.e[row * z.e_ld + c / kBlock8]);
          const Vec<uint32_t, VEC / 4> q = *reinterpret_cast<const Vec<uint32_t, VEC / 4>*>(ring_z[slot][t]);
#pragma unroll
          for (int j = 0; j < VEC / 4; ++j) block8_values(q.v[j], scale, zv + 4 * j);
        } else {
          to_f32<Z, VEC>(*reinterpret_cast<const Vec<Z, VEC>*>(ring_z[slot][t]), zv);
        }
        with_act(act, [&](auto A) { act_slopes<decltype(A)::value, VEC>(g, zv); });
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[j] += g[j];
      if (dz) store_f32<T, VEC>(dz + row * dz_ld + c, g);
    }
    copy(slot, row + kActDepth * step);   // what was there has been used
    slot = slot + 1 == kActDepth ? 0 : slot + 1;
  }
  if (!partial) return;
#pragma unroll
  for (int j = 0; j < VEC; ++j) joined[threadIdx.y][threadIdx.x * VEC + j] = sum[j];
  __syncthreads();
  for (int i = t; i < 32 * VEC; i += 256) {
    const int col = (int)(blockIdx.x * 32 * VEC) + i;
    if (col >= cols) break;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kRowWarps; ++k) s += joined[k][i];
    if (gridDim.y == 1) db[col] = from_f32<T>(s);
    else partial[(size_t)blockIdx.y * cols + col] = s;
  }
}

// ---- host -------------------------------------------------------------------------------------------------------
inline bool aligned(const void* p, long long ld, int elem, int vec) {
  return (uintptr_t)p % ((uintptr_t)elem * vec) == 0 && (ld * elem) % ((long long)elem * vec) == 0;
}

// Rows that a warp takes, so that the grid is a few CTAs an SM at least and its y fits.
inline bool row_grid(long long rows, unsigned strips, int* per_warp, unsigned* y) {
  long long per = rows * strips / (kRowWarps * 148LL * 8);
  per = per < 1 ? 1 : per > 8 ? 8 : per;
  while ((rows + kRowWarps * per - 1) / (kRowWarps * per) > 65535) per *= 2;
  if (per > 0x3fffffff) return false;
  *per_warp = (int)per;
  *y = (unsigned)((rows + kRowWarps * per - 1) / (kRowWarps * per));
  return true;
}

template <typename T>
int keep(const void* x, long long x_ld, signed char* q, long long q_ld, unsigned char* e, long long e_ld, long long rows, int cols, cudaStream_t stream) {
  auto go = [&](auto V) -> int {
    constexpr int VEC = decltype(V)::value;
    const int padded = (cols + kBlock8 - 1) / kBlock8 * kBlock8;
    const unsigned strips = (unsigned)((padded + 32 * VEC - 1) / (32 * VEC));
    int per;
    unsigned y;
    if (!row_grid(rows, strips, &per, &y)) return GTK_ERR_UNSUPPORTED;
    const cudaError_t err = launch_pdl(k7_keep<T, VEC>, dim3(strips, y), dim3(32, kRowWarps), stream, (const T*)x, x_ld, q, q_ld, e, e_ld, rows, cols, per);
    gtk_count_launch(1);
    return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
  };
  constexpr int wide = 16 / sizeof(T);
  const bool q_ok = aligned(q, q_ld, 1, wide);
  if (cols % wide == 0 && aligned(x, x_ld, sizeof(T), wide) && q_ok) return go(std::integral_constant<int, wide>{});
  if (cols % 4 == 0 && aligned(x, x_ld, sizeof(T), 4) && aligned(q, q_ld, 1, 4)) return go(std::integral_constant<int, 4>{});
  return go(std::integral_constant<int, 1>{});
}

template <typename S, typename T>
int restore(Source src, Apply<T> f, void* out, long long out_ld, long long rows, int cols, cudaStream_t stream) {
  auto go = [&](auto V) -> int {
    constexpr int VEC = decltype(V)::value;
    const unsigned strips = (unsigned)((cols + 32 * VEC - 1) / (32 * VEC));
    int per;
    unsigned y;
    if (!row_grid(rows, strips, &per, &y)) return GTK_ERR_UNSUPPORTED;
    const cudaError_t err = launch_pdl(k7_restore<S, T, VEC>, dim3(strips, y), dim3(32, kRowWarps), stream, src, f, (T*)out, out_ld, rows, cols, per);
    gtk_count_launch(1);
    return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
  };
  // a block's scale is read once per vector, so vectors do not cross blocks (they start at multiples of their length)
  constexpr int wide = sizeof(T) == 4 ? 4 : sizeof(S) == 1 ? 16 : 8;   // more elements a thread: fewer addresses
  auto fits = [&](int vec) {
    const int most = vec < 16 / (int)sizeof(T) ? vec : 16 / (int)sizeof(T);   // 16 bytes at a time
    return cols % vec == 0 && aligned(src.p, src.ld, sizeof(S), vec < 16 / (int)sizeof(S) ? vec : 16 / (int)sizeof(S)) && aligned(out, out_ld, sizeof(T), most);
  };
  if (fits(wide)) return go(std::integral_constant<int, wide>{});
  if constexpr (wide == 16) {
    if (fits(8)) return go(std::integral_constant<int, 8>{});
  }
  if constexpr (wide > 4) {
    if (fits(4)) return go(std::integral_constant<int, 4>{});
  }
  return go(std::integral_constant<int, 1>{});
}

template <typename T, typename Z>
int act_backward(const void* dy, long long dy_ld, Source z, int act, void* dz, long long dz_ld, void* db, float* partial, int max_lines, long long rows,
                 int cols, cudaStream_t stream) {
  unsigned lines = 0;
  auto go = [&](auto V) {
    constexpr int VEC = decltype(V)::value;
    const unsigned strips = (unsigned)((cols + 32 * VEC - 1) / (32 * VEC));
    long long y = 148LL * 4 / strips;
    if (y < 1) y = 1;
    const long long most = (rows + kRowWarps - 1) / kRowWarps;
    if (y > most) y = most;
    if (y > max_lines) y = max_lines;
    if (db && rows <= 8 * kRowWarps) y = 1;   // eight rows a warp: less than the launch that adds lines up
    lines = (unsigned)y;
    return launch_pdl(k7_act_backward<T, Z, VEC>, dim3(strips, lines), dim3(32, kRowWarps), stream, (const T*)dy, dy_ld, z, act, (T*)dz, dz_ld, (T*)db,
                      db ? partial : (float*)nullptr, rows, cols);
  };
  auto fits = [&](int vec) {
    const int most = vec < 16 / (int)sizeof(T) ? vec : 16 / (int)sizeof(T);   // 16 bytes at a time
    return cols % vec == 0 && aligned(dy, dy_ld, sizeof(T), most) && (act == kActNone || aligned(z.p, z.ld, sizeof(Z), vec)) &&
           (!dz || aligned(dz, dz_ld, sizeof(T), most));
  };
  constexpr int wide = sizeof(T) == 2 && sizeof(Z) == 1 ? 16 : 16 / sizeof(T);
  cudaError_t err;
  if (fits(wide)) {
    err = go(std::integral_constant<int, wide>{});
  } else if (wide > 8 && fits(8)) {
    err = go(std::integral_constant<int, (wide == 16 ? 8 : 1)>{});
  } else if (wide > 4 && fits(4)) {
    err = go(std::integral_constant<int, (wide > 4 ? 4 : 1)>{});
  } else {
    err = go(std::integral_constant<int, 1>{});
  }
  gtk_count_launch(1);
  if (err != cudaSuccess) return GTK_ERR_CUDA;
  if (!db || lines == 1) return GTK_OK;
  err = launch_col_finish<T>(partial, (int)lines, cols, cols, (T*)db, (T*)nullptr, (T*)nullptr, stream);
  gtk_count_launch(1);
  return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

constexpr int kActLines = 148;

}  // namespace gtk

using namespace gtk;

// Codes of a matrix: q has q_ld >= cols rounded up to 32 (the rest of the last block is written as zeros).
extern "C" int gtk_k7_keep(int type, const void* x, long long x_ld, signed char* q, long long q_ld, unsigned char* e, long long e_ld, long long rows,
                           long long cols, void* stream) {
  if (rows <= 0 || cols <= 0 || cols > 0x3fffffff || x_ld < 0 || q_ld < (cols + kBlock8 - 1) / kBlock8 * kBlock8 || e_ld < (cols + kBlock8 - 1) / kBlock8)
    return GTK_ERR_ARG;
  switch (type) {
    case kF32: return keep<float>(x, x_ld, q, q_ld, e, e_ld, rows, (int)cols, (cudaStream_t)stream);
    case kF16: return keep<__half>(x, x_ld, q, q_ld, e, e_ld, rows, (int)cols, (cudaStream_t)stream);
    case kBF16: return keep<__nv_bfloat16>(x, x_ld, q, q_ld, e, e_ld, rows, (int)cols, (cudaStream_t)stream);
  }
  return GTK_ERR_ARG;
}

// The matrix src (of `type`, or 8-bit codes where e is given), normalised again where mean is given, -> out, of `type`.
extern "C" int gtk_k7_restore(int type, const void* src, long long src_ld, const unsigned char* e, long long e_ld, const float* mean, const float* rstd,
                              const void* g, const void* b, void* out, long long out_ld, long long rows, long long cols, void* stream_) {
  if (rows <= 0 || cols <= 0 || out_ld < cols || cols > 0x3fffffff || src_ld < 0) return GTK_ERR_ARG;
  const cudaStream_t stream = (cudaStream_t)stream_;
  const Source s{src, src_ld, e, e_ld};
  auto of = [&](auto t) -> int {
    using T = decltype(t);
    const Apply<T> f{mean, rstd, (const T*)g, (const T*)b};
    return e ? restore<signed char, T>(s, f, out, out_ld, rows, (int)cols, stream) : restore<T, T>(s, f, out, out_ld, rows, (int)cols, stream);
  };
  switch (type) {
    case kF32: return of(float{});
    case kF16: return of(__half{});
    case kBF16: return of(__nv_bfloat16{});
  }
  return GTK_ERR_ARG;
}

// Up to four matrices to operands by one launch.  list: for each of them eight words - kind (0: f32 to three bf16 pieces,
// 1: 16 bits as they are, 2 and 3: codes to f16 and bf16, 4 and 5: f32 to two f16 pieces scaled by rows and by columns),
// address, leading dimension, exponents (codes) or largest magnitudes (pairs: an unsigned int for each row, written
// here, or for each column, zeros before the call), the exponents' leading dimension, rows, columns, address of the
// operand (pitch: the columns rounded up to 8; pieces follow one another), on 16 bytes.
extern "C" int gtk_k7_pack(gtk_addresses list, void* stream) {
  if (list.n == 0 || list.n % 8 || list.n > 8 * kPackItems) return GTK_ERR_ARG;
  PackList l{}, columns{};
  unsigned long long blocks = 0, column_blocks = 0;
  for (unsigned i = 0; i < list.n / 8; ++i) {
    const unsigned long long* w = list.p + 8 * i;
    PackItem& p = l.item[i];
    p.kind = (int)w[0];
    p.src = Source{(const void*)w[1], (long long)w[2], (const unsigned char*)w[3], (long long)w[4]};
    p.rows = (long long)w[5];
    p.out = (void*)w[7];
    p.most = (unsigned int*)w[3];
    const long long cols = (long long)w[6];
    if (w[0] > 5 || !p.src.p || !p.out || p.rows <= 0 || cols <= 0 || cols > 0x3ffffff0 || p.src.ld < 0 || (uintptr_t)p.out % 16 || (w[0] >= 2 && !w[3]))
      return GTK_ERR_ARG;
    p.cols = (int)cols;
    p.pitch = (p.cols + 7) / 8 * 8;
    const bool f32 = p.kind == kPackPieces || p.kind >= kPackPairsOfRows;
    const int elem = f32 ? 4 : p.kind == kPackCopy ? 2 : 1, vec = f32 ? 4 : 8;
    p.step = 1;
    for (int step : {vec, 4})
      if (p.step == 1 && p.cols % step == 0 && aligned(p.src.p, p.src.ld, elem, step)) p.step = step;
    p.first = (unsigned)blocks;
    if (p.kind == kPackPairsOfRows) {
      p.strips = p.cols <= kWarpRow ? 1u : 2u;
      blocks += (unsigned long long)(p.strips == 1 ? (p.rows + kRowWarps - 1) / kRowWarps : p.rows);
    } else {
      p.strips = (unsigned)((p.pitch + 32 * vec - 1) / (32 * vec));
      unsigned y;
      if (!row_grid(p.rows, p.strips, &p.per, &y)) return GTK_ERR_UNSUPPORTED;
      blocks += (unsigned long long)p.strips * y;
      if (p.kind == kPackPairsOfColumns) {
        PackItem& q = columns.item[columns.count++];
        q = p;
        q.first = (unsigned)column_blocks;
        column_blocks += (unsigned long long)p.strips * y;
      }
    }
    if (blocks > 0x7fffffffull) return GTK_ERR_UNSUPPORTED;
  }
  l.count = (int)(list.n / 8);
  cudaError_t err = cudaSuccess;
  if (columns.count) {
    err = launch_pdl(k7_column_most, dim3((unsigned)column_blocks), dim3(32, kRowWarps), (cudaStream_t)stream, columns);
    gtk_count_launch(1);
    if (err != cudaSuccess) return GTK_ERR_CUDA;
  }
  err = launch_pdl(k7_pack, dim3((unsigned)blocks), dim3(32, kRowWarps), (cudaStream_t)stream, l);
  gtk_count_launch(1);
  return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

// Lines of `cols` floats that `partial` has to hold.
extern "C" int gtk_k7_act_lines(void) { return kActLines; }

// dz = dy act'(z), db = sum of dz over the rows; z in `type`, or codes where e is given; dz and db may be null.
extern "C" int gtk_k7_act_backward(int type, const void* dy, long long dy_ld, const void* z, long long z_ld, const unsigned char* e, long long e_ld, int act,
                                   void* dz, long long dz_ld, void* db, float* partial, long long rows, long long cols, void* stream_) {
  if (rows <= 0 || cols <= 0 || cols > 0x3fffffff || act < 0 || act >= kActCount || (act != kActNone && !z) || (!dz && !db)) return GTK_ERR_ARG;
  const cudaStream_t stream = (cudaStream_t)stream_;
  const Source s{z, z_ld, e, e_ld};
  auto of = [&](auto t) {
    using T = decltype(t);
    return e ? act_backward<T, signed char>(dy, dy_ld, s, act, dz, dz_ld, db, partial, kActLines, rows, (int)cols, stream)
             : act_backward<T, T>(dy, dy_ld, s, act, dz, dz_ld, db, partial, kActLines, rows, (int)cols, stream);
  };
  switch (type) {
    case kF32: return of(float{});
    case kF16: return of(__half{});
    case kBF16: return of(__nv_bfloat16{});
  }
  return GTK_ERR_ARG;
}
