// K9: a linear layer over few rows (32 at most): one step of 20 sequences, a single token.
//
//   z = x W^T + b ; y = act(z) + r ; z kept in its type or in 8 bits
//
// Bound by the bytes of W, each read once (f32 above 16 rows: twice, for 16 rows of x each), and by latency.  A tile of a
// matrix product for 256 rows would wait for its few useful rows as long as for all, and wants rows of W on 16-byte
// boundaries; here W goes from memory to registers
// at any alignment and to the tensor cores by mma.sync, whose rate is of no account: W's rows are its rows, x's rows
// its columns.  Which element of the contracted axis stands at which place of a fragment is free as long as both
// operands agree: a lane takes 16 neighbours of a row, so that a warp reads whole lines of 16 rows.
//
// A CTA takes 32 rows of W (a block of the 8-bit form): two halves of 8 warps, which take 64 of k in turn and join
// their sums through shared memory, in order.  The next 64 of W and x are on their way meanwhile (x, too, comes from L2:
// no two warps of a half read the same part of it).  f32: three bf16 pieces a value and the six products that count; the
// large one is summed apart from the small ones, and both go to an f32 sum after every 64 of k, as in K8.  1500 x 6000 bf16
// (18 MB, 2.8 us at a copy's rate): 1, 8, 20 and 32 rows 7, 8, 12 and 14 us; f32 12, 12, 27 and 29.
#include "colsum.cuh"
#include "common.cuh"
#include "host_api.h"
#include "launch.cuh"

namespace gtk {

constexpr int kFewThreads = 512;
constexpr int kFewMost = 32;       // rows of x
constexpr int kFewChunk = 64;      // of k, a warp's turn: 16 for each lane of a quad

struct FewArgs {
  const void* x;
  const void* w;
  long long x_ld, w_ld;
  int m, n, k;
  void* y;
  long long y_ld;
  const void* bias;
  const void* add;
  long long add_ld;
  int act;
  void* z;
  signed char* q;
  long long q_ld;
  unsigned char* e;
  long long e_ld;
};

// A lane's N of 4 N elements of a row that the four lanes of a quad share, in registers, as words of two (16 bits) or one
// (f32); zeros past the row's end.  Vectors of VEC go round the quad, so that each load of a warp takes whole sectors.
template <typename T, int VEC, int N>
struct Strip {
  static constexpr int kWords = N * (int)sizeof(T) / 4;
  uint32_t w[kWords];
  // of the part of the row that starts at `at`
  __device__ __forceinline__ void load(const T* row, int at, int quad, int k, bool exists) {
    if constexpr (VEC * sizeof(T) >= 4) {
      constexpr int kEach = VEC * (int)sizeof(T) / 4;   // words a load
#pragma unroll
      for (int i = 0; i < N / VEC; ++i) {
        const int c = at + (i * 4 + quad) * VEC;
        Vec<uint32_t, kEach> v = {};
        if (exists && c < k) v = *reinterpret_cast<const Vec<uint32_t, kEach>*>(row + c);   // k is a multiple of VEC
#pragma unroll
        for (int j = 0; j < kEach; ++j) w[i * kEach + j] = v.v[j];
      }
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        const int c = at + (i * 4 + quad) * 2;
        const uint32_t low = exists && c < k ? p[c] : 0u, high = exists && c + 1 < k ? p[c + 1] : 0u;
        w[i] = low | (high << 16);
      }
    }
  }
  __device__ __forceinline__ float value(int i) const { return __uint_as_float(w[i]); }   // f32
};

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Three bf16 pieces of two neighbours, a word each: the significand cut after 8, 16 and 24 bits, which takes a third of the
// instructions of rounding the pieces.  What the products of pieces then leave out is 2^-22 of a product at most, 2^-24
// on average.  An infinity's lower pieces are NaN, which add_lower leaves out.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    w[i] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
    b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
  }
}

// TOK: groups of 8 rows of x, which a CTA takes; blockIdx.y: of which rows.
template <typename T, int TOK, int VEC>
__global__ void __launch_bounds__(kFewThreads) k9_few_rows(FewArgs g) {
  constexpr int kPitch = TOK * 8 + 1;
  constexpr int kSplits = 8;   // warps that share a row's k
  __shared__ float sums[kSplits][32][kPitch];
  pdl_begin(g.x, g.w, g.bias, g.add);
  const int r0 = (int)blockIdx.y * TOK * 8, rows = min(TOK * 8, g.m - r0);
  const int warp = (int)(threadIdx.x >> 5), lane = (int)lane_id(), half = warp & 1, split = warp >> 1, row = lane >> 2, quad = lane & 3;
  const int n0 = (int)blockIdx.x * 32 + half * 16;
  const T* w0 = (const T*)g.w + (long long)min(n0 + row, g.n - 1) * g.w_ld;
  const T* w1 = (const T*)g.w + (long long)min(n0 + row + 8, g.n - 1) * g.w_ld;
  const T* xr[TOK];
#pragma unroll
  for (int t = 0; t < TOK; ++t) xr[t] = (const T*)g.x + (long long)(r0 + min(t * 8 + row, rows - 1)) * g.x_ld;
  float large[TOK][4], small[TOK][4], total[TOK][4];
#pragma unroll
  for (int t = 0; t < TOK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) large[t][i] = small[t][i] = total[t][i] = 0.f;
  // Loads of single 16-bit elements are put together at once and cannot be ahead; f32 has registers for x's only with
  // up to 8 rows.
  constexpr bool kAhead = VEC * sizeof(T) >= 4, kXAhead = kAhead && (sizeof(T) == 2 || TOK == 1);
  Strip<T, VEC, 16> a0, a1, ax[TOK];
  auto fetch_w = [&](int from) {
    a0.load(w0, from, quad, g.k, true);
    a1.load(w1, from, quad, g.k, true);
  };
  auto fetch_x = [&](int from) {
#pragma unroll
    for (int t = 0; t < TOK; ++t) ax[t].load(xr[t], from, quad, g.k, t * 8 + row < rows);
  };
  const int end = n0 < g.n ? g.k : 0;   // nothing to do for rows past W's
  int c = split * kFewChunk;
  if (kAhead && c < end) fetch_w(c);
  if (kXAhead && c < end) fetch_x(c);
  for (; c < end; c += kSplits * kFewChunk) {
    if constexpr (!kAhead) fetch_w(c);
    if constexpr (!kXAhead) fetch_x(c);
    const Strip<T, VEC, 16> u0 = a0, u1 = a1;
    Strip<T, VEC, 16> x[TOK];
#pragma unroll
    for (int t = 0; t < TOK; ++t) x[t] = ax[t];
    const int next = c + kSplits * kFewChunk;
    if (kAhead && next < end) fetch_w(next);
    if (kXAhead && next < end) fetch_x(next);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int t = 0; t < TOK; ++t) mma16816(large[t], u0.w[2 * s], u1.w[2 * s], u0.w[2 * s + 1], u1.w[2 * s + 1], x[t].w[2 * s], x[t].w[2 * s + 1], T{});
      } else {
        uint32_t p0[3], p1[3], p2[3], p3[3];
        split_pair(u0.value(4 * s), u0.value(4 * s + 1), p0);
        split_pair(u1.value(4 * s), u1.value(4 * s + 1), p1);
        split_pair(u0.value(4 * s + 2), u0.value(4 * s + 3), p2);
        split_pair(u1.value(4 * s + 2), u1.value(4 * s + 3), p3);
#pragma unroll
        for (int t = 0; t < TOK; ++t) {
          uint32_t q0[3], q1[3];
          split_pair(x[t].value(4 * s), x[t].value(4 * s + 1), q0);
          split_pair(x[t].value(4 * s + 2), x[t].value(4 * s + 3), q1);
#pragma unroll
          for (int i = 2; i >= 0; --i)
#pragma unroll
            for (int j = 2 - i; j >= 0; --j) {
              if (i + j == 0) mma16816(large[t], p0[0], p1[0], p2[0], p3[0], q0[0], q1[0], __nv_bfloat16{});
              else mma16816(small[t], p0[i], p1[i], p2[i], p3[i], q0[j], q1[j], __nv_bfloat16{});
            }
        }
      }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int t = 0; t < TOK; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          total[t][i] = add_lower(total[t][i] + large[t][i], small[t][i]);
          large[t][i] = small[t][i] = 0.f;
        }
    }
  }
#pragma unroll
  for (int t = 0; t < TOK; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      sums[split][half * 16 + row + (i >> 1) * 8][t * 8 + quad * 2 + (i & 1)] = sizeof(T) == 2 ? large[t][i] : total[t][i];
  __syncthreads();
  // a lane is a column of y, a warp takes rows in turn
  const int col = (int)blockIdx.x * 32 + lane;
  const bool inside = col < g.n;
  const float bias = inside && g.bias ? to_f32(((const T*)g.bias)[col]) : 0.f;
  for (int i = warp; i < rows; i += kFewThreads / 32) {
    const long long r = r0 + i;
    float v = sums[0][lane][i];
#pragma unroll
    for (int k = 1; k < kSplits; ++k) v += sums[k][lane][i];
    v += bias;
    if (g.q) {
      const uint32_t byte = block8_byte(__reduce_max_sync(0xffffffffu, inside ? __float_as_uint(v) & 0x7fffffffu : 0u));
      g.q[r * g.q_ld + col] = inside ? (signed char)block8_code(v, byte) : (signed char)0;
      if (lane == 0) g.e[r * g.e_ld + blockIdx.x] = (unsigned char)byte;
    }
    if (inside) {
      if (g.z) ((T*)g.z)[r * g.n + col] = from_f32<T>(v);
      with_act(g.act, [&](auto A) { v = act_value<decltype(A)::value>(v); });
      if (g.add) v += to_f32(((const T*)g.add)[r * g.add_ld + col]);
      ((T*)g.y)[r * g.y_ld + col] = from_f32<T>(v);
    }
  }
}

template <typename T>
cudaError_t launch_few(const FewArgs& g, cudaStream_t stream) {
  auto fits = [&](int vec) {
    const long long bytes = (long long)sizeof(T) * vec;
    return g.k % vec == 0 && (uintptr_t)g.x % bytes == 0 && (uintptr_t)g.w % bytes == 0 && g.x_ld % vec == 0 && g.w_ld % vec == 0;
  };
  constexpr int wide = 16 / sizeof(T);
  auto go = [&](auto tok) {
    constexpr int TOK = decltype(tok)::value;
    const dim3 grid((unsigned)((g.n + 31) / 32), (unsigned)((g.m + TOK * 8 - 1) / (TOK * 8)));
    if (fits(wide)) return launch_pdl(k9_few_rows<T, TOK, wide>, grid, dim3(kFewThreads), stream, g);
    if (wide == 8 && fits(4)) return launch_pdl(k9_few_rows<T, TOK, 4>, grid, dim3(kFewThreads), stream, g);
    return launch_pdl(k9_few_rows<T, TOK, 1>, grid, dim3(kFewThreads), stream, g);
  };
  if (g.m <= 8) return go(std::integral_constant<int, 1>{});
  if (sizeof(T) == 4 || g.m <= 16) return go(std::integral_constant<int, 2>{});   // f32 has no registers for more
  if constexpr (sizeof(T) == 2) return go(std::integral_constant<int, 4>{});
  return cudaErrorInvalidValue;
}

}  // namespace gtk

using namespace gtk;

// y[m][n] = act(x W^T + bias) + add; z dense, everything of `type`.  q has q_ld >= n rounded up to 32.
extern "C" int gtk_k9_few_rows(int type, const void* x, long long x_ld, const void* w, long long w_ld, long long m, long long n, long long k, void* y,
                               long long y_ld, const void* bias, const void* add, long long add_ld, int act, void* z, signed char* q, long long q_ld, unsigned char* e,
                               long long e_ld, void* stream) {
  if (m <= 0 || m > kFewMost || n <= 0 || k <= 0 || !x || !w || !y || x_ld < 0 || w_ld < 0 || y_ld < n || act < 0 || act >= kActCount ||
      (q && (!e || q_ld < (n + kBlock8 - 1) / kBlock8 * kBlock8)))
    return GTK_ERR_ARG;
  if (n > 0x3fffffff || k > 0x3fffffff) return GTK_ERR_UNSUPPORTED;
  const FewArgs g{x, w, x_ld, w_ld, (int)m, (int)n, (int)k, y, y_ld, bias, add, add_ld, act, z, q, q_ld, e, e_ld};
  cudaError_t err;
  switch (type) {
    case kF32: err = launch_few<float>(g, (cudaStream_t)stream); break;
    case kF16: err = launch_few<__half>(g, (cudaStream_t)stream); break;
    case kBF16: err = launch_few<__nv_bfloat16>(g, (cudaStream_t)stream); break;
    default: return GTK_ERR_ARG;
  }
  gtk_count_launch(1);
  return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}
