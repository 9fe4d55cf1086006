// K8: matrix products of a linear layer, with what follows them in the epilogue.
//
//   forward    z = x W^T + b ; y = act(z) + r ; z kept in its type or in 8 bits
//   input      dx = dz W, or with the layer before: dz' = (dz W) act'(z'), h' = act(z'), sums of dz' over the rows
//   weight     dW = dz^T x
//
// All are D[m][n] = sum_k A[m][k] B[n][k] over operands of 16 bits whose contracted axis is either the inner one of
// its matrix ("k-major": x and W forward) or the outer one ("mn-major": W for dx, both for dW); the tensor cores
// take both, so nothing is transposed in memory.  f32 operands come as three bf16 pieces a value (8 + 8 + 8 bits of
// the significand) and are multiplied piece by piece: the six products down to 2^-18 of the largest; what is left
// out is below 2^-26.  Or, where a program has chosen it, as two f16 pieces of 11 + 11 bits, scaled by a power of two so
// that the largest of each row of A and B is just under 2^15: three products, and what is left out is below 2^-24 for
// entries down to 2^-17 of their row's largest, 2^-40 of that largest for smaller ones.  The tensor cores cut a sum to 24 bits where they add to it instead of rounding it, which over
// the 6 * 1500 / 16 additions of K = 1500 took 1e-5 off the result (measured; f32 summed in order: 7e-7).  So the large
// product has an accumulator apart from the five small ones, and every 256 of k both are added to f32 registers of the
// epilogue's warps and begun again.
//
// A pair of CTAs (a cluster of two) computes tiles of 256 x bn: each holds 128 rows of A, half of the columns' B and the
// accumulators of its 128 rows, and one thread of the first issues tcgen05.mma for both, which reads each half of B
// once for the two tensor cores.  (One CTA with 128 x 256 reads 96 bytes of shared memory a cycle for its products
// and has 96 written by TMA, of 128 that there are: 920 TFLOP/s at 8192 x 2048 x 8192 before any epilogue.)  In each
// CTA one thread brings operand tiles by TMA and eight warps take finished accumulators out of TMEM, a row per lane.
// Two accumulators alternate: the epilogue of a tile overlaps the products of the next.
//
// Where tiles are few and k is long, k is split over the pairs of a larger cluster (`splits`); their sums are joined
// through distributed shared memory in the order of the pairs, each CTA finishing a share of the columns.
//
// Matrices whose rows lie on 16-byte boundaries are read and written by each lane along its row; others go through
// a padded buffer in shared memory, so that a warp's accesses run along rows.
//
// 8192 x 2048 x 8192 bf16: forward 181 to 190 us (1.45 to 1.52 PFLOP/s, under the power cap), with gelu and its 8-bit input 200 to
// 216, the input gradient and the weight's 200 to 245 (256 tiles are 3.5 rounds of the 74 pairs); 700 x 1500 x 10000 f32
// 110 us of three pieces (1.15 PFLOP/s of bf16 products), as pairs 75 us (0.84 PFLOP/s of f16 products: shared memory, read
// for three products of 128 columns and written, is full).
//
// Every wait ends: after a time limit the waiter raises the CTA's abort flag and the status word, everybody leaves
// after its copies and products in flight, and TMEM is freed.
#include <cuda.h>

#include <atomic>

#include "colsum.cuh"
#include "common.cuh"
#include "host_api.h"
#include "launch.cuh"

namespace gtk {

constexpr int kTileM = 256;           // rows of a pair's tile
constexpr int kRows = 128;            // of one CTA
constexpr int kTileK = 64;            // 128 bytes of 16-bit elements: one swizzle span
constexpr int kMaxBn = 256;           // columns of a tile
constexpr int kGemmThreads = 384;     // warps 0 and 2 load A and B, warp 1 multiplies, warps 4 to 11 are the epilogue
constexpr int kEpiWarps = 8;
constexpr int kPatchPitch = 36;       // floats a row of the epilogue's buffer: no bank conflicts, 16 bytes a lane along rows or 4 across
constexpr int kPatchBytes = kEpiWarps * 32 * kPatchPitch * 4;
constexpr int kMaxStages = 8;
constexpr int kF32Blocks = 4;         // f32: blocks of k that are summed in TMEM before they go to registers
constexpr int kMaxSplits = 4;         // pairs of a cluster: 8 CTAs are portable
constexpr int kMaxShared = 227 * 1024;
constexpr int kStaticShared = 2048;   // room for the kernel's static part

__device__ unsigned int g_gemm_status;   // not 0: a wait ran out (its place in the code)

struct GemmShape {
  int m, n;
  int tiles_m, tiles_n, blocks_k;
  int bn, stages, splits;
  int wide;                            // the epilogue's matrices have rows on boundaries of 32 bytes (2), of 16 (1) or of neither (0)
  int a_pieces, b_pieces;
  int a_mn, b_mn;                      // 1: mn-major
  uint32_t idesc;
  unsigned long long limit_ns;         // of a wait
};

struct GemmEpilogue {
  void* out;              // y, dx, dW or dz'
  long long out_ld;
  const void* bias;       // forward
  const void* add;        // residual, added behind the activation
  long long add_ld;
  int act;
  void* z;                // forward: z is stored here; slope: z' is read from here
  long long z_ld;
  signed char* q;         // the same in 8 bits
  long long q_ld;
  unsigned char* e;
  long long e_ld;
  void* h;                // slope: act(z') is stored here
  long long h_ld;
  float* sums;            // slope: [rows / 32, rounded up][n], sums of dz' over 32 rows each
  void* db;               // with up to 32 rows, a single line, the sums themselves
  const unsigned int* a_most;   // operands of two f16 pieces: the largest magnitudes (bits) of A's m and B's n, from
  const unsigned int* b_most;   // which their scales follow
};

// ---- PTX ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// True in one lane of the warp.  The compiler knows that what it guards runs in a single thread, whose operands then are
// uniform: behind a comparison of the lane's number a product took 75 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n.reg .pred p;\n"
      "elect.sync _|p, 0xffffffff;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(is));
  return is != 0;
}
// The address of the same variable in another CTA of the cluster.
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_remote(uint32_t bar) {   // a cluster address
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\n"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// False where the CTA has given up; then nothing may be assumed about what was waited for.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint32_t where, uint64_t limit_ns) {
  uint64_t t0 = 0;
  for (uint32_t spins = 1;; ++spins) {
    if (mbar_try(bar, parity)) return true;
    if ((spins & 255u) == 0u) {   // the clock is slow to read: not before a wait is a long one
      if (*abort) return false;
      const uint64_t t = globaltimer_ns();
      if (t0 == 0) t0 = t;
      if (t - t0 > limit_ns) {
        *abort = 1;
        atomicCAS(&g_gemm_status, 0u, where);
        return false;
      }
    }
  }
}
// The same by a whole warp, with one answer for all its lanes: one may see the barrier complete where another gives up, and
// a part of a warp must not go on to instructions that all of it has to execute.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint32_t where, uint64_t limit_ns) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, where, limit_ns));
}
// Into this CTA's shared memory; `bar` may be the pair's other CTA's.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int piece, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(piece), "r"(bar)
               : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle.  k-major: rows of 128 bytes, 8 rows (1024 bytes) to the next
// group.  mn-major: 64 elements of m or n by 8 of k are 1024 bytes, the next 8 of k follow, the next 64 of m or n
// are `lead` bytes further.  The low word holds address / 16, to which offsets / 16 can be added.
__device__ __forceinline__ uint32_t operand_desc(uint32_t addr, uint32_t lead) { return ((addr & 0x3ffffu) >> 4) | ((lead >> 4) << 16); }
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void mma(uint32_t tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b64 a, b;\n"
      "setp.ne.b32 p, %5, 0;\n"
      "mov.b64 a, {%1, %3};\n"
      "mov.b64 b, {%2, %3};\n"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n}" ::"r"(tmem),
      "r"(a), "r"(b), "r"(kDescHigh), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The barrier, in both CTAs of the pair, is arrived on when all products issued before by this thread are done.
__device__ __forceinline__ void mma_commit(uint32_t bar, uint16_t pair) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(pair) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]),
        "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]),
        "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Tiles in groups of 8 rows of tiles, so that CTAs that run at the same time share operand tiles in L2.
__device__ __forceinline__ void tile_at(const GemmShape& s, int tile, int* tm, int* tn) {
  const int span = 8 * s.tiles_n;
  const int first = tile / span * 8;
  const int high = min(8, s.tiles_m - first);
  const int in = tile % span;
  *tm = first + in % high;
  *tn = in / high;
}

// Bytes of an operand's tile in shared memory, per piece.
__device__ __forceinline__ void load_operand(uint32_t dst, const CUtensorMap* map, int mn_major, int pieces, int rows, int mn0, int k0, uint32_t bar) {
  for (int p = 0; p < pieces; ++p) {
    if (mn_major) {
      for (int r = 0; r < rows; r += 64) tma_load(dst + (uint32_t)r * 128u, map, mn0 + r, k0, p, bar);
    } else {
      tma_load(dst, map, k0, mn0, p, bar);
    }
    dst += (uint32_t)rows * 128u;
  }
}

// Products of pieces, small ones first: (a, b) in two bits each.
__device__ __forceinline__ int piece_products(int a_pieces, int b_pieces, uint32_t* list) {
  // nibble = a | b << 2
  if (a_pieces == 3 && b_pieces == 3) {
    *list = 0x014528u;   // (0,2)=8, (2,0)=2, (1,1)=5, (0,1)=4, (1,0)=1, (0,0)=0
    return 6;
  }
  if (a_pieces == 3) {
    *list = 0x012u;      // (2,0), (1,0), (0,0)
    return 3;
  }
  if (a_pieces == 2) {
    *list = 0x014u;      // (0,1), (1,0), (0,0)
    return 3;
  }
  *list = 0;
  return 1;
}

// ---- epilogue: 32 rows by 32 columns a warp, a row per lane ------------------------------------------------------------
struct Patch {
  float* room;          // [32][kPatchPitch] of this warp
  int row, col0;        // this lane's row, the first column
  int row0, m, n, wide;
};

// The lane's row to and from the warp's buffer.
__device__ __forceinline__ void patch_put(const Patch& p, const float (&v)[32]) {
  __syncwarp();
#pragma unroll
  for (int g = 0; g < 8; ++g) *reinterpret_cast<float4*>(p.room + (int)lane_id() * kPatchPitch + 4 * g) = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
  __syncwarp();
}
__device__ __forceinline__ void patch_get(const Patch& p, float (&v)[32]) {
  __syncwarp();
#pragma unroll
  for (int g = 0; g < 8; ++g) {
    const float4 x = *reinterpret_cast<const float4*>(p.room + (int)lane_id() * kPatchPitch + 4 * g);
    v[4 * g] = x.x;
    v[4 * g + 1] = x.y;
    v[4 * g + 2] = x.z;
    v[4 * g + 3] = x.w;
  }
}

// 32 bytes at once: a lane's access touches a line of its own, so that half as many accesses take half the time.
__device__ __forceinline__ void load32b(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store32b(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
               "r"(w[6]), "r"(w[7])
               : "memory");
}

// Where rows lie on no boundary, so many rows' elements are loaded before the first is put into the buffer.  Left to the
// compiler, to which the buffer may be the matrix, every load waits for the one before: 7553 x 98 x 894 f32 with a
// residual 112 us instead of 46.  (16: 41, but the 16-bit types, whose loops did not wait, lose up to 10 %.)
constexpr int kRowsAhead = 8;

// v = the lane's row of a matrix of T, columns col0 .. col0 + 31; what is outside is left alone.
template <typename T>
__device__ __forceinline__ void read32(const void* base, long long ld, const Patch& p, float (&v)[32]) {
  constexpr int G = 16 / sizeof(T);
  if (p.wide == 2) {
    if (p.row < p.m) {
      const T* at = (const T*)base + (long long)p.row * ld + p.col0;
#pragma unroll
      for (int g = 0; g < 32; g += 2 * G) {
        if (p.col0 + g < p.n) {   // n is a multiple of 2 G
          uint32_t w[8];
          load32b(at + g, w);
          float x[2 * G];
          to_f32<T, 2 * G>(*reinterpret_cast<const Vec<T, 2 * G>*>(w), x);
#pragma unroll
          for (int i = 0; i < 2 * G; ++i) v[g + i] = x[i];
        }
      }
    }
  } else if (p.wide) {
    if (p.row < p.m) {
      const T* at = (const T*)base + (long long)p.row * ld + p.col0;
#pragma unroll
      for (int g = 0; g < 32; g += G) {
        if (p.col0 + g < p.n) {   // n is a multiple of G
          float x[G];
          load_f32<T, G>(at + g, x);
#pragma unroll
          for (int i = 0; i < G; ++i) v[g + i] = x[i];
        }
      }
    }
  } else {
    const int col = p.col0 + (int)lane_id(), rows = min(32, p.m - p.row0);
    __syncwarp();
    if (col < p.n) {
      const T* at = (const T*)base + (long long)p.row0 * ld + col;
      auto take = [&](int r, auto whole) {
        T x[kRowsAhead];
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i)
          if (decltype(whole)::value || r + i < rows) x[i] = at[(r + i) * ld];
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i)
          if (decltype(whole)::value || r + i < rows) p.room[(r + i) * kPatchPitch + (int)lane_id()] = to_f32(x[i]);
      };
      int r = 0;
      for (; r + kRowsAhead <= rows; r += kRowsAhead) take(r, std::true_type{});
      if (r < rows) take(r, std::false_type{});
    }
    patch_get(p, v);
  }
}

template <typename T>
__device__ __forceinline__ void write32(void* base, long long ld, const Patch& p, const float (&v)[32]) {
  constexpr int G = 16 / sizeof(T);
  if (p.wide == 2) {
    if (p.row < p.m) {
      T* at = (T*)base + (long long)p.row * ld + p.col0;
#pragma unroll
      for (int g = 0; g < 32; g += 2 * G) {
        if (p.col0 + g < p.n) {
          uint32_t w[8];
          if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pack2(v[g + 2 * i], v[g + 2 * i + 1], T{});
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[g + i]);
          }
          store32b(at + g, w);
        }
      }
    }
  } else if (p.wide) {
    if (p.row < p.m) {
      T* at = (T*)base + (long long)p.row * ld + p.col0;
#pragma unroll
      for (int g = 0; g < 32; g += G) {
        if (p.col0 + g < p.n) {
          float x[G];
#pragma unroll
          for (int i = 0; i < G; ++i) x[i] = v[g + i];
          store_f32<T, G>(at + g, x);
        }
      }
    }
  } else {
    const int col = p.col0 + (int)lane_id(), rows = min(32, p.m - p.row0);
    patch_put(p, v);
    if (col < p.n) {
      T* at = (T*)base + (long long)p.row0 * ld + col;
#pragma unroll 8
      for (int r = 0; r < rows; ++r) at[r * ld] = from_f32<T>(p.room[r * kPatchPitch + (int)lane_id()]);
    }
  }
}

// The 8-bit form of the lane's 32 columns, one block.  Codes past the matrix are zeros.
__device__ __forceinline__ void write_codes(const GemmEpilogue& e, const Patch& p, const float (&z)[32]) {
  if (p.row >= p.m) return;
  const bool whole = p.col0 + 32 <= p.n;
  float most = 0.f;
  uint32_t w[8], byte;
  if (whole) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) most = max_abs(most, z[i], z[i + 1]);
    byte = block8_byte(__float_as_uint(most));
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (p.col0 + i < p.n) most = max_abs(most, most, z[i]);
    byte = block8_byte(__float_as_uint(most));
  }
  if (whole && byte < kBlock8Last) {
    const float inverse = block8_inverse(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = block8_codes(z[4 * i], z[4 * i + 1], z[4 * i + 2], z[4 * i + 3], inverse);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[i] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (p.col0 + 4 * i + j < p.n) w[i] |= ((uint32_t)block8_code(z[4 * i + j], byte) & 255u) << (8 * j);
    }
  }
  store32b(e.q + (long long)p.row * e.q_ld + p.col0, w);   // rows of whole blocks
  e.e[(long long)p.row * e.e_ld + p.col0 / kBlock8] = (unsigned char)byte;
}

// What the lane's 32 codes stand for.
__device__ __forceinline__ void read_codes(const GemmEpilogue& e, const Patch& p, float (&z)[32]) {
  if (p.wide) {
    if (p.row < p.m) {
      const signed char* at = e.q + (long long)p.row * e.q_ld + p.col0;
      const float scale = block8_scale(e.e[(long long)p.row * e.e_ld + p.col0 / kBlock8]);
      if (p.wide == 2) {   // n is a multiple of 32
        uint32_t w[8];
        load32b(at, w);
        const Vec<signed char, 32>& q = *reinterpret_cast<const Vec<signed char, 32>*>(w);
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = (float)q.v[i] * scale;
        return;
      }
#pragma unroll
      for (int g = 0; g < 32; g += 16)
        if (p.col0 + g < p.n) {
          const Vec<signed char, 16> q = *reinterpret_cast<const Vec<signed char, 16>*>(at + g);
#pragma unroll
          for (int i = 0; i < 16; ++i) z[g + i] = (float)q.v[i] * scale;
        }
    }
  } else {
    const int col = p.col0 + (int)lane_id(), rows = min(32, p.m - p.row0);
    __syncwarp();
    if (col < p.n) {
      for (int r = 0; r < rows; r += kRowsAhead) {
        signed char q[kRowsAhead];
        unsigned char scale[kRowsAhead];
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) {
          const long long row = p.row0 + r + i;
          q[i] = r + i < rows ? e.q[row * e.q_ld + col] : (signed char)0;
          scale[i] = r + i < rows ? e.e[row * e.e_ld + col / kBlock8] : (unsigned char)0;
        }
#pragma unroll
        for (int i = 0; i < kRowsAhead; ++i) p.room[(r + i) * kPatchPitch + (int)lane_id()] = (float)q[i] * block8_scale(scale[i]);
      }
    }
    patch_get(p, z);
  }
}

// Sums of 32 columns over the 32 lanes; lane i gets column i's.  Halves the columns a lane holds at each step.  (Through
// the warp's buffer instead it is half the instructions, but two stages of operands less: no faster.)
__device__ __forceinline__ float transpose_sum(float (&v)[32]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool upper = (lane_id() & (uint32_t)o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float give = upper ? v[i] : v[i + o], keep = upper ? v[i + o] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  return v[0];
}

// bias: 32 floats of this warp in shared memory.
template <typename T>
__device__ __forceinline__ void finish_forward(float (&v)[32], float* bias, const GemmEpilogue& e, const Patch& p) {
  float r[32];
  if (e.add) read32<T>(e.add, e.add_ld, p, r);
  if (e.bias) {
    const int col = p.col0 + (int)lane_id();
    __syncwarp();
    bias[lane_id()] = col < p.n ? to_f32(((const T*)e.bias)[col]) : 0.f;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      const float4 b = *reinterpret_cast<const float4*>(bias + i);
      v[i] += b.x;
      v[i + 1] += b.y;
      v[i + 2] += b.z;
      v[i + 3] += b.w;
    }
  }
  if (e.q) write_codes(e, p, v);
  if (e.z) write32<T>(e.z, e.z_ld, p, v);
  if (e.act != kActNone)
    with_act(e.act, [&](auto A) {
      act_values<decltype(A)::value, 32>(v);
    });
  if (e.add) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += r[i];
  }
  write32<T>(e.out, e.out_ld, p, v);
}

template <typename T>
__device__ __forceinline__ void finish_slope(float (&v)[32], const GemmEpilogue& e, const Patch& p) {
  float h[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) h[i] = 0.f;
  if (e.q) read_codes(e, p, h);
  else read32<T>(e.z, e.z_ld, p, h);
  with_act(e.act, [&](auto A) {
    act_slopes<decltype(A)::value, 32>(v, h);
  });
  write32<T>(e.out, e.out_ld, p, v);
  if (e.h) write32<T>(e.h, e.h_ld, p, h);
  if (e.sums) {
    if (p.row >= p.m) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
    }
    const float sum = transpose_sum(v);
    const int col = p.col0 + (int)lane_id();
    if (col < p.n) {
      if (p.m <= 32) ((T*)e.db)[col] = from_f32<T>(sum);
      else e.sums[(long long)(p.row0 >> 5) * p.n + col] = sum;
    }
  }
}

// Takes the operands' scales out of the lane's 32 sums: times 2^-(shift of the row + shift of the column), in two steps,
// neither of which leaves f32's range where the result does not.
__device__ __forceinline__ void unscale(float (&v)[32], float* room, const GemmEpilogue& e, const Patch& p) {
  int* shifts = reinterpret_cast<int*>(room);
  const int col = p.col0 + (int)lane_id(), row = p.row < p.m ? pair_shift(e.a_most[p.row]) : 0;
  __syncwarp();
  shifts[lane_id()] = col < p.n ? pair_shift(e.b_most[col]) : 0;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int t = -(row + shifts[i]), half = t >> 1;   // -252 .. 228
    v[i] = v[i] * __uint_as_float((uint32_t)(half + 127) << 23) * __uint_as_float((uint32_t)(t - half + 127) << 23);
  }
  __syncwarp();
}

// T: type of what the epilogue reads and writes.  SLOPE: the input gradient through the layer before's activation.
// Clusters of 2 * splits CTAs; with splits 1 the pairs go through tiles in turn, else a cluster has one tile.
template <typename T, bool SLOPE>
__global__ void __launch_bounds__(kGemmThreads, 1)
k8_gemm(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const GemmShape s, GemmEpilogue e) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kMaxStages + 4];
  __shared__ alignas(16) float bias_room[kEpiWarps][32];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int abort;
  const int warp = (int)(threadIdx.x >> 5);
  const uint32_t ranks = (uint32_t)(2 * s.splits), rank = blockIdx.x % ranks, half = rank & 1u, split = rank >> 1, leader = rank & ~1u;
  const uint16_t pair = (uint16_t)(3u << leader);
  const int first_tile = (int)(blockIdx.x / ranks), step = (int)(gridDim.x / ranks), n_tiles = s.tiles_m * s.tiles_n;
  const int kb_begin = (int)((long long)s.blocks_k * split / s.splits), kb_end = (int)((long long)s.blocks_k * (split + 1) / s.splits);
  const int b_rows = s.bn / 2;          // of this CTA's half of B
  uint8_t* base = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
  const uint32_t a_bytes = (uint32_t)s.a_pieces * kRows * 128u, stage_bytes = a_bytes + (uint32_t)(s.b_pieces * b_rows) * 128u;
  float* patches = reinterpret_cast<float*>(base + (size_t)stage_bytes * s.stages);
  const uint32_t tiles = smem_addr(base);
  const uint32_t full = smem_addr(bars), empty = full + 8u * kMaxStages, acc_full = empty + 8u * kMaxStages, acc_empty = acc_full + 16u;
  constexpr bool kSplit = sizeof(T) == 4;          // f32: see the top of this file
  const uint32_t acc_columns = (uint32_t)(kSplit ? 2 * s.bn : s.bn), columns = 2 * acc_columns;   // a power of two, 32 at least
  const int run = kSplit ? kF32Blocks : s.blocks_k;   // blocks of k that one accumulator takes

  if (warp == 0 && lane_id() == 0) {
    abort = 0;
    for (int i = 0; i < s.stages; ++i) {
      mbar_init(full + 8u * i, 1);
      mbar_init(empty + 8u * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8u * i, 1);
      mbar_init(acc_empty + 8u * i, 2 * kEpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&a_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&b_map) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_at)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_begin(e.bias, e.add, e.z, e.q, e.e, e.a_most, e.b_most);

  if (warp == 0 || warp == 2) {   // one for each operand: a copy takes its thread 130 cycles, a block of k 512 with 256 columns
    if (elect_one()) {
      const bool is_a = warp == 0;
      const uint32_t pair_full = mapa(full, leader);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < n_tiles; tile += step) {
        int tm, tn;
        tile_at(s, tile, &tm, &tn);
        for (int kb = kb_begin; kb < kb_end; ++kb) {
          ok = mbar_wait(empty + 8u * stage, phase ^ 1u, &abort, 1, s.limit_ns);
          if (!ok) break;
          if (is_a && half == 0) mbar_expect(full + 8u * stage, 2u * stage_bytes);   // the pair's
          const uint32_t dst = tiles + (uint32_t)stage * stage_bytes, bar = pair_full + 8u * stage;
          if (is_a) load_operand(dst, &a_map, s.a_mn, s.a_pieces, kRows, tm * kTileM + (int)half * kRows, kb * kTileK, bar);
          else load_operand(dst + a_bytes, &b_map, s.b_mn, s.b_pieces, b_rows, tn * s.bn + (int)half * b_rows, kb * kTileK, bar);
          if (++stage == s.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // No copy and no arrival is left under way: the consumer has freed every stage.
      for (int i = 0; ok && i < s.stages; ++i) {
        ok = mbar_wait(empty + 8u * stage, phase ^ 1u, &abort, 5, s.limit_ns);
        if (++stage == s.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok && is_a && half == 0)   // given up: the pair's copies under way end
        for (int i = 0; i < s.stages; ++i) {
          const bool second = i >= stage;   // this stage's last copy belongs to the round before
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try(full + 8u * i, second ? phase ^ 1u : phase) && globaltimer_ns() - t0 < 100000000ull) {
          }
        }
    }
  } else if (warp == 1) {
    if (half == 0 && elect_one()) {
      int stage = 0;
      uint32_t phase = 0, list;
      const int products = piece_products(s.a_pieces, s.b_pieces, &list);
      const uint32_t a_step = s.a_mn ? 2048u / 16 : 32u / 16, b_step = s.b_mn ? 2048u / 16 : 32u / 16;   // to the next 16 of k
      const uint32_t a_desc = operand_desc(tiles, s.a_mn ? 8192u : 16u), b_desc = operand_desc(tiles + a_bytes, s.b_mn ? 8192u : 16u);
      const uint32_t a_piece = kRows * 128u / 16, b_piece = (uint32_t)(b_rows * 128) / 16, stage_step = stage_bytes / 16;
      int turn = 0;
      bool ok = true;
      for (int tile = first_tile; ok && tile < n_tiles; tile += step)
        for (int kb = kb_begin; ok && kb < kb_end; ++turn) {
          const int acc = turn & 1, stop = min(kb + run, kb_end);
          ok = mbar_wait(acc_empty + 8u * acc, ((uint32_t)(turn >> 1) & 1u) ^ 1u, &abort, 2, s.limit_ns);
          if (!ok) break;
          tc_fence_after();
          const uint32_t large = tmem + (uint32_t)acc * acc_columns, small = kSplit ? large + (uint32_t)s.bn : large;
          uint32_t on_large = 0, on_small = 0;   // whether the accumulator holds something already
          for (; kb < stop; ++kb) {
            ok = mbar_wait(full + 8u * stage, phase, &abort, 3, s.limit_ns);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a0 = a_desc + (uint32_t)stage * stage_step, b0 = b_desc + (uint32_t)stage * stage_step;
            for (int i = 0; i < products; ++i) {
              const uint32_t at = (list >> (4 * i)) & 15u;
              const uint32_t a1 = a0 + (at & 3u) * a_piece, b1 = b0 + (at >> 2) * b_piece;
              const bool to_small = kSplit && at != 0;
              uint32_t on = to_small ? on_small : on_large;
#pragma unroll
              for (int k = 0; k < kTileK / 16; ++k) {
                mma(to_small ? small : large, a1 + k * a_step, b1 + k * b_step, s.idesc, on);
                on = 1;
              }
              if (to_small) on_small = 1;
              else on_large = 1;
            }
            mma_commit(empty + 8u * stage, pair);
            if (++stage == s.stages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          mma_commit(acc_full + 8u * acc, pair);
        }
      if (!ok) {   // products in flight end before TMEM is given back: nobody else arrives on acc_full any more
        const uint32_t last = acc_full + 8u * (turn & 1);
        mma_commit(last, pair);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try(last, (uint32_t)(turn >> 1) & 1u) && globaltimer_ns() - t0 < 100000000ull) {
        }
      }
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, side = (warp - 4) >> 2, lane = (int)lane_id();
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), pair_acc_empty = mapa(acc_empty, leader);
    Patch p{patches + (size_t)(warp - 4) * 32 * kPatchPitch, 0, 0, 0, s.m, s.n, s.wide};
    int turn = 0;
    bool ok = true;
    for (int tile = first_tile; ok && tile < n_tiles; tile += step) {
      int tm, tn;
      tile_at(s, tile, &tm, &tn);
      p.row0 = tm * kTileM + (int)half * kRows + quad * 32;
      p.row = p.row0 + lane;
      const bool some = p.row0 < s.m;   // rows of this warp
      auto finish = [&](int c, float (&v)[32]) {
        p.col0 = tn * s.bn + c;
        if (!some || p.col0 >= s.n) return;
        if (kSplit && e.a_most) unscale(v, bias_room[warp - 4], e, p);
        if constexpr (SLOPE) finish_slope<T>(v, e, p);
        else finish_forward<T>(v, bias_room[warp - 4], e, p);
      };
      // Accumulators of one of the splits, 16 bytes of every lane side by side: the lanes of a read from another CTA
      // have to be neighbours (rows 128 bytes apart took 15 us for 128 KB).
      auto put = [&](int c, const float (&v)[32]) {
        float4* at = reinterpret_cast<float4*>(base) + (size_t)((c / 32) * 4 + quad) * 256 + lane;
#pragma unroll
        for (int g = 0; g < 8; ++g) at[g * 32] = make_float4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]);
      };
      if constexpr (kSplit) {   // bn is 128 at most: two patches a warp
        float sum[2][32];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[j][i] = 0.f;
        for (int kb = kb_begin; kb < kb_end; kb += run, ++turn) {
          const int acc = turn & 1;
          ok = warp_wait(acc_full + 8u * acc, (uint32_t)(turn >> 1) & 1u, &abort, 4, s.limit_ns);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int c = side * 32 + j * 64;
            if (c < s.bn) {
              float v[32];   // (one after the other: both at once spill)
              tmem_load32(lanes + (uint32_t)acc * acc_columns + (uint32_t)c, v);
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[j][i] += v[i];
              tmem_load32(lanes + (uint32_t)acc * acc_columns + (uint32_t)(s.bn + c), v);
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[j][i] = add_lower(sum[j][i], v[i]);
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(pair_acc_empty + 8u * acc);
        }
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int c = side * 32 + j * 64;
          if (c < s.bn) {
            if (s.splits > 1) put(c, sum[j]);
            else finish(c, sum[j]);
          }
        }
      } else {
        const int acc = turn & 1;
        ok = warp_wait(acc_full + 8u * acc, (uint32_t)(turn >> 1) & 1u, &abort, 4, s.limit_ns);
        if (!ok) break;
        tc_fence_after();
        for (int c = side * 32; c < s.bn; c += 64) {
          float v[32];
          tmem_load32(lanes + (uint32_t)acc * acc_columns + (uint32_t)c, v);
          if (s.splits > 1) put(c, v);
          else finish(c, v);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote(pair_acc_empty + 8u * acc);
        ++turn;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // every CTA's sums lie in its shared memory; nothing of the pair's products is under way
  if (s.splits > 1 && warp >= 4 && !abort) {
    // This CTA finishes every splits-th 32 columns of its rows, adding the pairs' sums up in their order.
    const int quad = warp & 3, side = (warp - 4) >> 2, lane = (int)lane_id();
    int tm, tn;
    tile_at(s, first_tile, &tm, &tn);
    Patch p{patches + (size_t)(warp - 4) * 32 * kPatchPitch, 0, 0, tm * kTileM + (int)half * kRows + quad * 32, s.m, s.n, s.wide};
    p.row = p.row0 + lane;
    if (p.row0 < s.m)
      for (int c = ((int)split + side * s.splits) * 32; c < s.bn; c += 64 * s.splits) {
        p.col0 = tn * s.bn + c;
        if (p.col0 >= s.n) break;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
        const uint32_t at = tiles + (uint32_t)(((c / 32) * 4 + quad) * 256 + lane) * 16u;
        for (int k = 0; k < s.splits; ++k) {
          const uint32_t from = mapa(at, (uint32_t)(2 * k) + half);
          float4 x[8];   // all on their way before the first is used
#pragma unroll
          for (int g = 0; g < 8; ++g)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(x[g].x), "=f"(x[g].y), "=f"(x[g].z), "=f"(x[g].w)
                         : "r"(from + (uint32_t)g * 512u)
                         : "memory");
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            v[4 * g] += x[g].x;
            v[4 * g + 1] += x[g].y;
            v[4 * g + 2] += x[g].z;
            v[4 * g + 3] += x[g].w;
          }
        }
        if (kSplit && e.a_most) unscale(v, bias_room[warp - 4], e, p);
        if constexpr (SLOPE) finish_slope<T>(v, e, p);
        else finish_forward<T>(v, bias_room[warp - 4], e, p);
      }
  }
  if (s.splits > 1) {   // shared memory stays until all have read it
    __syncwarp();
    cluster_sync();
  }
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
}

// A wait that runs out, by itself: the first lane of a warp waits for a barrier that is complete, the others for one on
// which nothing arrives.  answers: what each lane is told.
__global__ void __launch_bounds__(32) k8_rehearse_wait(unsigned long long limit_ns, unsigned int* answers) {
  __shared__ uint64_t bars[2];
  __shared__ volatile int abort;
  pdl_begin(answers);
  const uint32_t complete = smem_addr(bars), never = complete + 8u;
  if (threadIdx.x == 0) {
    abort = 0;
    mbar_init(complete, 1);
    mbar_init(never, 1);
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(complete) : "memory");
  }
  __syncwarp();
  answers[threadIdx.x] = warp_wait(threadIdx.x == 0 ? complete : never, 0u, &abort, 6, limit_ns) ? 1u : 0u;
}

// ---- host -------------------------------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// One operand: rows (of m or n) by k, `pieces` matrices piece_stride elements apart.
struct Operand {
  const void* p;
  long long ld;
  int pieces;
  long long piece_stride;
  int mn_major;
  const unsigned int* most;   // two pieces: the largest magnitudes
};

inline bool encode(CUtensorMap* map, const Operand& o, int half, long long rows, long long k, int box_rows) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  const long long inner = o.mn_major ? rows : k, outer = o.mn_major ? k : rows;
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)o.pieces};
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)(o.pieces > 1 ? o.piece_stride : o.ld) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)(o.mn_major ? kTileK : box_rows), 1};
  cuuint32_t ones[3] = {1, 1, 1};
  return fn(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims, strides, box, ones,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

inline bool operand_ok(const Operand& o) {
  return o.p && (uintptr_t)o.p % 16 == 0 && o.ld > 0 && o.ld % 8 == 0 &&
         (o.pieces == 1 || ((o.pieces == 3 || (o.pieces == 2 && o.most)) && o.piece_stride > 0 && o.piece_stride % 8 == 0));
}

// Pairs that run side by side in clusters of `splits` of them (74, 66 and 56 of 1, 2 and 4 on B200: a cluster lies within
// one group of SMs).  Asked once per device.
template <typename Kernel>
int pairs_of(Kernel kernel, int splits, const DeviceInfo* info) {
  static std::atomic<int> known[64][kMaxSplits + 1];
  std::atomic<int>& slot = known[info->device][splits];
  int pairs = slot.load(std::memory_order_relaxed);
  if (pairs) return pairs;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(info->sms / (2 * splits) * 2 * splits));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = kMaxShared - kStaticShared;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)(2 * splits);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int clusters = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared - kStaticShared) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters <= 0) {
    cudaGetLastError();
    clusters = 1;
  }
  pairs = clusters * splits;
  slot.store(pairs, std::memory_order_relaxed);
  return pairs;
}

// Tiles and splits.  In cycles, a pair takes about 2 * bn for the products of a block of k (times six with pieces), at
// least 330 for its copies (pieces: 5/4 of it, as shared memory is read faster than it can be), 24 a column for a tile's
// last epilogue and 3000 + 16 a column for joining several pairs' sums (256 x 256: 3.6 us with two, 4.8 with four) and
// as much again where clusters follow one another.  The choice is the one whose busiest pair is done first.
struct GemmPlan {
  int bn, splits;
};
inline GemmPlan plan_gemm(long long m, long long n, int blocks_k, int products, int most, const DeviceInfo* info) {
  GemmPlan best{128, 1};
  long long least = -1;
  for (int bn = most; bn >= 128; bn /= 2) {
    const long long tiles = ((m + kTileM - 1) / kTileM) * ((n + bn - 1) / bn);
    const long long block = products > 1 ? 2 * bn * products * 5 / 4 : 2 * bn > 330 ? 2 * bn : 330;
    for (int splits = 1; splits <= kMaxSplits; ++splits) {
      const int pairs = pairs_of(k8_gemm<__nv_bfloat16, false>, splits, info);
      if (splits > 1 && blocks_k < 4 * splits) break;
      const long long rounds = (tiles * splits + pairs - 1) / pairs;
      const long long cost = rounds * ((blocks_k + splits - 1) / splits) * block + bn * 24 / splits + (splits > 1 ? rounds * (3000 + 16 * bn) : 0);
      if (least < 0 || cost < least) {
        least = cost;
        best = GemmPlan{bn, splits};
      }
    }
  }
  return best;
}

inline bool on(int bytes, const void* p, long long ld, int elem) { return !p || ((uintptr_t)p % bytes == 0 && ld * elem % bytes == 0); }

template <typename T>
cudaError_t launch_gemm(int device, bool slope, int grid, size_t shared, cudaStream_t stream, const CUtensorMap& a, const CUtensorMap& b, const GemmShape& s,
                        const GemmEpilogue& e) {
  static std::atomic<unsigned long long> devices[2];   // whose kernel has been given its shared memory
  const unsigned long long bit = 1ull << device;
  const bool allowed = devices[slope].load(std::memory_order_relaxed) & bit;
  auto go = [&](auto kernel) {
    cudaError_t err = cudaSuccess;
    if (!allowed) err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared - kStaticShared);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)(2 * s.splits);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (!allowed) devices[slope].fetch_or(bit, std::memory_order_relaxed);
    return cudaLaunchKernelEx(&cfg, kernel, a, b, s, e);
  };
  return slope ? go(k8_gemm<T, true>) : go(k8_gemm<T, false>);
}

}  // namespace gtk

using namespace gtk;

// Status word of the current device's products: 0, or where a wait ran out.  Synchronises.
extern "C" unsigned int gtk_k8_status(void) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_gemm_status, sizeof(v)) != cudaSuccess) return ~0u;
  return v;
}

// Sets the status word to 0.  Synchronises.
extern "C" int gtk_k8_clear_status(void) {
  const unsigned int v = 0;
  return cudaMemcpyToSymbol(g_gemm_status, &v, sizeof(v)) == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

// answers: 32 words, 1 for each lane that takes the wait for complete (see k8_rehearse_wait).
extern "C" int gtk_k8_rehearse_wait(unsigned long long limit_ns, unsigned int* answers, void* stream) {
  if (!answers) return GTK_ERR_ARG;
  const cudaError_t err = launch_pdl(k8_rehearse_wait, dim3(1), dim3(32), (cudaStream_t)stream, limit_ns, answers);
  gtk_count_launch(1);
  return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

// out[m][n] = epilogue(sum_k a[m][k] b[n][k]).  type: of what the epilogue reads and writes.  half: the operands are
// f16, else bf16; their pieces 1 and 1 in the 16-bit types, 2 and 2, 3 and 3 or 3 and 1 in f32.  Leading dimensions and piece strides of operands are multiples of 8 elements, their addresses of
// 16 bytes.  slope: see the top of this file.  sums, room for (m + 31) / 32 lines of n, with db: the sums over all rows of what the slope form stores.
// limit_ns: how long a wait lasts at most.
extern "C" int gtk_k8_gemm(int type, int half, long long m, long long n, long long k, const void* a, long long a_ld, int a_pieces, long long a_stride, int a_mn,
                           const unsigned int* a_most, const void* b, long long b_ld, int b_pieces, long long b_stride, int b_mn, const unsigned int* b_most,
                           void* out, long long out_ld, const void* bias,
                           const void* add, long long add_ld, int act, int slope, void* z, long long z_ld, signed char* q, long long q_ld, unsigned char* e8,
                           long long e_ld, void* h, long long h_ld, float* sums, void* db, unsigned long long limit_ns, void* stream_) {
  const Operand oa{a, a_ld, a_pieces, a_stride, a_mn != 0, a_most}, ob{b, b_ld, b_pieces, b_stride, b_mn != 0, b_most};
  if (m <= 0 || n <= 0 || k <= 0 || !out || act < 0 || act >= kActCount || !operand_ok(oa) || !operand_ok(ob) || (q && !e8) ||
      (q && !slope && (q_ld < (n + kBlock8 - 1) / kBlock8 * kBlock8 || q_ld % 32 || (uintptr_t)q % 32)) || (sums == nullptr) != (db == nullptr) ||
      ((a_pieces == 2) != (b_pieces == 2)) || (a_pieces == 2 && (!half || type != kF32)) || ((a_pieces == 3 || b_pieces == 3) && (a_pieces != 3 || half || type != kF32)) ||
      (type == kF32 && a_pieces == 1))   // (f32 has an accumulator for lower pieces, which then nothing would write)
    return GTK_ERR_ARG;
  if (m > 0x7fffff00LL || n > 0x7fffff00LL || k > 0x7fffff00LL) return GTK_ERR_UNSUPPORTED;
  const DeviceInfo* info = gtk_device_info();
  if (!info) return GTK_ERR_CUDA;
  GemmShape s{};
  s.m = (int)m;
  s.n = (int)n;
  s.limit_ns = limit_ns;
  s.a_pieces = a_pieces;
  s.b_pieces = b_pieces;
  s.a_mn = oa.mn_major;
  s.b_mn = ob.mn_major;
  s.tiles_m = (int)((m + kTileM - 1) / kTileM);
  s.blocks_k = (int)((k + kTileK - 1) / kTileK);
  const GemmPlan plan = plan_gemm(m, n, s.blocks_k, a_pieces * b_pieces == 9 ? 6 : a_pieces == 2 ? 3 : a_pieces * b_pieces, type == kF32 ? 128 : kMaxBn, info);
  s.bn = plan.bn;
  s.splits = plan.splits;
  s.tiles_n = (int)((n + s.bn - 1) / s.bn);
  if ((long long)s.tiles_m * s.tiles_n > 0x3fffffffLL) return GTK_ERR_UNSUPPORTED;
  const int elem = elem_bytes(type);
  for (const int bytes : {16, 32})
    if (n * elem % bytes == 0 && on(bytes, out, out_ld, elem) && on(bytes, add, add_ld, elem) && on(bytes, z, z_ld, elem) && on(bytes, h, h_ld, elem) &&
        (!q || !slope || (n % bytes == 0 && on(bytes, q, q_ld, 1))))
      s.wide = bytes / 16;
  const int stage_bytes = a_pieces * kRows * 128 + b_pieces * s.bn / 2 * 128;
  const int fixed = 1024 + (s.wide ? 0 : kPatchBytes);
  s.stages = (kMaxShared - kStaticShared - fixed) / stage_bytes;
  if (s.stages > kMaxStages) s.stages = kMaxStages;
  const uint32_t fmt = half ? 0u : 1u;
  s.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)s.a_mn << 15) | ((uint32_t)s.b_mn << 16) | ((uint32_t)(s.bn >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
  CUtensorMap am, bm;
  if (!encode(&am, oa, half, m, k, kRows) || !encode(&bm, ob, half, n, k, s.bn / 2)) return GTK_ERR_CUDA;
  const GemmEpilogue ep{out, out_ld, bias, add, add_ld, act, z, z_ld, q, q_ld, e8, e_ld, h, h_ld, sums, db, a_pieces == 2 ? a_most : nullptr, b_most};
  const int tiles = s.tiles_m * s.tiles_n, pairs = info->sms / 2;
  const int grid = 2 * (s.splits > 1 ? tiles * s.splits : tiles < pairs ? tiles : pairs);
  const size_t shared = (size_t)stage_bytes * s.stages + fixed;
  const cudaStream_t stream = (cudaStream_t)stream_;
  cudaError_t err;
  switch (type) {
    case kF32: err = launch_gemm<float>(info->device, slope, grid, shared, stream, am, bm, s, ep); break;
    case kF16: err = launch_gemm<__half>(info->device, slope, grid, shared, stream, am, bm, s, ep); break;
    case kBF16: err = launch_gemm<__nv_bfloat16>(info->device, slope, grid, shared, stream, am, bm, s, ep); break;
    default: return GTK_ERR_ARG;
  }
  gtk_count_launch(1);
  if (err != cudaSuccess) return GTK_ERR_CUDA;
  const int lines = (s.m + 31) / 32;
  if (!db || lines == 1) return GTK_OK;
  switch (type) {
    case kF32: err = launch_col_finish<float>(sums, lines, n, n, (float*)db, (float*)nullptr, (float*)nullptr, stream); break;
    case kF16: err = launch_col_finish<__half>(sums, lines, n, n, (__half*)db, (__half*)nullptr, (__half*)nullptr, stream); break;
    default: err = launch_col_finish<__nv_bfloat16>(sums, lines, n, n, (__nv_bfloat16*)db, (__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr, stream); break;
  }
  gtk_count_launch(1);
  return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}
