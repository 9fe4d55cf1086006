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
// out is below 2^-26.  The tensor cores cut a sum to 24 bits where they add to it instead of rounding it, which over
// the 6 * 1500 / 16 additions of K = 1500 took 1e-5 off the result (measured; f32 summed in order: 7e-7).  So the large
// product has an accumulator apart from the five small ones, and every 256 of k both are added to f32 registers of the
// epilogue's warps and begun again.
//
// A CTA computes tiles of 128 x bn.  One thread brings operand tiles to shared memory by TMA, one issues tcgen05.mma
// on them into TMEM, eight warps take finished accumulators out of TMEM and through a padded buffer in shared memory,
// so that a warp's accesses to global memory run along rows.  Two accumulators alternate: the epilogue of a tile
// overlaps the products of the next.
//
// Every wait ends: after a time limit the waiter raises the CTA's abort flag and the status word, everybody leaves
// after its copies and products in flight, and TMEM is freed.
#include <cuda.h>

#include "colsum.cuh"
#include "common.cuh"
#include "host_api.h"
#include "launch.cuh"

namespace gtk {

constexpr int kTileM = 128;
constexpr int kTileK = 64;            // 128 bytes of 16-bit elements: one swizzle span
constexpr int kGemmThreads = 384;     // warp 0 loads, warp 1 multiplies, warps 4 to 11 are the epilogue
constexpr int kEpiWarps = 8;
constexpr int kStagePitch = 33;       // floats a row of the epilogue's buffer: no bank conflict along or across
constexpr int kEpiBytes = kEpiWarps * 32 * kStagePitch * 4;
constexpr int kMaxStages = 8;
constexpr int kF32Blocks = 4;         // f32: blocks of k that are summed in TMEM before they go to registers
constexpr int kMaxShared = 227 * 1024;
constexpr unsigned long long kWaitLimitNs = 2000000000ull;

__device__ unsigned int g_gemm_status;   // not 0: a wait ran out (its place in the code)

struct GemmShape {
  int m, n, k;
  int tiles_m, tiles_n, blocks_k;
  int bn, stages;
  int a_pieces, b_pieces;
  int a_mn, b_mn;                      // 1: mn-major
  uint32_t idesc;
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
};

// ---- PTX ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
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
// False where the CTA has given up; then nothing may be assumed about what was waited for.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint32_t where) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  for (uint32_t spins = 1;; ++spins) {
    if (mbar_try(bar, parity)) return true;
    if ((spins & 63u) == 0u) {
      if (*abort) return false;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        *abort = 1;
        atomicCAS(&g_gemm_status, 0u, where);
        return false;
      }
    }
  }
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, int piece, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map),
               "r"(x), "r"(y), "r"(piece), "r"(bar)
               : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle.  k-major: rows of 128 bytes, 8 rows (1024 bytes) to the next
// group.  mn-major: 64 elements of m or n by 8 of k are 1024 bytes, the next 8 of k follow, the next 64 of m or n
// are `lead` bytes further.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma(uint32_t tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The barrier is arrived on when all products issued before by this thread are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
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
  if (b_pieces == 3) {
    *list = 0x048u;      // (0,2), (0,1), (0,0)
    return 3;
  }
  *list = 0;
  return 1;
}

// ---- epilogue of 32 rows by 32 columns: a warp, whose lanes are columns ---------------------------------------------
struct Patch {
  const float* at;      // [32][kStagePitch]
  int row0, col, rows;  // first row, this lane's column, rows inside the matrix
  bool inside;          // the lane's column is
};

template <typename T>
__device__ __forceinline__ void finish_forward(const Patch& p, const GemmShape& s, const GemmEpilogue& e) {
  const float bias = p.inside && e.bias ? to_f32(((const T*)e.bias)[p.col]) : 0.f;
  with_act(e.act, [&](auto A) {
#pragma unroll 4
    for (int r = 0; r < 32; ++r) {
      if (r >= p.rows) break;
      const long long row = p.row0 + r;
      const float z = p.at[r * kStagePitch + (int)lane_id()] + bias;
      if (e.q) {
        const uint32_t bits = p.inside ? __float_as_uint(z) & 0x7fffffffu : 0u;
        const uint32_t byte = block8_byte(__reduce_max_sync(0xffffffffu, bits));
        e.q[row * e.q_ld + p.col] = p.inside ? (signed char)block8_code(z, byte) : (signed char)0;
        if (lane_id() == 0) e.e[row * e.e_ld + p.col / kBlock8] = (unsigned char)byte;
      }
      if (p.inside) {
        if (e.z) ((T*)e.z)[row * e.z_ld + p.col] = from_f32<T>(z);
        float y = act_value<decltype(A)::value>(z);
        if (e.add) y += to_f32(((const T*)e.add)[row * e.add_ld + p.col]);
        ((T*)e.out)[row * e.out_ld + p.col] = from_f32<T>(y);
      }
    }
  });
}

template <typename T>
__device__ __forceinline__ float finish_slope(const Patch& p, const GemmShape& s, const GemmEpilogue& e) {
  float sum = 0.f;
  if (p.inside)
    with_act(e.act, [&](auto A) {
#pragma unroll 4
      for (int r = 0; r < 32; ++r) {
        if (r >= p.rows) break;
        const long long row = p.row0 + r;
        const float z = e.q ? (float)e.q[row * e.q_ld + p.col] * block8_scale(e.e[row * e.e_ld + p.col / kBlock8]) : to_f32(((const T*)e.z)[row * e.z_ld + p.col]);
        float h;
        const float dz = p.at[r * kStagePitch + (int)lane_id()] * act_slope<decltype(A)::value>(z, &h);
        sum += dz;
        ((T*)e.out)[row * e.out_ld + p.col] = from_f32<T>(dz);
        if (e.h) ((T*)e.h)[row * e.h_ld + p.col] = from_f32<T>(h);
      }
    });
  return sum;
}

// T: type of what the epilogue reads and writes.  SLOPE: the input gradient through the layer before's activation.
template <typename T, bool SLOPE>
__global__ void __launch_bounds__(kGemmThreads, 1)
k8_gemm(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const GemmShape s, GemmEpilogue e) {
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t bars[2 * kMaxStages + 4];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int abort;
  const int warp = (int)(threadIdx.x >> 5);
  uint8_t* base = raw + ((1024u - (smem_addr(raw) & 1023u)) & 1023u);
  const uint32_t a_bytes = (uint32_t)s.a_pieces * kTileM * 128u, stage_bytes = a_bytes + (uint32_t)s.b_pieces * s.bn * 128u;
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
      mbar_init(acc_empty + 8u * i, kEpiWarps);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&a_map) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&b_map) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&tmem_at)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    tc_fence_before();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  pdl_begin(e.bias, e.add, e.z, e.q, e.e);
  const int n_tiles = s.tiles_m * s.tiles_n;

  if (warp == 0) {
    if (lane_id() == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = (int)blockIdx.x; ok && tile < n_tiles; tile += (int)gridDim.x) {
        int tm, tn;
        tile_at(s, tile, &tm, &tn);
        for (int kb = 0; kb < s.blocks_k; ++kb) {
          ok = mbar_wait(empty + 8u * stage, phase ^ 1u, &abort, 1);
          if (!ok) break;
          mbar_expect(full + 8u * stage, stage_bytes);
          const uint32_t dst = tiles + (uint32_t)stage * stage_bytes;
          load_operand(dst, &a_map, s.a_mn, s.a_pieces, kTileM, tm * kTileM, kb * kTileK, full + 8u * stage);
          load_operand(dst + a_bytes, &b_map, s.b_mn, s.b_pieces, s.bn, tn * s.bn, kb * kTileK, full + 8u * stage);
          if (++stage == s.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // No arrival is left under way: the consumer has freed every stage.
      for (int i = 0; ok && i < s.stages; ++i) {
        ok = mbar_wait(empty + 8u * stage, phase ^ 1u, &abort, 5);
        if (++stage == s.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok)   // given up: the copies under way end
        for (int i = 0; i < s.stages; ++i) {
          const bool second = i >= stage;   // this stage's last copy belongs to the round before
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try(full + 8u * i, second ? phase ^ 1u : phase) && globaltimer_ns() - t0 < 100000000ull) {
          }
        }
    }
  } else if (warp == 1) {
    if (lane_id() == 0) {
      int stage = 0;
      uint32_t phase = 0, list;
      const int products = piece_products(s.a_pieces, s.b_pieces, &list);
      const uint32_t a_step = s.a_mn ? 2048u : 32u, b_step = s.b_mn ? 2048u : 32u;   // bytes to the next 16 of k
      const uint32_t a_lead = s.a_mn ? 8192u : 16u, b_lead = s.b_mn ? 8192u : 16u;
      int turn = 0;
      bool ok = true;
      for (int tile = (int)blockIdx.x; ok && tile < n_tiles; tile += (int)gridDim.x)
        for (int kb = 0; ok && kb < s.blocks_k; ++turn) {
          const int acc = turn & 1, stop = min(kb + run, s.blocks_k);
          ok = mbar_wait(acc_empty + 8u * acc, ((uint32_t)(turn >> 1) & 1u) ^ 1u, &abort, 2);
          if (!ok) break;
          tc_fence_after();
          const uint32_t large = tmem + (uint32_t)acc * acc_columns, small = kSplit ? large + (uint32_t)s.bn : large;
          uint32_t on_large = 0, on_small = 0;   // whether the accumulator holds something already
          for (; kb < stop; ++kb) {
            ok = mbar_wait(full + 8u * stage, phase, &abort, 3);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a0 = tiles + (uint32_t)stage * stage_bytes, b0 = a0 + a_bytes;
            for (int i = 0; i < products; ++i) {
              const uint32_t pair = (list >> (4 * i)) & 15u;
              const uint32_t a1 = a0 + (pair & 3u) * (kTileM * 128u), b1 = b0 + (pair >> 2) * (uint32_t)(s.bn * 128);
              const bool to_small = kSplit && pair != 0;
              uint32_t on = to_small ? on_small : on_large;
#pragma unroll
              for (int k = 0; k < kTileK / 16; ++k) {
                mma(to_small ? small : large, operand_desc(a1 + k * a_step, a_lead), operand_desc(b1 + k * b_step, b_lead), s.idesc, on);
                on = 1;
              }
              if (to_small) on_small = 1;
              else on_large = 1;
            }
            mma_commit(empty + 8u * stage);
            if (++stage == s.stages) {
              stage = 0;
              phase ^= 1u;
            }
          }
          if (!ok) break;
          mma_commit(acc_full + 8u * acc);
        }
      if (!ok) {   // products in flight end before TMEM is given back: nobody else arrives on acc_full any more
        const uint32_t last = acc_full + 8u * (turn & 1);
        mma_commit(last);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try(last, (uint32_t)(turn >> 1) & 1u) && globaltimer_ns() - t0 < 100000000ull) {
        }
      }
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, half = (warp - 4) >> 2;
    float* patch = patches + (size_t)(warp - 4) * 32 * kStagePitch;
    const int lane = (int)lane_id();
    int turn = 0;
    bool ok = true;
    for (int tile = (int)blockIdx.x; ok && tile < n_tiles; tile += (int)gridDim.x) {
      int tm, tn;
      tile_at(s, tile, &tm, &tn);
      const int row0 = tm * kTileM + quad * 32;
      // 32 columns of this warp's 32 rows, a row per lane
      auto finish = [&](int c, const auto& v) {
        const int col0 = tn * s.bn + c;
        if (row0 >= s.m || col0 >= s.n) return;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; ++i) patch[lane * kStagePitch + i] = v[i];
        __syncwarp();
        const Patch p{patch, row0, col0 + lane, min(32, s.m - row0), col0 + lane < s.n};
        if constexpr (SLOPE) {
          const float sum = finish_slope<T>(p, s, e);
          if (e.sums && p.inside) e.sums[(size_t)(tm * 4 + quad) * s.n + p.col] = sum;
        } else {
          finish_forward<T>(p, s, e);
        }
      };
      const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
      if constexpr (kSplit) {   // bn is 128 at most: two patches a warp
        float sum[2][32];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int i = 0; i < 32; ++i) sum[j][i] = 0.f;
        for (int kb = 0; kb < s.blocks_k; kb += run, ++turn) {
          const int acc = turn & 1;
          ok = mbar_wait(acc_full + 8u * acc, (uint32_t)(turn >> 1) & 1u, &abort, 4);
          if (!ok) break;
          __syncwarp();
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int c = half * 32 + j * 64;
            if (c < s.bn) {
              float large[32], small[32];
              tmem_load32(lanes + (uint32_t)acc * acc_columns + (uint32_t)c, large);
              tmem_load32(lanes + (uint32_t)acc * acc_columns + (uint32_t)(s.bn + c), small);
#pragma unroll
              for (int i = 0; i < 32; ++i) sum[j][i] += large[i] + small[i];
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty + 8u * acc);
        }
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          if (half * 32 + j * 64 < s.bn) finish(half * 32 + j * 64, sum[j]);
      } else {
        const int acc = turn & 1;
        ok = mbar_wait(acc_full + 8u * acc, (uint32_t)(turn >> 1) & 1u, &abort, 4);
        if (!ok) break;
        __syncwarp();
        tc_fence_after();
        for (int c = half * 32; c < s.bn; c += 64) {
          float v[32];
          tmem_load32(lanes + (uint32_t)acc * acc_columns + (uint32_t)c, v);
          finish(c, v);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(acc_empty + 8u * acc);
        ++turn;
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(columns) : "memory");
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
  return o.p && (uintptr_t)o.p % 16 == 0 && o.ld > 0 && o.ld % 8 == 0 && (o.pieces == 1 || (o.pieces == 3 && o.piece_stride > 0 && o.piece_stride % 8 == 0));
}

// Columns of a tile: the width with the least work on the longest-running SM.
inline int pick_bn(long long m, long long n, int most, int sms) {
  int best = 64;
  long long least = -1;
  for (int bn = 64; bn <= most; bn *= 2) {
    const long long tiles = ((m + kTileM - 1) / kTileM) * ((n + bn - 1) / bn);
    const long long cost = ((tiles + sms - 1) / sms) * (bn + 32);
    if (least < 0 || cost <= least) {
      least = cost;
      best = bn;
    }
  }
  return best;
}

template <typename T>
cudaError_t launch_gemm(bool slope, int grid, size_t shared, cudaStream_t stream, const CUtensorMap& a, const CUtensorMap& b, const GemmShape& s,
                        const GemmEpilogue& e) {
  auto go = [&](auto kernel) {
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxShared - 1024);
    if (err != cudaSuccess) return err;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a, b, s, e);
  };
  return slope ? go(k8_gemm<T, true>) : go(k8_gemm<T, false>);
}

}  // namespace gtk

using namespace gtk;

// Lines of n floats that `sums` has to hold for m rows.
extern "C" long long gtk_k8_sum_lines(long long m) { return (m + 31) / 32; }

// Status word of the current device's products: 0, or where a wait ran out.  Synchronises.
extern "C" unsigned int gtk_k8_status(void) {
  unsigned int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_gemm_status, sizeof(v)) != cudaSuccess) return ~0u;
  return v;
}

// out[m][n] = epilogue(sum_k a[m][k] b[n][k]).  type: of what the epilogue reads and writes.  half: the operands are
// f16, else bf16.  Leading dimensions and piece strides of operands are multiples of 8 elements, their addresses of
// 16 bytes.  slope: see the top of this file.  sums with db: the sums over all rows of what the slope form stores.
extern "C" int gtk_k8_gemm(int type, int half, long long m, long long n, long long k, const void* a, long long a_ld, int a_pieces, long long a_stride, int a_mn,
                           const void* b, long long b_ld, int b_pieces, long long b_stride, int b_mn, void* out, long long out_ld, const void* bias,
                           const void* add, long long add_ld, int act, int slope, void* z, long long z_ld, signed char* q, long long q_ld, unsigned char* e8,
                           long long e_ld, void* h, long long h_ld, float* sums, void* db, void* stream_) {
  const Operand oa{a, a_ld, a_pieces, a_stride, a_mn != 0}, ob{b, b_ld, b_pieces, b_stride, b_mn != 0};
  if (m <= 0 || n <= 0 || k <= 0 || !out || act < 0 || act >= kActCount || !operand_ok(oa) || !operand_ok(ob) || (q && !e8) || (q && !slope && q_ld < (n + kBlock8 - 1) / kBlock8 * kBlock8) || (sums == nullptr) != (db == nullptr))
    return GTK_ERR_ARG;
  if (m > 0x7fffff00LL || n > 0x7fffff00LL || k > 0x7fffff00LL) return GTK_ERR_UNSUPPORTED;
  const DeviceInfo* info = gtk_device_info();
  if (!info) return GTK_ERR_CUDA;
  GemmShape s{};
  s.m = (int)m;
  s.n = (int)n;
  s.k = (int)k;
  s.a_pieces = a_pieces;
  s.b_pieces = b_pieces;
  s.a_mn = oa.mn_major;
  s.b_mn = ob.mn_major;
  s.bn = pick_bn(m, n, a_pieces * b_pieces > 1 ? 128 : 256, info->sms);
  s.tiles_m = (int)((m + kTileM - 1) / kTileM);
  s.tiles_n = (int)((n + s.bn - 1) / s.bn);
  s.blocks_k = (int)((k + kTileK - 1) / kTileK);
  if ((long long)s.tiles_m * s.tiles_n > 0x3fffffffLL) return GTK_ERR_UNSUPPORTED;
  const int stage_bytes = a_pieces * kTileM * 128 + b_pieces * s.bn * 128;
  const int fixed = 1024 + kEpiBytes;
  s.stages = (kMaxShared - 1024 - fixed) / stage_bytes;
  if (s.stages > kMaxStages) s.stages = kMaxStages;
  const uint32_t fmt = half ? 0u : 1u;
  s.idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)s.a_mn << 15) | ((uint32_t)s.b_mn << 16) | ((uint32_t)(s.bn >> 3) << 17) | ((kTileM >> 4) << 24);
  CUtensorMap am, bm;
  if (!encode(&am, oa, half, m, k, kTileM) || !encode(&bm, ob, half, n, k, s.bn)) return GTK_ERR_CUDA;
  const GemmEpilogue ep{out, out_ld, bias, add, add_ld, act, z, z_ld, q, q_ld, e8, e_ld, h, h_ld, sums};
  const int tiles = s.tiles_m * s.tiles_n, grid = tiles < info->sms ? tiles : info->sms;
  const size_t shared = (size_t)stage_bytes * s.stages + fixed;
  const cudaStream_t stream = (cudaStream_t)stream_;
  cudaError_t err;
  switch (type) {
    case kF32: err = launch_gemm<float>(slope, grid, shared, stream, am, bm, s, ep); break;
    case kF16: err = launch_gemm<__half>(slope, grid, shared, stream, am, bm, s, ep); break;
    case kBF16: err = launch_gemm<__nv_bfloat16>(slope, grid, shared, stream, am, bm, s, ep); break;
    default: return GTK_ERR_ARG;
  }
  gtk_count_launch(1);
  if (err != cudaSuccess) return GTK_ERR_CUDA;
  if (!db) return GTK_OK;
  const int lines = (s.m + 31) / 32;
  switch (type) {
    case kF32: err = launch_col_finish<float>(sums, lines, n, n, (float*)db, (float*)nullptr, stream); break;
    case kF16: err = launch_col_finish<__half>(sums, lines, n, n, (__half*)db, (__half*)nullptr, stream); break;
    default: err = launch_col_finish<__nv_bfloat16>(sums, lines, n, n, (__nv_bfloat16*)db, (__nv_bfloat16*)nullptr, stream); break;
  }
  gtk_count_launch(1);
  return err == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}
