// K6's entry points: layer norm forward, and backward by itself (k6_norm.cuh has the kernels and their reasons).
#include "k6_norm.cuh"

namespace gtk {

template <typename T>
int norm_forward(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, NormShape s, cudaStream_t stream) {
  const int vec = pick_vec<T>(s.cols, {{x, s.x_ld}, {w, 0}, {b, 0}, {y, s.y_ld}});
  const bool async = ring_async(vec);
  const NormPlan p = norm_plan(s.rows, s.cols, vec, async, 32);
  s.warps = p.warps;
  cudaError_t e = cudaSuccess;
  if (p.nv == 0) {
    const long long grid = s.rows < 65535 ? s.rows : 65535;
    e = launch_pdl(k6_norm_forward_long<T>, dim3((unsigned)grid), dim3(1024), stream, (const T*)x, (const T*)w, (const T*)b, (T*)y, mean, rstd, s);
  } else {
    // CTAs of 512 threads, two of which fill an SM's registers; few rows: one a CTA, to spread them over the SMs
    int groups = 16 / p.warps > 8 ? 8 : 16 / p.warps > 1 ? 16 / p.warps : 1;
    while (groups > 1 && s.rows < 148LL * groups) --groups;
    const int ctas = 32 / (p.warps * groups);
    const size_t slot = (size_t)groups * p.warps * 32 * p.nv * p.vec * sizeof(T);
    s.depth = ring_depth(slot, (size_t)kNormShared / ctas);
    const long long all = (s.rows + groups - 1) / groups, grid = all < 148LL * ctas ? all : 148LL * ctas;
    while (s.depth > 1 && ((s.depth - 1) * grid >= all || !async)) --s.depth;
    if (!with_plan<T>(p, [&](auto V, auto N) {
          e = launch_norm<k6_norm_forward<T, decltype(V)::value, decltype(N)::value>>(grid, p.warps, groups, slot * s.depth, stream, (const T*)x, (const T*)w,
                          (const T*)b, (T*)y, mean, rstd, s);
        }))
      return GTK_ERR_UNSUPPORTED;
  }
  gtk_count_launch(1);
  return e == cudaSuccess ? GTK_OK : GTK_ERR_CUDA;
}

}  // namespace gtk

using namespace gtk;

// x: rows of `cols` elements, x_ld apart; y's are y_ld apart; w and b may be null.
extern "C" int gtk_k6_norm_forward(int type, const void* x, long long x_ld, const void* w, const void* b, void* y, long long y_ld, float* mean, float* rstd,
                                   long long rows, long long cols, float eps, void* stream) {
  if (rows <= 0 || cols <= 0 || cols > 0x3fffffff || x_ld < 0 || y_ld < cols) return GTK_ERR_ARG;
  const NormShape s{rows, x_ld, 0, 0, y_ld, (int)cols, 1, 1, eps};
  switch (type) {
    case kF32: return norm_forward<float>(x, w, b, y, mean, rstd, s, (cudaStream_t)stream);
    case kF16: return norm_forward<__half>(x, w, b, y, mean, rstd, s, (cudaStream_t)stream);
    case kBF16: return norm_forward<__nv_bfloat16>(x, w, b, y, mean, rstd, s, (cudaStream_t)stream);
  }
  return GTK_ERR_ARG;
}

// Lines of 2 * cols (with y: 3 * cols) floats that `partial` has to hold.
extern "C" int gtk_k6_norm_lines(void) { return kNormLines; }

// dx dense; add (may be null): a gradient that is added to dx; dw, db may be null.  With y (rows of up to 16384 elements,
// and w, b, add, dw, db, dadd): the norm's output is made again there, and dadd is the sum of add over the rows; x may
// then be codes, with exponents e.
extern "C" int gtk_k6_norm_backward(int type, const void* dy, long long dy_ld, const void* x, long long x_ld, const unsigned char* e, long long e_ld,
                                    const float* mean, const float* rstd, const void* w, const void* b, const void* add, long long add_ld, void* dx,
                                    void* dw, void* db, void* y, long long y_ld, void* dadd, float* partial, long long rows, long long cols,
                                    void* stream_) {
  if (rows <= 0 || cols <= 0 || cols > 0x3fffffff || x_ld < 0 || dy_ld < 0 || add_ld < 0 || ((dw || db) && !partial)) return GTK_ERR_ARG;
  if (y ? (!w || !b || !add || !dw || !db || !dadd || y_ld < cols) : (e || dadd)) return GTK_ERR_ARG;
  const NormShape s{rows, x_ld, dy_ld, add_ld, y_ld, (int)cols, 1, 1, 0.f};
  const cudaStream_t stream = (cudaStream_t)stream_;
  auto of = [&](auto t) -> int {
    using T = decltype(t);
    const NormMore<T> more{e, e_ld, (const T*)b, (T*)y, (T*)dadd};
    if (!y) return norm_backward<T, T, false>(dy, x, mean, rstd, w, add, dx, dw, db, partial, s, NormMore<T>{}, stream);
    return norm_backward_block<T>(e != nullptr, dy, x, mean, rstd, w, add, dx, dw, db, partial, s, more, stream);
  };
  switch (type) {
    case kF32: return of(float{});
    case kF16: return of(__half{});
    case kBF16: return of(__nv_bfloat16{});
  }
  return GTK_ERR_ARG;
}
