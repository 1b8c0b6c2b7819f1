// Layer norm over the last axis with an optional residual add, forward and
// backward, for gfx950.
//
//   z = x + residual           (in fp32; never rounded, never stored)
//   mean = sum(z) / H          rstd = 1 / sqrt(sum((z - mean)^2) / H + eps)
//   n = (z - mean) * rstd      y = n * weight + bias
// backward, with g = dy * weight:
//   dz = rstd * (g - mean(g) - n * mean(g * n))    dx = dresidual = dz
//   dweight = sum over rows of dy * n              dbias = sum over rows of dy
//
// The backward reads x and the residual again and adds them again: as many
// bytes as a stored z would cost, and no rounding of z in between. Sums and
// statistics are fp32; results are rounded once, to their own type.
#include <hip/hip_runtime.h>

#include "lm_common.h"

namespace {

using namespace dear_lm;

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 1 << 20;   // a launch holds under 2^32 threads

template <typename TX, typename TR, bool RES>
__device__ __forceinline__ float load_z(const TX* x, const TR* r, int i) {
  float z = to_f(x[i]);
  if constexpr (RES) z += to_f(r[i]);
  return z;
}

template <typename TX, typename TR, typename TY, bool RES>
__global__ __launch_bounds__(kThreads) void ln_fwd_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const void* __restrict__ w, const void* __restrict__ b, int wtype,
    TY* __restrict__ y, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, int64_t rows, int H, float eps) {
  __shared__ float scratch[kThreads / 64];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TX* xr = x + row * xs;
    const TR* rr = RES ? r + row * rs : nullptr;
    float s = 0.f;
    for (int i = threadIdx.x; i < H; i += kThreads)
      s += load_z<TX, TR, RES>(xr, rr, i);
    const float mean = block_reduce(s, Add{}, scratch) / (float)H;
    float v = 0.f;
    for (int i = threadIdx.x; i < H; i += kThreads) {
      const float d = load_z<TX, TR, RES>(xr, rr, i) - mean;
      v += d * d;
    }
    const float var = block_reduce(v, Add{}, scratch) / (float)H;
    const float rstd = 1.0f / sqrtf(var + eps);
    for (int i = threadIdx.x; i < H; i += kThreads) {
      float n = (load_z<TX, TR, RES>(xr, rr, i) - mean) * rstd;
      if (w) n *= load_as_float(w, wtype, i);
      if (b) n += load_as_float(b, wtype, i);
      y[row * H + i] = static_cast<TY>(n);
    }
    if (mean_out && threadIdx.x == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
  }
}

template <typename TX, typename TR, typename TY, bool RES>
__global__ __launch_bounds__(kThreads) void ln_bwd_dx_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const TY* __restrict__ dy, int64_t dys, const void* __restrict__ w,
    int wtype, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, TX* __restrict__ dx,
    TR* __restrict__ dr, int64_t rows, int H) {
  __shared__ float scratch[kThreads / 64];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TX* xr = x + row * xs;
    const TR* rr = RES ? r + row * rs : nullptr;
    const TY* gr = dy + row * dys;
    const float mean = mean_in[row], rstd = rstd_in[row];
    float sg = 0.f, sgn = 0.f;
    for (int i = threadIdx.x; i < H; i += kThreads) {
      float g = to_f(gr[i]);
      if (w) g *= load_as_float(w, wtype, i);
      sg += g;
      sgn += g * ((load_z<TX, TR, RES>(xr, rr, i) - mean) * rstd);
    }
    sg = block_reduce(sg, Add{}, scratch) / (float)H;
    sgn = block_reduce(sgn, Add{}, scratch) / (float)H;
    for (int i = threadIdx.x; i < H; i += kThreads) {
      float g = to_f(gr[i]);
      if (w) g *= load_as_float(w, wtype, i);
      const float n = (load_z<TX, TR, RES>(xr, rr, i) - mean) * rstd;
      const float dz = rstd * (g - sg - n * sgn);
      if (dx) dx[row * H + i] = static_cast<TX>(dz);
      if (RES && dr) dr[row * H + i] = static_cast<TR>(dz);
    }
  }
}

// Column sums of dy * n and of dy over one stripe of rows: part[stripe][2][H].
template <typename TX, typename TR, typename TY, bool RES>
__global__ __launch_bounds__(kThreads) void ln_bwd_dw_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const TY* __restrict__ dy, int64_t dys, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, float* __restrict__ part, int64_t rows,
    int H) {
  __shared__ float sw[4][64], sb[4][64];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int col = blockIdx.y * 64 + lane;
  float aw = 0.f, ab = 0.f;
  if (col < H)
    for (int64_t row = (int64_t)blockIdx.x * 4 + sub; row < rows;
         row += (int64_t)gridDim.x * 4) {
      const float g = to_f(dy[row * dys + col]);
      const float z = load_z<TX, TR, RES>(x + row * xs,
                                          RES ? r + row * rs : nullptr, col);
      aw += g * ((z - mean_in[row]) * rstd_in[row]);
      ab += g;
    }
  sw[sub][lane] = aw;
  sb[sub][lane] = ab;
  __syncthreads();
  if (sub == 0 && col < H) {
    float* p = part + (int64_t)blockIdx.x * 2 * H;
    p[col] = (sw[0][lane] + sw[1][lane]) + (sw[2][lane] + sw[3][lane]);
    p[H + col] = (sb[0][lane] + sb[1][lane]) + (sb[2][lane] + sb[3][lane]);
  }
}

__global__ __launch_bounds__(kThreads) void ln_dw_join_kernel(
    const float* __restrict__ part, int nparts, int H, void* __restrict__ dw,
    void* __restrict__ db, int wtype) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= 2 * H) return;
  void* out = i < H ? dw : db;
  if (!out) return;
  float s = 0.f;
  for (int k = 0; k < nparts; ++k) s += part[(int64_t)k * 2 * H + i];
  store_as(out, wtype, i < H ? i : i - H, s);
}

template <typename TX, typename TR, typename TY, bool RES>
void fwd(hipStream_t st, const void* x, int64_t xs, const void* r, int64_t rs,
         const void* w, const void* b, int wtype, void* y, float* mean,
         float* rstd, int64_t rows, int H, float eps) {
  const int grid = (int)(rows < kMaxBlocks ? rows : kMaxBlocks);
  hipLaunchKernelGGL((ln_fwd_kernel<TX, TR, TY, RES>), dim3(grid), dim3(kThreads), 0, st, 
      (const TX*)x, xs, (const TR*)r, rs, w, b, wtype, (TY*)y, mean, rstd,
      rows, H, eps);
}

template <typename TX, typename TR, typename TY, bool RES>
void bwd(hipStream_t st, const void* x, int64_t xs, const void* r, int64_t rs,
         const void* dy, int64_t dys, const void* w, int wtype,
         const float* mean, const float* rstd, void* dx, void* dr, void* dw,
         void* db, float* part, int nparts, int64_t rows, int H) {
  if (dx || dr) {
    const int grid = (int)(rows < kMaxBlocks ? rows : kMaxBlocks);
    hipLaunchKernelGGL((ln_bwd_dx_kernel<TX, TR, TY, RES>), dim3(grid), dim3(kThreads), 0, st, 
        (const TX*)x, xs, (const TR*)r, rs, (const TY*)dy, dys, w, wtype, mean,
        rstd, (TX*)dx, (TR*)dr, rows, H);
  }
  if (dw || db) {
    hipLaunchKernelGGL((ln_bwd_dw_kernel<TX, TR, TY, RES>), dim3(dim3(nparts, (H + 63) / 64)), dim3(kThreads), 0, st, 
            (const TX*)x, xs, (const TR*)r, rs, (const TY*)dy, dys, mean, rstd,
            part, rows, H);
    hipLaunchKernelGGL((ln_dw_join_kernel), dim3((2 * H + kThreads - 1) / kThreads), dim3(kThreads), 0, st, 
        part, nparts, H, dw, db, wtype);
  }
}

}  // namespace

// The pairs (x, residual) that exist; rtype < 0: no residual. The result has
// the wider type, which is the residual's.
#define LN_DISPATCH(CALL)                                                     \
  if (rtype < 0) {                                                            \
    if (xtype == kF32) CALL(float, float, float, false);                      \
    else if (xtype == kBF16) CALL(bf16, bf16, bf16, false);                   \
    else CALL(f16, f16, f16, false);                                          \
  } else if (xtype == rtype) {                                                \
    if (xtype == kF32) CALL(float, float, float, true);                       \
    else if (xtype == kBF16) CALL(bf16, bf16, bf16, true);                    \
    else CALL(f16, f16, f16, true);                                           \
  } else if (xtype == kBF16) CALL(bf16, float, float, true);                  \
  else CALL(f16, float, float, true)

// Floats of workspace that the backward's column sums need.
int64_t dear_ln_parts(int64_t rows, int H) {
  const int64_t stripes = (rows + 31) / 32;
  return stripes < 256 ? stripes : 256;
}

int dear_ln_fwd(hipStream_t st, int xtype, int rtype, int wtype, const void* x,
                int64_t xs, const void* r, int64_t rs, const void* w,
                const void* b, void* y, float* mean, float* rstd, int64_t rows,
                int H, float eps) {
#define CALL(TX, TR, TY, RES)                                                 \
  fwd<TX, TR, TY, RES>(st, x, xs, r, rs, w, b, wtype, y, mean, rstd, rows, H, \
                       eps)
  LN_DISPATCH(CALL);
#undef CALL
  return (int)hipGetLastError();
}

int dear_ln_bwd(hipStream_t st, int xtype, int rtype, int wtype, const void* x,
                int64_t xs, const void* r, int64_t rs, const void* dy,
                int64_t dys, const void* w, const float* mean,
                const float* rstd, void* dx, void* dr, void* dw, void* db,
                float* part, int nparts, int64_t rows, int H) {
#define CALL(TX, TR, TY, RES)                                                 \
  bwd<TX, TR, TY, RES>(st, x, xs, r, rs, dy, dys, w, wtype, mean, rstd, dx,   \
                       dr, dw, db, part, nparts, rows, H)
  LN_DISPATCH(CALL);
#undef CALL
  return (int)hipGetLastError();
}
