// Layer norm over the last axis with an optional residual add, forward and
// backward, for gfx950.
//
//   z = x + residual           (an fp32 sum; never stored)
//   mean = sum(z) / H          rstd = 1 / sqrt(sum((z - mean)^2) / H + eps)
//   n = (z - mean) * rstd      y = n * weight + bias
// backward, with g = dy * weight:
//   dz = rstd * (g - mean(g) - n * mean(g * n))    dx = dresidual = dz
//   dweight = sum over rows of dy * n              dbias = sum over rows of dy
//
// The backward reads x and the residual again and adds them again: as many
// bytes as a stored z would cost, and no rounding of z in between. Sums and
// statistics are fp32; results are rounded once, to their own type.
//
// A mean in fp32 is off by some 2^-22 of itself, which may be more than the
// row's whole spread. What it is off by is the mean of the distances to it: that
// is summed with their squares, and kept as a second number. Where it is more
// than an eighth of the spread, the sum of squares says too little, and another
// round is taken from the mean that both numbers give; the distances to that are
// exact, and those of equal elements are 0.
//
// A row lies in the registers of a group of 16, 32, 64, 256 or 1024 threads,
// up to 16 elements of each, so that it is read once. Groups go round the rows
// with their columns' weights, and in the backward their columns' sums of
// dweight and dbias, in registers as well; each block leaves one record of the
// sums, and a second kernel adds the records up in a fixed order. Rows over
// 16384 elements are read again for each pass instead (the *_long kernels).
#include <hip/hip_runtime.h>

#include "lm_common.h"

namespace {

using namespace dear_lm;

constexpr int kMaxBlocks = 1 << 20;   // a launch holds under 2^32 threads
constexpr int kPerThread = 16;        // elements of a row in one thread

// E consecutive elements of type T as they lie in memory.
template <typename T, int E>
struct Chunk {
  static constexpr int kLoads = E / kVec<T>;
  u32x4 raw[kLoads];

  // elements [i, i + E) of a row of H; what lies behind it is zero
  __device__ __forceinline__ void load(const T* row, int i, int H) {
    if (i + E <= H) {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) raw[q] = load16(row + i + q * kVec<T>);
    } else {
#pragma unroll
      for (int q = 0; q < kLoads; ++q) raw[q] = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (i + j < H) put(raw[j / kVec<T>], j % kVec<T>, row[i + j]);
    }
  }
  __device__ __forceinline__ float at(int j) const {
    return elem<T>(raw[j / kVec<T>], j % kVec<T>);
  }
};

template <typename T, int E>
__device__ __forceinline__ void store_chunk(T* row, int i, int H,
                                            const float* v) {
  if (i + E <= H) {
#pragma unroll
    for (int q = 0; q < E / kVec<T>; ++q)
      store16(row + i + q * kVec<T>, pack<T>(v + q * kVec<T>));
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (i + j < H) row[i + j] = static_cast<T>(v[j]);
  }
}

// Sums over a group of G threads, in every one of them. Groups of more than a
// wave are the whole block, and meet at one barrier: `scratch`, two of a wave,
// takes turns.
template <int G>
struct GroupSum {
  float (*scratch)[G > 64 ? G / 64 : 1][2];
  int turn = 0;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    auto step = [&](auto o) {
      a = sum_of(lanes<decltype(o)::value>(a));
      b = sum_of(lanes<decltype(o)::value>(b));
    };
    step(Int<1>{});
    step(Int<2>{});
    step(Int<4>{});
    step(Int<8>{});
    if constexpr (G >= 32) step(Int<16>{});
    if constexpr (G >= 64) step(Int<32>{});
    if constexpr (G > 64) {
      if ((threadIdx.x & 63) == 0) {
        scratch[turn][threadIdx.x >> 6][0] = a;
        scratch[turn][threadIdx.x >> 6][1] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int i = 0; i < G / 64; ++i) {
        a += scratch[turn][i][0];
        b += scratch[turn][i][1];
      }
      turn ^= 1;
    }
  }
  __device__ __forceinline__ float operator()(float a) {
    float none = 0.f;
    (*this)(a, none);
    return a;
  }
};

// What a row leaves for its backward pass: its mean is the sum of two numbers.
// [3][rows]
struct RowNorm {
  float mean, off, rstd;
};
__device__ __forceinline__ void put_stats(float* stats, int64_t rows,
                                          int64_t row, float mean, float off,
                                          float rstd) {
  stats[row] = mean;
  stats[rows + row] = off;
  stats[2 * rows + row] = rstd;
}
__device__ __forceinline__ RowNorm get_stats(const float* stats, int64_t rows,
                                             int64_t row) {
  return {stats[row], stats[rows + row], stats[2 * rows + row]};
}
__device__ __forceinline__ float norm_of(float z, const RowNorm& s) {
  return ((z - s.mean) - s.off) * s.rstd;
}

// E elements a chunk: 16 bytes of the narrowest type.
template <typename TX>
constexpr int kChunk = kVec<TX>;

// A thread's columns of the weight or bias; `none` where there is neither.
template <typename T, int NV, int E>
__device__ __forceinline__ void load_typed(float (&v)[NV * E], const void* p,
                                           int first, int step, int H) {
  Chunk<T, E> c[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    c[i].load(static_cast<const T*>(p), first + i * step, H);
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) v[i * E + j] = c[i].at(j);
}

template <int NV, int E>
__device__ __forceinline__ void load_columns(float (&v)[NV * E], const void* p,
                                             int type, int first, int step,
                                             int H, float none) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < NV * E; ++i) v[i] = none;
  } else if (type == kF32) {
    load_typed<float, NV, E>(v, p, first, step, H);
  } else if constexpr (E == 8) {
    if (type == kBF16) load_typed<bf16, NV, E>(v, p, first, step, H);
    else load_typed<f16, NV, E>(v, p, first, step, H);
  }
}

// Bound by memory: 16384 x 1024, a bf16 branch on an fp32 residual, takes 26 us
// (6.4 TB/s, part of it from the last-level cache; 34 us where nothing of it is
// there), 4096 x 768 fp32 5.9 us. One row takes 2.2 us, a launch's own time.
// 256 threads hold one to sixteen rows: a wave to a row of up to 1024 elements
// needs no barrier, and the lanes' sums go through DPP, not LDS. Against one
// block to a row with elements loaded one by one: 254 us for this pass and the
// backward's, 84 now.
template <typename TX, typename TR, typename TY, bool RES, int G, int NV>
__global__ __launch_bounds__(G > 256 ? G : 256, 4) void ln_fwd_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const void* __restrict__ w, const void* __restrict__ b, int wtype,
    TY* __restrict__ y, float* __restrict__ stats, int64_t rows, int H,
    float eps) {
  constexpr int E = kChunk<TX>, NT = G > 256 ? G : 256, N = NV * E;
  __shared__ float scratch[2][G > 64 ? G / 64 : 1][2];
  GroupSum<G> group_sum{scratch};
  const int first = (int)(threadIdx.x % G) * E;
  float wv[N], bv[N];
  load_columns<NV, E>(wv, w, wtype, first, G * E, H, 1.f);
  load_columns<NV, E>(bv, b, wtype, first, G * E, H, 0.f);
  const float inv_h = 1.0f / (float)H;
  for (int64_t row = (int64_t)blockIdx.x * (NT / G) + threadIdx.x / G;
       row < rows; row += (int64_t)gridDim.x * (NT / G)) {
    Chunk<TX, E> cx[NV];
    Chunk<TR, E> cr[RES ? NV : 1];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      cx[c].load(x + row * xs, first + c * G * E, H);
      if constexpr (RES) cr[c].load(r + row * rs, first + c * G * E, H);
    }
    float z[N], s = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        float v = cx[c].at(j);
        if constexpr (RES) v += cr[c].at(j);
        z[c * E + j] = v;
        s += v;
      }
    // a quotient: a product could be joined with the differences to it, which
    // would then be to another number than this one
    float mean = group_sum(s) / (float)H, off = 0.f, q = 0.f;
    auto inside = [&](int c, int j) { return first + c * G * E + j < H; };
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float d = inside(c, j) ? z[c * E + j] - mean : 0.f;
        z[c * E + j] = d;
        off += d;
        q = fmaf(d, d, q);
      }
    group_sum(off, q);
    // the same in all threads of the group, which meet again in the sums
    off *= inv_h;
    q *= inv_h;
    const bool again = 64.f * off * off > q;
    float var = q - off * off;
    if (again) {
      const float better = mean + off, step = better - mean;
      mean = better;
      off = q = 0.f;
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          if (inside(c, j)) z[c * E + j] -= step;
          off += z[c * E + j];
        }
      off = group_sum(off) * inv_h;
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const float d = inside(c, j) ? z[c * E + j] - off : 0.f;
          q = fmaf(d, d, q);
        }
      var = group_sum(q) * inv_h;
    }
    const float rstd = 1.0f / sqrtf(var + eps);
#pragma unroll
    for (int c = 0; c < NV; ++c) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        z[c * E + j] = fmaf((z[c * E + j] - off) * rstd, wv[c * E + j],
                            bv[c * E + j]);
      store_chunk<TY, E>(y + row * H, first + c * G * E, H, z + c * E);
    }
    if (stats && threadIdx.x % G == 0)
      put_stats(stats, rows, row, mean, off, rstd);
  }
}

// Bound by memory as well: the same case takes 47 us (5.8 TB/s); 4096 x 768
// fp32, 12.7 us, by its few waves. Few blocks, each of many rows, as many as
// leave 256 records: a record per row would be as many bytes again as the
// gradient. Gradients that are stored past the caches are written no faster here
// (93 us for a pass instead of 83): what reads them next then has to fetch them.
template <typename TX, typename TR, typename TY, bool RES, int G, int NV>
__global__ __launch_bounds__(G > 512 ? G : G > 64 ? 256 : 512,
                             G > 512 ? 4 : 2)
void ln_bwd_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const TY* __restrict__ dy, int64_t dys, const void* __restrict__ w,
    int wtype, const float* __restrict__ stats, TX* __restrict__ dx,
    TR* __restrict__ dr, float* __restrict__ records, int64_t rows, int H) {
  constexpr int E = kChunk<TX>, N = NV * E;
  constexpr int NT = G > 512 ? G : G > 64 ? 256 : 512;
  __shared__ float scratch[2][G > 64 ? G / 64 : 1][2];
  GroupSum<G> group_sum{scratch};
  const int first = (int)(threadIdx.x % G) * E;
  float wv[N], aw[N] = {}, ab[N] = {};
  load_columns<NV, E>(wv, w, wtype, first, G * E, H, 1.f);
  const float inv_h = 1.0f / (float)H;
  for (int64_t row = (int64_t)blockIdx.x * (NT / G) + threadIdx.x / G;
       row < rows; row += (int64_t)gridDim.x * (NT / G)) {
    Chunk<TX, E> cx[NV];
    Chunk<TR, E> cr[RES ? NV : 1];
    Chunk<TY, E> cg[NV];
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      cx[c].load(x + row * xs, first + c * G * E, H);
      if constexpr (RES) cr[c].load(r + row * rs, first + c * G * E, H);
      cg[c].load(dy + row * dys, first + c * G * E, H);
    }
    const RowNorm stat = get_stats(stats, rows, row);
    float n[N], g[N], sg = 0.f, sgn = 0.f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = c * E + j;
        float z = cx[c].at(j);
        if constexpr (RES) z += cr[c].at(j);
        n[i] = norm_of(z, stat);
        const float up = cg[c].at(j);
        aw[i] = fmaf(up, n[i], aw[i]);
        ab[i] += up;
        g[i] = up * wv[i];
        sg += g[i];
        sgn = fmaf(g[i], n[i], sgn);
      }
    group_sum(sg, sgn);
    sg *= inv_h;
    sgn *= inv_h;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int i = c * E + j;
        g[i] = stat.rstd * (g[i] - sg - n[i] * sgn);
      }
      if (dx) store_chunk<TX, E>(dx + row * H, first + c * G * E, H, g + c * E);
      if constexpr (RES)
        if (dr)
          store_chunk<TR, E>(dr + row * H, first + c * G * E, H, g + c * E);
    }
  }
  if (!records) return;
  // the block's groups, one after the other: a fixed order
  if constexpr (G < 64) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (G < 32) {
        aw[i] = sum_of(lanes<16>(aw[i]));
        ab[i] = sum_of(lanes<16>(ab[i]));
      }
      aw[i] = sum_of(lanes<32>(aw[i]));
      ab[i] = sum_of(lanes<32>(ab[i]));
    }
  }
  float* record = records + (int64_t)blockIdx.x * 2 * H;
  if constexpr (G > 64) {
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      store_chunk<float, E>(record, first + c * G * E, H, aw + c * E);
      store_chunk<float, E>(record + H, first + c * G * E, H, ab + c * E);
    }
  } else {
    __shared__ float total[2][G * N];
    const int lane = threadIdx.x & 63;
    for (int turn = 0; turn < NT / 64; ++turn) {
      if ((int)threadIdx.x >> 6 == turn && lane < G) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          total[0][i * G + lane] = turn ? total[0][i * G + lane] + aw[i]
                                        : aw[i];
          total[1][i * G + lane] = turn ? total[1][i * G + lane] + ab[i]
                                        : ab[i];
        }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * H; i += NT) {
      const int col = i < H ? i : i - H;
      // element j of chunk c of thread t: column c * G * E + t * E + j
      const int c = col / (G * E), t = col % (G * E) / E, j = col % E;
      record[i] = total[i >= H][(c * E + j) * G + t];
    }
  }
}

// Adds up the records: 64 columns to a block of 1024, 16 threads to a column.
// No atomics, so that the result does not depend on the order of the blocks.
// Bound by latency: 256 records of 2 x 1024 columns, 2 MB, take 4 us.
__global__ __launch_bounds__(1024) void ln_records_kernel(
    const float* __restrict__ records, int n, int H, void* __restrict__ dw,
    void* __restrict__ db, int wtype) {
  __shared__ float part[16][64];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  const int64_t columns = 2 * (int64_t)H;
  for (int64_t first = (int64_t)blockIdx.x * 64; first < columns;
       first += (int64_t)gridDim.x * 64) {
    const int64_t i = first + lane;
    float s = 0.f;
    if (i < columns) {
#pragma unroll 8
      for (int k = sub; k < n; k += 16) s += records[k * columns + i];
    }
    part[sub][lane] = s;
    __syncthreads();
    if (sub == 0 && i < columns) {
      for (int k = 1; k < 16; ++k) s += part[k][lane];
      void* out = i < H ? dw : db;
      if (out) store_as(out, wtype, i < H ? i : i - H, s);
    }
    __syncthreads();                     // before `part` is written again
  }
}

// ------------------------------------------------------------- long rows
// A thread adds up a thousandth of the row: in fp64, for a chain of that many
// float32 additions would be as far off as its length. Three reads of the row,
// by loads of one element: 512 x 20011 fp32 take 47 us forward, 48 backward and
// 15 for the weights' records, where the bytes would take 12 and 18.
constexpr int kLongThreads = 1024;

template <typename TX, typename TR, bool RES>
__device__ __forceinline__ float load_z(const TX* x, const TR* r, int i) {
  float z = to_f(x[i]);
  if constexpr (RES) z += to_f(r[i]);
  return z;
}

template <typename TX, typename TR, typename TY, bool RES>
__global__ __launch_bounds__(kLongThreads) void ln_fwd_long_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const void* __restrict__ w, const void* __restrict__ b, int wtype,
    TY* __restrict__ y, float* __restrict__ stats, int64_t rows, int H,
    float eps) {
  __shared__ double scratch[kLongThreads / 64];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TX* xr = x + row * xs;
    const TR* rr = RES ? r + row * rs : nullptr;
    double s = 0.0, v = 0.0;
    for (int i = threadIdx.x; i < H; i += kLongThreads)
      s += load_z<TX, TR, RES>(xr, rr, i);
    const double mean = block_reduce(s, Add{}, scratch) / H;
    for (int i = threadIdx.x; i < H; i += kLongThreads) {
      const double d = load_z<TX, TR, RES>(xr, rr, i) - mean;
      v += d * d;
    }
    v = block_reduce(v, Add{}, scratch) / H;
    RowNorm stat;
    stat.mean = (float)mean;
    stat.off = (float)(mean - (double)stat.mean);
    stat.rstd = 1.0f / sqrtf((float)v + eps);
    for (int i = threadIdx.x; i < H; i += kLongThreads) {
      float n = norm_of(load_z<TX, TR, RES>(xr, rr, i), stat);
      if (w) n *= load_as_float(w, wtype, i);
      if (b) n += load_as_float(b, wtype, i);
      y[row * H + i] = static_cast<TY>(n);
    }
    if (stats && threadIdx.x == 0)
      put_stats(stats, rows, row, stat.mean, stat.off, stat.rstd);
  }
}

template <typename TX, typename TR, typename TY, bool RES>
__global__ __launch_bounds__(kLongThreads) void ln_bwd_long_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const TY* __restrict__ dy, int64_t dys, const void* __restrict__ w,
    int wtype, const float* __restrict__ stats, TX* __restrict__ dx,
    TR* __restrict__ dr, int64_t rows, int H) {
  __shared__ double scratch[kLongThreads / 64];
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const TX* xr = x + row * xs;
    const TR* rr = RES ? r + row * rs : nullptr;
    const TY* gr = dy + row * dys;
    const RowNorm stat = get_stats(stats, rows, row);
    double all_g = 0.0, all_gn = 0.0;
    for (int i = threadIdx.x; i < H; i += kLongThreads) {
      float g = to_f(gr[i]);
      if (w) g *= load_as_float(w, wtype, i);
      all_g += g;
      all_gn += g * norm_of(load_z<TX, TR, RES>(xr, rr, i), stat);
    }
    const float sg = (float)(block_reduce(all_g, Add{}, scratch) / H);
    const float sgn = (float)(block_reduce(all_gn, Add{}, scratch) / H);
    for (int i = threadIdx.x; i < H; i += kLongThreads) {
      float g = to_f(gr[i]);
      if (w) g *= load_as_float(w, wtype, i);
      const float n = norm_of(load_z<TX, TR, RES>(xr, rr, i), stat);
      const float dz = stat.rstd * (g - sg - n * sgn);
      if (dx) dx[row * H + i] = static_cast<TX>(dz);
      if (RES && dr) dr[row * H + i] = static_cast<TR>(dz);
    }
  }
}

// Records of stripes of rows, for long rows.
template <typename TX, typename TR, typename TY, bool RES>
__global__ __launch_bounds__(256) void ln_dw_long_kernel(
    const TX* __restrict__ x, int64_t xs, const TR* __restrict__ r, int64_t rs,
    const TY* __restrict__ dy, int64_t dys, const float* __restrict__ stats,
    float* __restrict__ records, int64_t rows, int H) {
  __shared__ float sw[4][64], sb[4][64];
  const int lane = threadIdx.x & 63, sub = threadIdx.x >> 6;
  for (int64_t at = (int64_t)blockIdx.y * 64; at < H;
       at += (int64_t)gridDim.y * 64) {
    const int col = (int)at + lane;
    float aw = 0.f, ab = 0.f;
    if (col < H)
      for (int64_t row = (int64_t)blockIdx.x * 4 + sub; row < rows;
           row += (int64_t)gridDim.x * 4) {
        const float g = to_f(dy[row * dys + col]);
        const float z = load_z<TX, TR, RES>(x + row * xs,
                                            RES ? r + row * rs : nullptr, col);
        aw += g * norm_of(z, get_stats(stats, rows, row));
        ab += g;
      }
    sw[sub][lane] = aw;
    sb[sub][lane] = ab;
    __syncthreads();
    if (sub == 0 && col < H) {
      float* p = records + (int64_t)blockIdx.x * 2 * H;
      p[col] = (sw[0][lane] + sw[1][lane]) + (sw[2][lane] + sw[3][lane]);
      p[H + col] = (sb[0][lane] + sb[1][lane]) + (sb[2][lane] + sb[3][lane]);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------ launches
// Threads of a row's group, by its width; 0: too long for registers.
int group_of(int H, int chunk) {
  return H <= 16 * chunk           ? 16
         : H <= 32 * chunk         ? 32
         : H <= 64 * kPerThread    ? 64
         : H <= 256 * kPerThread   ? 256
         : H <= 1024 * kPerThread  ? 1024
                                   : 0;
}

int64_t at_most(int64_t n, int64_t most) { return n < most ? n : most; }

// f(group, chunks of a thread) for the smallest that hold a row
template <int E, typename F>
void with_group(int H, F f) {
  const int group = group_of(H, E);
  auto chunks = [&](auto g) {
    constexpr int G = decltype(g)::value;
    const int n = (H + G * E - 1) / (G * E);
    if constexpr (G < 64) f(g, Int<1>{});
    else if constexpr (E == 8) n <= 1 ? f(g, Int<1>{}) : f(g, Int<2>{});
    else if (n <= 1) f(g, Int<1>{});
    else if (n <= 2) f(g, Int<2>{});
    else if (n <= 3) f(g, Int<3>{});
    else f(g, Int<4>{});
  };
  if (group == 16) chunks(Int<16>{});
  else if (group == 32) chunks(Int<32>{});
  else if (group == 64) chunks(Int<64>{});
  else if (group == 256) chunks(Int<256>{});
  else if (group == 1024) chunks(Int<1024>{});
}

int64_t bwd_blocks(int64_t rows, int H, int chunk) {
  const int group = group_of(H, chunk);
  if (group == 0) return at_most((rows + 31) / 32, 256);
  const int per_block = group > 64 ? 1 : 512 / group;
  return at_most((rows + per_block - 1) / per_block, group == 256 ? 512 : 256);
}

template <typename TX, typename TR, typename TY, bool RES>
void fwd(hipStream_t st, const void* x, int64_t xs, const void* r, int64_t rs,
         const void* w, const void* b, int wtype, void* y, float* stats,
         int64_t rows, int H, float eps) {
  if (group_of(H, kChunk<TX>) == 0) {
    hipLaunchKernelGGL((ln_fwd_long_kernel<TX, TR, TY, RES>),
                       dim3(at_most(rows, kMaxBlocks)), dim3(kLongThreads), 0,
                       st, (const TX*)x, xs, (const TR*)r, rs, w, b, wtype,
                       (TY*)y, stats, rows, H, eps);
    return;
  }
  with_group<kChunk<TX>>(H, [&](auto g, auto nv) {
    constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
    constexpr int NT = G > 256 ? G : 256;
    const int64_t blocks = (rows + NT / G - 1) / (NT / G);
    hipLaunchKernelGGL((ln_fwd_kernel<TX, TR, TY, RES, G, NV>),
                       dim3(at_most(blocks, 2048)), dim3(NT), 0, st,
                       (const TX*)x, xs, (const TR*)r, rs, w, b, wtype, (TY*)y,
                       stats, rows, H, eps);
  });
}

template <typename TX, typename TR, typename TY, bool RES>
void bwd(hipStream_t st, const void* x, int64_t xs, const void* r, int64_t rs,
         const void* dy, int64_t dys, const void* w, int wtype,
         const float* stats, void* dx, void* dr, void* dw, void* db,
         float* records, int n, int64_t rows, int H) {
  if (group_of(H, kChunk<TX>) == 0) {
    if (dx || dr)
      hipLaunchKernelGGL((ln_bwd_long_kernel<TX, TR, TY, RES>),
                         dim3(at_most(rows, kMaxBlocks)), dim3(kLongThreads),
                         0, st, (const TX*)x, xs, (const TR*)r, rs,
                         (const TY*)dy, dys, w, wtype, stats, (TX*)dx,
                         (TR*)dr, rows, H);
    if (records)
      hipLaunchKernelGGL((ln_dw_long_kernel<TX, TR, TY, RES>),
                         dim3(n, at_most((H + 63) / 64, 65535)), dim3(256), 0,
                         st, (const TX*)x, xs, (const TR*)r, rs, (const TY*)dy,
                         dys, stats, records, rows, H);
  } else {
    with_group<kChunk<TX>>(H, [&](auto g, auto nv) {
      constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
      constexpr int NT = G > 512 ? G : G > 64 ? 256 : 512;
      hipLaunchKernelGGL((ln_bwd_kernel<TX, TR, TY, RES, G, NV>), dim3(n),
                         dim3(NT), 0, st, (const TX*)x, xs, (const TR*)r, rs,
                         (const TY*)dy, dys, w, wtype, stats, (TX*)dx,
                         (TR*)dr, records, rows, H);
    });
  }
  if (records)
    hipLaunchKernelGGL(ln_records_kernel,
                       dim3(at_most((2 * (int64_t)H + 63) / 64, kMaxBlocks)),
                       dim3(1024), 0, st, records, n, H, dw, db, wtype);
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

// Blocks of the backward, and records of dweight and dbias (2 H floats each).
int64_t dear_ln_blocks(int xtype, int64_t rows, int H) {
  return bwd_blocks(rows, H, xtype == kF32 ? 4 : 8);
}

int dear_ln_fwd(hipStream_t st, int xtype, int rtype, int wtype, const void* x,
                int64_t xs, const void* r, int64_t rs, const void* w,
                const void* b, void* y, float* stats, int64_t rows, int H,
                float eps) {
#define CALL(TX, TR, TY, RES)                                                 \
  fwd<TX, TR, TY, RES>(st, x, xs, r, rs, w, b, wtype, y, stats, rows, H, eps)
  LN_DISPATCH(CALL);
#undef CALL
  return (int)hipGetLastError();
}

// records: n times 2 H floats, or null where neither dw nor db is wanted.
int dear_ln_bwd(hipStream_t st, int xtype, int rtype, int wtype, const void* x,
                int64_t xs, const void* r, int64_t rs, const void* dy,
                int64_t dys, const void* w, const float* stats, void* dx,
                void* dr, void* dw, void* db, float* records, int n,
                int64_t rows, int H) {
#define CALL(TX, TR, TY, RES)                                                 \
  bwd<TX, TR, TY, RES>(st, x, xs, r, rs, dy, dys, w, wtype, stats, dx, dr,    \
                       dw, db, records, n, rows, H)
  LN_DISPATCH(CALL);
#undef CALL
  return (int)hipGetLastError();
}
