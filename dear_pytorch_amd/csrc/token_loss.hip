// Log probabilities of given tokens with entropy and top alternatives, and
// distillation from a teacher's top logits, forward and backward, for gfx950.
//
// With t_j = (z_j - m) / T, m the row's largest logit:
//   s = sum exp(t_j)            l_j = t_j - log s       p_j = exp(l_j)
//   entropy H = log s - sum(exp(t_j) t_j) / s
//   distillation from entries (id_k, q_k), q_t the share of all other tokens:
//   loss = T^2 (sum q_k (log q_k - l_{id_k}) + q_t (log q_t - log p_t)),
//   p_t = sum of p over the tokens that no entry names.
// backward:
//   dz_j = 1/T (sum_i c_i (1[id_i = j] - p_j) - dH p_j (l_j + H))
//   dz_j = T dloss (W p_j - sum_{id_k = j} q_k - [j not named] p_j q_t / p_t),
//   W = sum q_k + q_t. Where the student gives nothing to the tokens outside
//   (p_t = 0) the term of q_t is left out of loss and W.
//
// Elements are fp32; the sums of a thread are fp32 and those over threads
// fp64. s is 1 + r for a row that is sure of its token: the elements equal to
// m are counted and the others are added up by themselves, so that
// log s = log1p(r) keeps the digits of a probability near one.
#include <hip/hip_runtime.h>

#include "lm_common.h"

namespace {

using namespace dear_lm;

constexpr int kThreads = 256;
constexpr int kMaxBlocks = 1 << 20;   // a launch holds under 2^32 threads
constexpr int kMaxTop = 128;          // entries of a row, a thread for each
constexpr int kChunk = 1 << 16;       // tokens of one bitmap of named ones
constexpr double kLn2 = 0.69314718055994530942;

// A key that orders as the logits do: larger is better, NaN above all, both
// zeros equal.
__device__ __forceinline__ uint32_t order_key(float z) {
  if (z != z) return 0xffffffffu;
  const uint32_t u = __float_as_uint(z + 0.0f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// What a row leaves for its backward pass. inv_s == 0: nothing, its gradient
// is zero.
struct RowStats {
  float m, inv_s, a, b;
};

struct RowSums {
  float m;
  bool bad;         // the largest logit is not a number that can be a maximum
  double log_s, s, e2, out;
};

// Top of a row by bisection: the largest key that at least k elements reach,
// then, among the elements equal to it, the lowest indices.
template <typename T>
__device__ void row_top(const T* z, int V, int k, uint64_t* found, int* count,
                        int* scratch) {
  uint32_t key = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t want = key | (1u << bit);
    int n = 0;
    for (int i = threadIdx.x; i < V; i += kThreads)
      n += order_key(to_f(z[i])) >= want;
    if (block_reduce(n, Add{}, scratch) >= k) key = want;
  }
  int above = 0;
  for (int i = threadIdx.x; i < V; i += kThreads)
    above += order_key(to_f(z[i])) > key;
  const int need = k - block_reduce(above, Add{}, scratch);
  uint32_t low = 0, high = (uint32_t)V - 1;   // smallest index with `need`
  while (low < high) {
    const uint32_t mid = low + (high - low) / 2;
    int n = 0;
    for (int i = threadIdx.x; i <= (int)mid; i += kThreads)
      n += order_key(to_f(z[i])) == key;
    if (block_reduce(n, Add{}, scratch) >= need) high = mid;
    else low = mid + 1;
  }
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const uint32_t u = order_key(to_f(z[i]));
    if (u > key || (u == key && (uint32_t)i <= low))
      found[atomicAdd(count, 1)] = (uint64_t)u << 32 | ~(uint32_t)i;
  }
  __syncthreads();
}

// NAMED: `out` adds up the elements that no entry of `ids` names.
template <typename T, bool NAMED>
__device__ RowSums row_sums(const T* z, int V, float c, const int64_t* ids,
                            int k, uint32_t* bits, double* scratch) {
  RowSums r;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += kThreads)
    m = MaxNan{}(m, to_f(z[i]));
  r.m = m = block_reduce(m, MaxNan{}, reinterpret_cast<float*>(scratch));
  r.bad = !(fabsf(m) < INFINITY);
  float rest = 0.f, e2 = 0.f, out = 0.f;
  int top = 0;
  for (int base = 0; base < V; base += kChunk) {
    const int end = V - base < kChunk ? V - base : kChunk;
    if constexpr (NAMED) {
      __syncthreads();
      for (int i = threadIdx.x; i < kChunk / 32; i += kThreads) bits[i] = 0;
      __syncthreads();
      if (threadIdx.x < k) {
        const int64_t at = ids[threadIdx.x] - base;
        if (at >= 0 && at < end) atomicOr(&bits[at >> 5], 1u << (at & 31));
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < end; i += kThreads) {
      const float v = to_f(z[base + i]);
      const float y = (v - m) * c;
      const float e = __builtin_amdgcn_exp2f(y);
      if (v == m) ++top;
      else rest += e;
      e2 += e * fmaxf(y, -256.f);           // 0 for a logit of -inf
      if constexpr (NAMED)
        if (!(bits[i >> 5] >> (i & 31) & 1)) out += e;
    }
  }
  const double others = block_reduce((double)rest, Add{}, scratch) +
                        (block_reduce((double)top, Add{}, scratch) - 1.0);
  r.s = 1.0 + others;
  r.log_s = log1p(others);
  r.e2 = block_reduce((double)e2, Add{}, scratch);
  r.out = NAMED ? block_reduce((double)out, Add{}, scratch) : 0.0;
  return r;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_fwd_kernel(
    const T* __restrict__ logits, int64_t zs,
    const int64_t* __restrict__ tokens, int64_t ignore, int64_t rows, int V,
    int k, float c, double inv_t, float* __restrict__ logprob,
    float* __restrict__ entropy, float* __restrict__ top_lp,
    int64_t* __restrict__ top_ids, RowStats* __restrict__ stats) {
  __shared__ double scratch[kThreads / 64];
  __shared__ uint64_t found[kMaxTop];
  __shared__ int count;
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* z = logits + row * zs;
    const int64_t token = tokens ? tokens[row] : 0;
    if (tokens && token == ignore) {
      if (tid == 0) {
        logprob[row] = 0.f;
        entropy[row] = 0.f;
        if (stats) stats[row] = {0.f, 0.f, 0.f, 0.f};
      }
      for (int i = tid; i < k; i += kThreads) {
        top_lp[row * k + i] = -INFINITY;
        top_ids[row * k + i] = -1;
      }
      continue;
    }
    const RowSums r = row_sums<T, false>(z, V, c, nullptr, 0, nullptr,
                                         scratch);
    if (tid == 0) {
      const double h = r.bad ? NAN : r.log_s - kLn2 * r.e2 / r.s;
      entropy[row] = (float)h;
      if (tokens) {
        const bool ok = token >= 0 && token < V && !r.bad;
        logprob[row] =
            ok ? (float)(((double)to_f(z[token]) - (double)r.m) * inv_t -
                         r.log_s)
               : NAN;
      }
      if (stats)
        stats[row] = {r.m, r.bad ? NAN : (float)(1.0 / r.s),
                      (float)(h - r.log_s), 0.f};
    }
    if (k) {
      row_top(z, V, k, found, &count, reinterpret_cast<int*>(scratch));
      if (tid < k) {
        const uint64_t mine = found[tid];
        int rank = 0;
        for (int i = 0; i < k; ++i) rank += found[i] > mine;
        const uint32_t id = ~(uint32_t)mine;
        top_ids[row * k + rank] = id;
        top_lp[row * k + rank] =
            r.bad ? NAN
                  : (float)(((double)to_f(z[id]) - (double)r.m) * inv_t -
                            r.log_s);
      }
      __syncthreads();
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void logprobs_bwd_kernel(
    const T* __restrict__ logits, int64_t zs,
    const int64_t* __restrict__ tokens, const int64_t* __restrict__ top_ids,
    const RowStats* __restrict__ stats, const float* __restrict__ d_logprob,
    const float* __restrict__ d_entropy, const float* __restrict__ d_top,
    T* __restrict__ dz, int64_t rows, int V, int k, float c, float inv_t) {
  __shared__ float scratch[kThreads / 64];
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* z = logits + row * zs;
    T* out = dz + row * V;
    const RowStats s = stats[row];
    if (s.inv_s == 0.f) {
      for (int i = tid; i < V; i += kThreads) out[i] = static_cast<T>(0.f);
      continue;
    }
    const int64_t token = d_logprob ? tokens[row] : -1;
    const float up = d_logprob ? d_logprob[row] : 0.f;
    const float dh = d_entropy ? d_entropy[row] : 0.f;
    float a = d_top && tid < k ? d_top[row * k + tid] : 0.f;
    a = block_reduce(a, Add{}, scratch) + up;
    // a token outside of the vocabulary has no gradient that is a number
    if (d_logprob && (token < 0 || token >= V)) a = NAN;
    auto base = [&](float v) {
      const float d = v - s.m;
      const float p = __builtin_amdgcn_exp2f(d * c) * s.inv_s;
      float f = a;
      if (d_entropy) f += dh * (fmaxf(d * inv_t, -1e30f) + s.a);
      return -p * f;
    };
    for (int i = tid; i < V; i += kThreads)
      out[i] = static_cast<T>(base(to_f(z[i])) * inv_t);
    __syncthreads();
    // the named tokens once more, with what is theirs: thread k has the token
    if (tid <= k) {
      const int64_t id = tid == k ? token
                         : d_top  ? top_ids[row * k + tid]
                                  : -1;
      if (id >= 0 && id < V) {
        float g = id == token ? up : 0.f;
        if (d_top)
          for (int i = 0; i < k; ++i)
            if (top_ids[row * k + i] == id) g += d_top[row * k + i];
        out[id] = static_cast<T>((base(to_f(z[id])) + g) * inv_t);
      }
    }
    __syncthreads();
  }
}

template <typename T, bool TAIL>
__global__ __launch_bounds__(kThreads) void distill_fwd_kernel(
    const T* __restrict__ logits, int64_t zs,
    const int64_t* __restrict__ ids, const float* __restrict__ teacher,
    int64_t rows, int V, int k, float c, double t, float* __restrict__ loss,
    float* __restrict__ q_out, RowStats* __restrict__ stats) {
  __shared__ double scratch[kThreads / 64];
  __shared__ uint32_t bits[TAIL ? kChunk / 32 : 1];
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* z = logits + row * zs;
    const int64_t id = tid < k ? ids[row * k + tid] : -1;
    const bool present = id >= 0;
    const bool live = block_reduce((int)present, Add{},
                                   reinterpret_cast<int*>(scratch)) > 0;
    if (!live) {
      if (tid == 0) loss[row] = 0.f;
      if (stats) {
        if (tid == 0) stats[row] = {0.f, 0.f, 0.f, 0.f};
        if (tid < k) q_out[row * k + tid] = 0.f;
      }
      continue;
    }
    const float lp = present ? teacher[row * k + tid] : -INFINITY;
    double q, rest = 0.0;
    if constexpr (TAIL) {
      q = exp((double)lp);
      const double left = 1.0 - block_reduce(q, Add{}, scratch);
      rest = left <= 0.0 ? 0.0 : left;
    } else {
      const float top = block_reduce(lp, MaxNan{},
                                     reinterpret_cast<float*>(scratch));
      q = top == -INFINITY ? 0.0 : exp((double)lp - (double)top);
      const double sum = block_reduce(q, Add{}, scratch);
      q = sum == 0.0 ? 0.0 : q / sum;
    }
    const RowSums r = row_sums<T, TAIL>(z, V, c, ids + row * k, k, bits,
                                        scratch);
    double term = 0.0;
    if (id >= V) term = NAN;                 // no such token
    else if (present && q != 0.0)
      term = q * (log(q) -
                  (((double)to_f(z[id]) - (double)r.m) / t - r.log_s));
    double total = block_reduce(term, Add{}, scratch);
    double share = block_reduce(q, Add{}, scratch), shift = 0.0;
    if (TAIL && rest != 0.0 && r.out > 0.0) {
      share += rest;
      total += rest * (log(rest) - (log(r.out) - r.log_s));
      shift = rest * r.s / r.out;
    }
    if (r.bad) total = NAN;
    if (tid == 0) loss[row] = (float)(total * t * t);
    if (stats) {
      if (tid == 0)
        stats[row] = {r.m, total != total ? NAN : (float)(1.0 / r.s),
                      (float)share, (float)(share - shift)};
      if (tid < k) q_out[row * k + tid] = (float)q;
    }
    __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(
    const T* __restrict__ logits, int64_t zs,
    const int64_t* __restrict__ ids, const float* __restrict__ q,
    const RowStats* __restrict__ stats, const float* __restrict__ d_loss,
    T* __restrict__ dz, int64_t rows, int V, int k, float c, float t) {
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* z = logits + row * zs;
    T* out = dz + row * V;
    const RowStats s = stats[row];
    if (s.inv_s == 0.f) {
      for (int i = tid; i < V; i += kThreads) out[i] = static_cast<T>(0.f);
      continue;
    }
    const float g = d_loss[row] * t;
    for (int i = tid; i < V; i += kThreads) {
      const float p = __builtin_amdgcn_exp2f((to_f(z[i]) - s.m) * c) * s.inv_s;
      out[i] = static_cast<T>(p * s.b * g);
    }
    __syncthreads();
    if (tid < k) {
      const int64_t id = ids[row * k + tid];
      if (id >= 0 && id < V) {
        float taught = 0.f;
        for (int i = 0; i < k; ++i)
          if (ids[row * k + i] == id) taught += q[row * k + i];
        const float p =
            __builtin_amdgcn_exp2f((to_f(z[id]) - s.m) * c) * s.inv_s;
        out[id] = static_cast<T>((p * s.a - taught) * g);
      }
    }
    __syncthreads();
  }
}

int grid_for(int64_t rows) {
  return (int)(rows < kMaxBlocks ? rows : kMaxBlocks);
}

// log2(e) / T: exp(t) is exp2 of the distance times this
float exp2_factor(double t) { return (float)(1.4426950408889634074 / t); }

}  // namespace

#define BY_TYPE(type, CALL)                                                   \
  if ((type) == kF32) CALL(float);                                            \
  else if ((type) == kBF16) CALL(bf16);                                       \
  else CALL(f16)

int dear_logprobs_fwd(hipStream_t st, int type, const void* logits, int64_t zs,
                      const int64_t* tokens, int64_t ignore, int64_t rows,
                      int V, int k, double t, float* logprob, float* entropy,
                      float* top_lp, int64_t* top_ids, void* stats) {
#define CALL(T)                                                               \
  hipLaunchKernelGGL((logprobs_fwd_kernel<T>), dim3(grid_for(rows)), dim3(kThreads), 0, st,                 \
      (const T*)logits, zs, tokens, ignore, rows, V, k, exp2_factor(t),       \
      1.0 / t, logprob, entropy, top_lp, top_ids, (RowStats*)stats)
  BY_TYPE(type, CALL);
#undef CALL
  return (int)hipGetLastError();
}

int dear_logprobs_bwd(hipStream_t st, int type, const void* logits, int64_t zs,
                      const int64_t* tokens, const int64_t* top_ids,
                      const void* stats, const float* d_logprob,
                      const float* d_entropy, const float* d_top, void* dz,
                      int64_t rows, int V, int k, double t) {
#define CALL(T)                                                               \
  hipLaunchKernelGGL((logprobs_bwd_kernel<T>), dim3(grid_for(rows)), dim3(kThreads), 0, st,                 \
      (const T*)logits, zs, tokens, top_ids, (const RowStats*)stats,          \
      d_logprob, d_entropy, d_top, (T*)dz, rows, V, k, exp2_factor(t),        \
      (float)(1.0 / t))
  BY_TYPE(type, CALL);
#undef CALL
  return (int)hipGetLastError();
}

int dear_distill_fwd(hipStream_t st, int type, bool tail, const void* logits,
                     int64_t zs, const int64_t* ids, const float* teacher,
                     int64_t rows, int V, int k, double t, float* loss,
                     float* q, void* stats) {
#define CALL(T)                                                               \
  if (tail)                                                                   \
    hipLaunchKernelGGL((distill_fwd_kernel<T, true>), dim3(grid_for(rows)), dim3(kThreads), 0, st,          \
        (const T*)logits, zs, ids, teacher, rows, V, k, exp2_factor(t), t,    \
        loss, q, (RowStats*)stats);                                           \
  else                                                                        \
    hipLaunchKernelGGL((distill_fwd_kernel<T, false>), dim3(grid_for(rows)), dim3(kThreads), 0, st,         \
        (const T*)logits, zs, ids, teacher, rows, V, k, exp2_factor(t), t,    \
        loss, q, (RowStats*)stats)
  if (type == kF32) { CALL(float); }
  else if (type == kBF16) { CALL(bf16); }
  else { CALL(f16); }
#undef CALL
  return (int)hipGetLastError();
}

int dear_distill_bwd(hipStream_t st, int type, const void* logits, int64_t zs,
                     const int64_t* ids, const float* q, const void* stats,
                     const float* d_loss, void* dz, int64_t rows, int V, int k,
                     double t) {
#define CALL(T)                                                               \
  hipLaunchKernelGGL((distill_bwd_kernel<T>), dim3(grid_for(rows)), dim3(kThreads), 0, st,                  \
      (const T*)logits, zs, ids, q, (const RowStats*)stats, d_loss, (T*)dz,   \
      rows, V, k, exp2_factor(t), (float)t)
  BY_TYPE(type, CALL);
#undef CALL
  return (int)hipGetLastError();
}
