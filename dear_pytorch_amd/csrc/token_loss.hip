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
//   (all of their logits are -inf) the term of q_t is left out of loss and W.
// With a tail the outside has a largest logit m_o of its own, and its sum
// s_o = sum exp((z_j - m_o) / T) is relative to that: however far below m it
// lies, log p_t = (m_o - m) / T + log s_o - log s, and p_j q_t / p_t is
// exp((z_j - m_o) / T) q_t / s_o.
//
// Forward: a block takes a slice of one row into registers, 16 bytes a load,
// passes over it there (the maximum, then the sums, then the top) and leaves a
// record; a second kernel joins a row's records, a wave for each row, and does
// the fp64 arithmetic, whose registers would cost the first one half of its
// waves. Of few rows a block takes one whole and finishes it. Backward: one
// pass, elementwise, then the few named tokens again.
//
// Precision: exp(t) is exp2((z - m) c) with c = log2(e) / T: the difference is
// taken first, so that it is 0 for the largest element and errors stay small
// whatever the size of m. (One fma of z c - m c instead was no faster: 53.7 us
// for 52.8 at 4096 x 30528 bf16.) What c loses in fp32, at most 2^-24 of t, is
// the same for all elements; where the entropy's sum is at hand it is taken out
// of s in fp64. (Distillation has no such sum, and would take 67 us for 55 with
// one.) Sums of a wave are fp32, those over waves fp64. The elements equal to m
// are counted apart: s = 1 + r for a row that is sure of its token, and
// log(1 + r) keeps the digits of a probability near one.
#include <hip/hip_runtime.h>

#include "lm_common.h"

namespace {

using namespace dear_lm;

constexpr int kMaxTop = 128;          // entries of a row
constexpr int kMaxBlocks = 1 << 20;   // a launch holds under 2^32 threads
constexpr int kCandidates = 1024;     // of a slice's top, kept for ranking
constexpr int kPieces = 1024;         // of 16 bytes, with one of them or more
constexpr double kLn2 = 0.69314718055994530942;

// A key that orders as the logits do: larger is better, NaN above all, both
// zeros equal. No logit has the key 0.
__device__ __forceinline__ uint32_t order_key(float z) {
  if (z != z) return 0xffffffffu;
  const uint32_t u = __float_as_uint(z + 0.0f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Key and id of an alternative in one word: no two are equal, and of equal
// logits the lower id is the larger word.
__device__ __forceinline__ uint64_t candidate(float z, int id) {
  return (uint64_t)order_key(z) << 32 | ~(uint32_t)id;
}
__device__ __forceinline__ int id_of(uint64_t c) { return ~(uint32_t)c; }
__device__ __forceinline__ float logit_of(uint64_t c) {
  const uint32_t key = (uint32_t)(c >> 32);
  return __uint_as_float(key >> 31 ? key ^ 0x80000000u : ~key);
}

// What a row leaves for its backward pass: p_j = exp2((z_j - m) c) inv_s.
// inv_s == 0: the row was not looked at, its gradient is zero.
struct RowStats {
  float m, inv_s, a, unused;
};

// The same of a distillation's row. With m the largest logit of the tokens
// outside (without a tail: of all) the gradient is exp2((z_j - m) c) outside,
// in units of T dloss; the named tokens have theirs from the forward pass.
// live == 0: the row was not looked at.
struct DistillRow {
  float m, outside, live, unused;
};

// log2(e) / T, what fp32 leaves of it, and ln 2 times what that loses.
struct Factor {
  float c;
  double exact, lost;
};

// The sums of a slice or of a row, relative to its maximum m: n elements are
// equal to m, `rest` and e2 (of e log2 e) are over the others. With a tail all
// of this is over the elements outside.
struct Sums {
  double m, n, rest, e2;
};

__device__ __forceinline__ bool no_distribution(float m) {
  return !(fabsf(m) < INFINITY);
}

// log(1 + x), x >= 0, in few registers: with 1 + x = 2^k (1 + f), 1 + f from
// sqrt(1/2) to sqrt(2), and r = f / (2 + f), |r| < 0.1716,
//   log(1 + f) = 2 (r + r^3/3 + r^5/5 + ...)
// up to r^17/17, relatively to 2^-50; f is x itself where k = 0.
__device__ __forceinline__ double log_1p(double x) {
  double f = x;
  float k = 0.f;
  if (x > 0.41421356237309504880) {
    const double y = 1.0 + x;
    int e = __builtin_amdgcn_frexp_exp(y);
    f = __builtin_amdgcn_frexp_mant(y);
    if (f < 0.70710678118654752440) {
      f += f;
      --e;
    }
    f -= 1.0;
    k = (float)e;
  }
  const double r = f / (2.0 + f), r2 = r * r;
  double p = 1.0 / 17.0;
#pragma unroll
  for (int i = 15; i > 0; i -= 2) p = fma(p, r2, 1.0 / i);
  return fma((double)k, kLn2, 2.0 * r * p);
}

// ------------------------------------------------------- a slice in registers
template <typename T, int NT, int NV>
struct Slice {
  static constexpr int E = kVec<T>;
  u32x4 raw[NV];
  float vmax[NV];

  static __device__ __forceinline__ int first(int v) {
    return (v * NT + (int)threadIdx.x) * E;
  }
  __device__ __forceinline__ float at(int v, int j) const {
    return elem<T>(raw[v], j);
  }
  // tokens [0, len) of z; what lies behind is -inf, which adds nothing. One
  // 32-bit offset serves all loads, with the row's address in scalar registers.
  __device__ __forceinline__ void load(const T* z, int len) {
    const uint32_t mine = threadIdx.x * 16u;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const char* p = reinterpret_cast<const char*>(z + v * NT * E);
      if ((v + 1) * NT * E <= len) {          // the same for all threads
        raw[v] = load16(reinterpret_cast<const T*>(p + mine));
      } else {
        const int i = first(v);
        raw[v] = minus_inf<T>();
        if (i + E <= len) {
          raw[v] = load16(reinterpret_cast<const T*>(p + mine));
        } else {
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (i + j < len) put(raw[v], j, z[i + j]);
        }
      }
    }
  }
  // The compiler is not to keep the fp32 values of one pass for the next: they
  // would take twice the registers, and half of the waves.
  __device__ __forceinline__ void fresh(int v) {
    asm volatile("" : "+v"(raw[v]));
  }
  // the elements of `mask` become -inf
  __device__ __forceinline__ void drop(int v, uint32_t mask) {
    const u32x4 none = minus_inf<T>();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t bits;
      if constexpr (E == 4) {
        bits = mask >> w & 1 ? 0xffffffffu : 0u;
      } else {
        bits = (mask >> 2 * w & 1 ? 0xffffu : 0u) |
               (mask >> 2 * w & 2 ? 0xffff0000u : 0u);
      }
      raw[v][w] = (raw[v][w] & ~bits) | (none[w] & bits);
    }
  }
  // NaN if the thread holds one
  __device__ __forceinline__ float max() {
    float m = -INFINITY;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float a = at(v, 0);
#pragma unroll
      for (int j = 1; j < E; ++j) a = MaxNan{}(a, at(v, j));
      vmax[v] = a;
      m = MaxNan{}(m, a);
    }
    return m;
  }
};

// A slice's top by counting in memory, for rows whose order the quick way
// cannot use: NaN, or very many equal elements (a mask that leaves less than k
// tokens). bar: k elements at least reach it, or NaN where nothing is known.
// Where less than k are above it, these and the first ones equal to it are the
// top: the row is passed over once, and again to where the last one is found.
// Else the largest key that k elements reach comes first, in 32 more passes.
template <typename T, int NT>
__device__ __noinline__ void count_top(const T* z, int len, int base, int k,
                                       float bar, uint64_t* found, int* count,
                                       int* scratch) {
  constexpr int W = NT / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  auto reach = [&](uint32_t key) {       // elements with this key or a larger
    int n = 0;
    for (int i = threadIdx.x; i < len; i += NT)
      n += order_key(to_f(z[i])) >= key;
    return block_reduce(n, Add{}, scratch);
  };
  uint32_t key = order_key(bar);
  int above = key == 0xffffffffu ? k : reach(key + 1);
  if (above >= k) {
    key = 0;
    for (int bit = 31; bit >= 0; --bit)
      if (reach(key | (1u << bit)) >= k) key |= 1u << bit;
    above = key == 0xffffffffu ? 0 : reach(key + 1);
  }
  if (threadIdx.x == 0) *count = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < len && above > 0; i += NT) {
    const float v = to_f(z[i]);
    if (order_key(v) > key) found[atomicAdd(count, 1)] = candidate(v, base + i);
  }
  // found[above, k): those equal to it, in the order of their ids
  for (int first = 0, at = above; first < len && at < k; first += NT) {
    const int i = first + (int)threadIdx.x;
    const float v = i < len ? to_f(z[i]) : 0.f;
    const bool equal = i < len && order_key(v) == key;
    const uint64_t them = __ballot(equal);
    __syncthreads();                     // `scratch` has been read
    if (lane == 0) scratch[wave] = __popcll(them);
    __syncthreads();
    int place = at;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < wave) place += scratch[w];
      at += scratch[w];
    }
    place += lanes_before(them);
    if (equal && place < k) found[place] = candidate(v, base + i);
  }
  __syncthreads();
}

// Lanes' values in falling order (bitonic, 21 exchanges). Which lanes keep the
// larger value is known when compiled, as a mask in scalar registers.
template <int Size, int O>
__device__ __forceinline__ float exchange(float v) {
  constexpr uint64_t keep = [] {
    uint64_t m = 0;
    for (int lane = 0; lane < 64; ++lane)
      if (((lane & O) == 0) == ((lane & Size) == 0)) m |= 1ull << lane;
    return m;
  }();
  const Pair p = lanes<O>(v);
  v = __builtin_amdgcn_inverse_ballot_w64(keep) ? fmaxf(p.x, p.y)
                                                : fminf(p.x, p.y);
  if constexpr (O > 1) return exchange<Size, O / 2>(v);
  else return v;
}
__device__ __forceinline__ float wave_sort(float v) {
  v = exchange<2, 1>(v);
  v = exchange<4, 2>(v);
  v = exchange<8, 4>(v);
  v = exchange<16, 8>(v);
  v = exchange<32, 16>(v);
  return exchange<64, 32>(v);
}

// A wave's ceil(k / waves)-th best of its threads' maxima, written before the
// waves meet for the row's maximum.
template <int NT>
__device__ __forceinline__ void put_floor(float mine, int k,
                                          float* wave_floor) {
  const int each = (k + NT / 64 - 1) / (NT / 64);
  const float bar = each == 1 ? wave_reduce(mine, Max{})
                              : __shfl(wave_sort(mine), each - 1);
  if ((threadIdx.x & 63) == 0) wave_floor[threadIdx.x >> 6] = bar;
}

// The k best of a slice into found[0..n), in no order; every thread gets n.
// k is at most NT. Each of the NT / 64 waves has ceil(k / waves) elements that
// reach the smallest of the waves' floors: k elements at least reach it, and
// about twice k do if the row is in no order. Two steps collect them: the
// 16-byte pieces that have one, known by their maxima, and then a thread for
// each element of those, from memory again. count[0] and [1] are zero.
template <typename T, int NT, int NV>
__device__ int slice_top(const Slice<T, NT, NV>& s, const T* z, int len,
                         int base, int k, bool has_nan, uint64_t* found,
                         int* count, const float* wave_floor, int* scratch) {
  constexpr int W = NT / 64, E = kVec<T>;
  const int lane = threadIdx.x & 63;
  uint16_t* pieces = reinterpret_cast<uint16_t*>(found + kCandidates);
  float bar = NAN;
  if (!has_nan) {
    bar = wave_floor[0];
#pragma unroll
    for (int i = 1; i < W; ++i) bar = fminf(bar, wave_floor[i]);
    uint64_t has[NV];
    int all = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      has[v] = __ballot(s.vmax[v] >= bar);
      all += __popcll(has[v]);
    }
    int at = 0;
    if (lane == 0 && all) at = atomicAdd(count, all);
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int place = at + lanes_before(has[v]);
      if (s.vmax[v] >= bar && place < kPieces)
        pieces[place] = (uint16_t)(v * NT + threadIdx.x);
      at += __popcll(has[v]);
    }
    __syncthreads();
    const int n_pieces = *count;
    if (n_pieces <= kPieces) {
      // whole waves go round together
      for (int first = 0; first < n_pieces * E; first += NT) {
        const int e = first + (int)threadIdx.x;
        const int i = e < n_pieces * E ? pieces[e / E] * E + e % E : len;
        const float x = i < len ? to_f(z[i]) : -INFINITY;
        const bool kept = i < len && x >= bar;
        const uint64_t them = __ballot(kept);
        if (them == 0) continue;
        int place = 0;
        if (lane == 0) place = atomicAdd(count + 1, __popcll(them));
        place = __builtin_amdgcn_readfirstlane(place) + lanes_before(them);
        if (kept && place < kCandidates) found[place] = candidate(x, base + i);
      }
      __syncthreads();
      if (count[1] <= kCandidates) return count[1];
    }
    __syncthreads();                     // before `count` is used again
  }
  count_top<T, NT>(z, len, base, k, bar, found, count, scratch);
  return k;
}

// Calls put(rank, candidate) for the k best of found[0..n): the rank is how
// many are better, counted by 2^share lanes together.
template <int NT, typename Put>
__device__ __forceinline__ void ranked(const uint64_t* found, int n, int k,
                                       Put put) {
  int share = 0;
  while (share < 3 && (n << (share + 1)) <= NT) ++share;
  const int sub = threadIdx.x & ((1 << share) - 1);
  // whole waves go round together, for their lanes add up each other's counts
  for (int first = 0; first < n; first += NT >> share) {
    const int i = first + ((int)threadIdx.x >> share);
    const uint64_t mine = i < n ? found[i] : 0;
    int count = 0, j = sub;
    for (; j + (3 << share) < n; j += 4 << share) {
#pragma unroll
      for (int u = 0; u < 4; ++u) count += found[j + (u << share)] > mine;
    }
    for (; j < n; j += 1 << share) count += found[j] > mine;
    float better = (float)count;
    if (share > 0) better = sum_of(lanes<1>(better));
    if (share > 1) better = sum_of(lanes<2>(better));
    if (share > 2) better = sum_of(lanes<4>(better));
    if (i < n && sub == 0 && better < (float)k) put((int)better, mine);
  }
}

// ------------------------------------------------------ sums of one slice
// Adds up one slice against the maximum m (not NaN, finite). ENT: e2 too.
// Results in every thread of the first wave.
template <typename T, int NT, int NV, bool ENT>
__device__ __forceinline__ Sums slice_sums(Slice<T, NT, NV>& s, float m,
                                           Factor f, float (*scratch)[3]) {
  constexpr int W = NT / 64, E = kVec<T>;
  float rest = 0.f, e2 = 0.f, n = 0.f;
  auto add = [&](int v) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const float y = (s.at(v, j) - m) * f.c;
      const float e = __builtin_amdgcn_exp2f(y);
      rest += e;
      if constexpr (ENT) e2 = fmaf(e, fmaxf(y, -256.f), e2);  // 0 for -inf
    }
  };
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    s.fresh(v);
    if (s.vmax[v] != m) {
      add(v);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float x = s.at(v, j), y = (x - m) * f.c;
        const float e = __builtin_amdgcn_exp2f(y);
        if (x == m) {
          n += 1.f;
        } else {
          rest += e;
          if constexpr (ENT) e2 = fmaf(e, fmaxf(y, -256.f), e2);
        }
      }
    }
  }
  rest = wave_reduce(rest, Add{});
  n = wave_reduce(n, Add{});
  if constexpr (ENT) e2 = wave_reduce(e2, Add{});
  if ((threadIdx.x & 63) == 0) {
    float* p = scratch[threadIdx.x >> 6];
    p[0] = rest; p[1] = n; p[2] = e2;
  }
  __syncthreads();
  Sums r = {};
  if (threadIdx.x < 64) {
    for (int i = 0; i < W; ++i) {
      const float* p = scratch[i];
      r.rest += p[0];
      r.n += p[1];
      if constexpr (ENT) r.e2 += p[2];
    }
    // exp2(y c_exact / c) of every element, to first order (2^-24 squared)
    if constexpr (ENT) r.rest += f.lost * r.e2;
  }
  r.m = m;
  return r;
}

// Joins the records of a row's slices; to be called by a whole wave. `mine` is
// the lane's first record, loaded by record_of before there is use for it. A
// slice of -inf alone adds nothing.
__device__ __forceinline__ Sums record_of(const Sums* part, int64_t ns) {
  const int lane = threadIdx.x & 63;
  return part[lane < ns ? lane : 0];
}
__device__ __forceinline__ Sums join_sums(const Sums& mine, const Sums* part,
                                          int64_t ns, Factor f) {
  if (ns == 1) return mine;
  const int lane = threadIdx.x & 63;
  float m = (float)mine.m;
  for (int64_t i = lane + 64; i < ns; i += 64)
    m = MaxNan{}(m, (float)part[i].m);
  m = wave_reduce(m, MaxNan{});
  Sums r = {};
  r.m = m;
  auto add = [&](const Sums& p) {
    if (p.m == (double)m) {
      r.n += p.n;
      r.rest += p.rest;
      r.e2 += p.e2;
    } else if (p.m > -INFINITY) {
      const double y = (p.m - (double)m) * f.exact, g = exp2(y);
      const double all = p.n + p.rest;
      r.rest += g * all;
      r.e2 += g == 0.0 ? 0.0 : g * (p.e2 + y * all);
    }
  };
  if (lane < ns) add(mine);
  for (int64_t i = lane + 64; i < ns; i += 64) add(part[i]);
  for (int o = 1; o < 64 && o < ns; o <<= 1) {    // the lanes with a record
    r.n += __shfl_xor(r.n, o);
    r.rest += __shfl_xor(r.rest, o);
    r.e2 += __shfl_xor(r.e2, o);
  }
  r.n = __shfl(r.n, 0);
  r.rest = __shfl(r.rest, 0);
  r.e2 = __shfl(r.e2, 0);
  return r;
}

// ------------------------------------------------- log probabilities, forward
struct LogprobArgs {
  const int64_t* tokens;
  int64_t zs, ignore, rows;
  int V, k, per_slice;       // tokens of a slice
  int64_t slices;
  Factor f;
  double inv_t;
  float *logprob, *entropy, *top_lp;
  int64_t* top_ids;
  RowStats* stats;
  Sums* part;                // [rows][slices]
  uint64_t* lists;           // [rows][slices][k], best first, 0: no such one
};

// A row that is not looked at, by `threads` threads.
__device__ __forceinline__ void leave_out(const LogprobArgs& a, int64_t row,
                                          int thread, int threads) {
  if (thread == 0) {
    a.logprob[row] = 0.f;
    a.entropy[row] = 0.f;
    if (a.stats) a.stats[row] = {0.f, 0.f, 0.f, 0.f};
  }
  for (int i = thread; i < a.k; i += threads) {
    a.top_lp[row * a.k + i] = -INFINITY;
    a.top_ids[row * a.k + i] = -1;
  }
}

// The token's logit; NaN of one outside of the vocabulary.
template <typename T>
__device__ __forceinline__ float logit_at(const LogprobArgs& a, int64_t token,
                                          const T* z) {
  return a.tokens && token >= 0 && token < a.V ? to_f(z[token]) : NAN;
}

// The numbers of a row from its sums and its token's logit, written by the
// `first` thread; log s to all.
__device__ __forceinline__ double finish_row(const LogprobArgs& a, int64_t row,
                                             float at, const Sums& s,
                                             bool first) {
  const float m = (float)s.m;
  const bool bad = no_distribution(m);
  const double others = s.rest + (s.n - 1.0);
  const double log_s = bad ? NAN : log_1p(others);
  if (!first) return log_s;
  const double inv = 1.0 / (1.0 + others), h = log_s - kLn2 * s.e2 * inv;
  a.entropy[row] = (float)h;
  if (a.tokens) a.logprob[row] = (float)(((double)at - s.m) * a.inv_t - log_s);
  if (a.stats)
    a.stats[row] = {m, bad ? NAN : (float)inv, (float)(h - log_s), 0.f};
  return log_s;
}

__device__ __forceinline__ void put_top(const LogprobArgs& a, int64_t place,
                                        uint64_t c, double m, double log_s) {
  a.top_ids[place] = id_of(c);
  a.top_lp[place] = (float)(((double)logit_of(c) - m) * a.inv_t - log_s);
}

// WHOLE: a slice is a whole row, and is finished here.
// 4096 x 30528 bf16: 49 us without a top (5.1 TB/s), bound by memory and by the
// vector unit alike, which is busy for 81 % of that: a conversion, a
// subtraction, a product, exp2, two sums and the maximum for each element. 74 us
// with a top of 32 (84 % busy), and 112 with one of 128, where the ranking reads
// LDS for each pair. The row is never read again from memory but for some
// hundred pieces that may hold one of the top.
template <typename T, int NT, int NV, bool TOP, bool WHOLE>
__global__ __launch_bounds__(NT, WHOLE ? 4 : 6) void logprobs_slice_kernel(
    const T* __restrict__ logits, const LogprobArgs a) {
  __shared__ float wave_max[NT / 64], wave_floor[NT / 64];
  __shared__ float sums[NT / 64][3];
  __shared__ int scratch[NT / 64];
  __shared__ uint64_t found[TOP ? kCandidates + kPieces / 4 : 1];
  __shared__ int count[2];
  __shared__ double row_log_s;
  const int64_t work = a.rows * a.slices;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int64_t row = WHOLE || a.slices == 1 ? w : w / a.slices;
    const int base = (int)(w - row * a.slices) * a.per_slice;
    const int64_t token = a.tokens ? a.tokens[row] : 0;
    if (a.tokens && token == a.ignore) {
      if constexpr (WHOLE) leave_out(a, row, threadIdx.x, NT);
      continue;
    }
    const T* z = logits + row * a.zs + base;
    const int len = min(a.per_slice, a.V - base);
    Slice<T, NT, NV> s;
    s.load(z, len);
    float at = NAN;
    if constexpr (WHOLE) at = logit_at(a, token, z);
    const float mine = s.max();
    if constexpr (TOP) {
      put_floor<NT>(mine, min(a.k, len), wave_floor);
      if (threadIdx.x < 2) count[threadIdx.x] = 0;
    }
    const float m = block_max<NT>(mine, wave_max);
    Sums r = {};
    if (!no_distribution(m))
      r = slice_sums<T, NT, NV, true>(s, m, a.f, sums);
    r.m = m;
    if constexpr (!WHOLE) {
      if (threadIdx.x == 0) a.part[w] = r;
    } else if (threadIdx.x < 64) {       // while the others begin with the top
      const double log_s = finish_row(a, row, at, r, threadIdx.x == 0);
      if (threadIdx.x == 0) row_log_s = log_s;
    }
    if constexpr (TOP) {
      const int k = min(a.k, len);
      const int n = slice_top(s, z, len, base, k, m != m, found, count,
                              wave_floor, scratch);
      if constexpr (WHOLE) {             // k is a.k
        const double log_s = row_log_s;
        ranked<NT>(found, n, k, [&](int rank, uint64_t c) {
          put_top(a, row * a.k + rank, c, m, log_s);
        });
      } else {
        uint64_t* list = a.lists + w * a.k;
        ranked<NT>(found, n, k, [&](int rank, uint64_t c) { list[rank] = c; });
        for (int i = k + threadIdx.x; i < a.k; i += NT) list[i] = 0;
      }
    }
    __syncthreads();                     // before the arrays are used again
  }
}

// Four rows to a block, a wave each. Bound by the latency of its loads, one
// after the other: 5 us of 4096 rows of one or two slices, 6 of 167 rows of
// four slices with a top of 20.
template <typename T>
__global__ __launch_bounds__(256) void logprobs_finish_kernel(
    const T* __restrict__ logits, const LogprobArgs a) {
  constexpr int kHeld = 1024, kAhead = 8;
  __shared__ uint64_t held[4][kHeld];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t row = (int64_t)blockIdx.x * 4 + wave; row < a.rows;
       row += (int64_t)gridDim.x * 4) {
    const Sums* part = a.part + row * a.slices;
    const Sums mine = record_of(part, a.slices);
    const int64_t token = a.tokens ? a.tokens[row] : 0;
    if (a.tokens && token == a.ignore) {
      leave_out(a, row, lane, 64);
      continue;
    }
    const float at = logit_at(a, token, logits + row * a.zs);
    const Sums s = join_sums(mine, part, a.slices, a.f);
    const double log_s = finish_row(a, row, at, s, lane == 0);
    if (a.k == 0) continue;              // there are no lists
    const uint64_t* lists = a.lists + row * a.slices * a.k;
    const int64_t entries = a.slices * a.k;
    auto put = [&](int rank, uint64_t c) {
      put_top(a, row * a.k + rank, c, s.m, log_s);
    };
    if (a.slices == 1) {
      for (int i = lane; i < a.k; i += 64) put(i, lists[i]);
      continue;
    }
    // No better than the last of some list: not in the top. And k of them at
    // least are as good as the r-th best of the lists' d-th, r d >= k. The
    // others, most often little more than k, count how many are better.
    const int heads = (int)min(a.slices, (int64_t)64);
    const int d = (a.k + heads - 1) / heads, r = (a.k + d - 1) / d;
    uint64_t last = 0, head = 0;         // a lane's lists, the best of them
    for (int64_t l = lane; l < a.slices; l += 64) {
      last = max(last, lists[l * a.k + a.k - 1]);
      head = max(head, lists[l * a.k + d - 1]);
    }
    int ahead = 0;
    for (int j = 0; j < heads; ++j) ahead += __shfl(head, j) > head;
    const uint64_t bar =
        wave_reduce(max(last, ahead >= r - 1 ? head : 0), Larger{});
    int64_t n = 0;
    for (int64_t first = 0; first < entries; first += 64 * kAhead) {
      uint64_t c[kAhead];                // loads that do not wait for another
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t i = first + 64 * j + lane;
        c[j] = i < entries ? lists[i] : 0;
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool kept = c[j] != 0 && c[j] >= bar;
        const uint64_t all = __ballot(kept);
        const int64_t place = n + lanes_before(all);
        if (kept && place < kHeld) held[wave][place] = c[j];
        n += __popcll(all);
      }
    }
    wave_fence();
    if (n <= kHeld) {
      for (int i = 0; i < n; i += 64) {
        const uint64_t mine = i + lane < n ? held[wave][i + lane] : 0;
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < (int)n; ++j) rank += held[wave][j] > mine;
        if (mine != 0 && rank < a.k) put(rank, mine);
      }
    } else {
      // the place of a candidate: its place in its own list, and how many of
      // each other list are better
      for (int64_t i = lane; i < entries; i += 64) {
        const uint64_t mine = lists[i];
        if (mine == 0) continue;
        const int64_t own = i / a.k;
        int64_t rank = i - own * a.k;
        for (int64_t l = 0; l < a.slices && rank < a.k; ++l) {
          if (l == own) continue;
          const uint64_t* list = lists + l * a.k;
          int lo = 0, hi = a.k;          // entries that are better
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (list[mid] > mine) lo = mid + 1;
            else hi = mid;
          }
          rank += lo;
        }
        if (rank < a.k) put((int)rank, mine);
      }
    }
    wave_fence();                        // `held` is written again
  }
}

// ------------------------------------------------------ distillation, forward
struct DistillArgs {
  const int64_t* ids;
  const float* teacher;
  int64_t zs, rows;
  int V, k, per_slice;
  int64_t slices;
  Factor f;
  double t, inv_t;
  float *loss, *named_out;   // and the named tokens' gradients, a.k a row
  DistillRow* stats;
  Sums* part;
};

// A row's entries, N to a lane of the wave that finishes the row.
template <int N>
struct Entries {
  int64_t id[N];
  float lp[N], z[N];       // the teacher's, and the student's logit
  template <typename T>
  __device__ __forceinline__ void load(const DistillArgs& a, int64_t row,
                                       const T* logits) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = (threadIdx.x & 63) + 64 * e;
      id[e] = i < a.k ? a.ids[row * a.k + i] : -1;
      lp[e] = id[e] >= 0 ? a.teacher[row * a.k + i] : -INFINITY;
      // an id outside of the vocabulary: NaN
      z[e] = id[e] < 0 ? 0.f : id[e] < a.V ? to_f(logits[id[e]]) : NAN;
    }
  }
};

// Whether a lane's id is another entry's as well, and which of the entries of
// one id stands for it. All write their number into the slot of their id; whose
// number is read there is done, and so are the entries with the same id. The
// others, of another id in the same slot, go on.
// 614 rows of 64 entries: 2.5 us less than comparing each id with all others.
constexpr int kSlots = 2048;
template <int N>
__device__ __forceinline__ bool named_twice(const int (&id)[N], bool (&one)[N],
                                            uint8_t* slots) {
  const int lane = threadIdx.x & 63;
  bool twice = false, open[N];
  uint32_t slot[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    slot[e] = ((uint32_t)id[e] * 0x9e3779b1u) >> 21;     // under kSlots
    open[e] = true;
    one[e] = false;
  }
  bool go_on = true;
  while (__any(go_on)) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (open[e]) slots[slot[e]] = (uint8_t)(lane + 64 * e);
    wave_fence();
    go_on = false;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int owner = slots[slot[e]];
      int theirs = __shfl(id[0], owner & 63);
      if constexpr (N > 1) {
        const int other = __shfl(id[1], owner & 63);
        if (owner >= 64) theirs = other;
      }
      if (open[e] && theirs == id[e]) {
        one[e] = owner == lane + 64 * e;
        twice |= !one[e];
        open[e] = false;
      }
      go_on |= open[e];
    }
    wave_fence();                        // before the slots are written again
  }
  return twice;
}

// One wave: the loss of a row. log q is the teacher's own number, less what
// it is normalised by: no logarithm of an entry is taken. Without a tail, with
// u_k = exp(lp_k - top) and U = sum u, q_k = u_k / U and
//   sum q_k (log q_k - l_k) = sum u_k ((lp_k - top) - l_k) / U - log U.
template <bool TAIL, int N>
__device__ __forceinline__ void finish_distill(const DistillArgs& a,
                                               int64_t row, const Sums& s,
                                               const Entries<N>& t,
                                               uint8_t* slots) {
  const int lane = threadIdx.x & 63;
  float top = 0.f;
  if constexpr (!TAIL) {
    top = t.lp[0];
    if constexpr (N > 1) top = MaxNan{}(top, t.lp[1]);
    top = wave_reduce(top, MaxNan{});
  }
  // The absent entries are no id's; of ids past 32 bits the loss is NaN anyway.
  int id[N];
  bool one[N], twice = false;
#pragma unroll
  for (int e = 0; e < N; ++e)
    id[e] = t.id[e] < 0 ? -1 - lane - 64 * e : (int)t.id[e];
  if (TAIL || a.stats) twice = __any(named_twice<N>(id, one, slots));
  // the largest logit of the tokens outside, and of the row
  const float m_out = (float)s.m;
  float m = m_out;
  if constexpr (TAIL) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      m = MaxNan{}(m, t.id[e] < 0 ? -INFINITY : t.z[e]);
    m = wave_reduce(m, MaxNan{});
  }
  const bool bad = no_distribution(m);
  double x[N] = {}, in = 0.0, n_in = 0.0;    // exp of the entries, each id once
  if (!bad && (TAIL || a.stats)) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (t.id[e] >= 0) x[e] = exp(((double)t.z[e] - (double)m) * a.inv_t);
  }
  double n = s.n, less = s.rest, gap = 0.0, shrink = 1.0;
  const double outside = s.n + s.rest;
  if constexpr (TAIL) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if (t.id[e] < 0 || !one[e]) continue;
      if (t.z[e] == m) n_in += 1.0;
      else in += x[e];
    }
    wave_sum(in, n_in);
    if (m_out < m) {
      gap = ((double)m_out - (double)m) * a.inv_t;
      shrink = exp(gap);
      n = 0.0;
      less = shrink * outside;
    }
  }
  const double others = (less + in) + ((n + n_in) - 1.0);
  const double sum = 1.0 + others, log_s = log_1p(others);
  double q[N], all_q = 0.0, total = 0.0, rest = 0.0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const double lq = (double)t.lp[e] - (double)top;
    q[e] = top == -INFINITY ? 0.0 : exp(lq);
    all_q += q[e];
    if (t.z[e] != t.z[e])                    // no such token, or a NaN
      total = NAN;
    else if (q[e] != 0.0)
      total += q[e] * (lq - (((double)t.z[e] - (double)m) * a.inv_t - log_s));
  }
  wave_sum(all_q, total);
  if constexpr (TAIL) {
    rest = 1.0 - all_q <= 0.0 ? 0.0 : 1.0 - all_q;    // NaN stays
  } else if (all_q != 0.0) {             // at least 1, or NaN
    const double by = 1.0 / all_q;
    total = total * by - log(all_q);
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] *= by;
    all_q = 1.0;
  }
  double share = all_q, tail = 0.0;
  if (TAIL && rest != 0.0 && m_out != -INFINITY) {
    share += rest;
    tail = rest / outside;               // q_t / s_o
    total += rest * (log(tail * sum) - gap);
  }
  if (bad) total = NAN;
  if (lane == 0) a.loss[row] = (float)(total * a.t * a.t);
  if (!a.stats) return;
  const double inv = total != total ? NAN : 1.0 / sum;
  if (lane == 0)
    a.stats[row] = {m_out == -INFINITY ? 0.f : m_out,
                    (float)(share * (shrink * inv) - tail), 1.f, 0.f};
  // an id that is named more than once: each of its entries gets the sum
  if (twice) {
    double sum_q[N] = {};
    for (int i = 0; i < 64; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int theirs = __shfl(id[e], i);
        const double share_of_one = __shfl(q[e], i);
#pragma unroll
        for (int d = 0; d < N; ++d)
          if (theirs == id[d]) sum_q[d] += share_of_one;
      }
#pragma unroll
    for (int e = 0; e < N; ++e) q[e] = sum_q[e];
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (lane + 64 * e < a.k)
      a.named_out[row * a.k + lane + 64 * e] =
          (float)(share * (x[e] * inv) - q[e]);
}

// 4096 x 30528 bf16, 32 entries: 46 us without a tail (5.4 TB/s), 51 with one
// (4.9 TB/s), and 9 for the kernel that joins the slices. With a tail the
// elements that are named have to be left out of maximum and sum exactly: taking
// them from the sum afterwards, or summing the others relative to them, would
// leave nothing of a small tail. They are known by a bit for each element of a
// thread, which cost less than comparing the ids (67 us).
template <typename T, int NT, int NV, bool TAIL>
__global__ __launch_bounds__(NT, 6) void distill_slice_kernel(
    const T* __restrict__ logits, const DistillArgs a) {
  constexpr int E = kVec<T>;
  constexpr int kOwn = (kMaxTop + NT - 1) / NT;     // entries of a thread
  __shared__ float wave_max[NT / 64];
  __shared__ float sums[NT / 64][3];
  __shared__ uint64_t masks[TAIL ? NT : 1];         // a bit for each element
  const int64_t work = a.rows * a.slices;
  const int tid = threadIdx.x;
  for (int64_t w = blockIdx.x; w < work; w += gridDim.x) {
    const int64_t row = a.slices == 1 ? w : w / a.slices;
    const int base = (int)(w - row * a.slices) * a.per_slice;
    const int64_t* ids = a.ids + row * a.k;
    int64_t id[kOwn];
    bool live = false;
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      const int i = tid + e * NT;
      id[e] = i < a.k ? ids[i] : -1;
      live |= id[e] >= 0;
    }
    if constexpr (TAIL) masks[tid] = 0;
    if (!__syncthreads_or(live)) continue;
    const T* z = logits + row * a.zs + base;
    const int len = min(a.per_slice, a.V - base);
    Slice<T, NT, NV> s;
    s.load(z, len);
    if constexpr (TAIL) {
      // the named ones become -inf, which adds nothing
#pragma unroll
      for (int e = 0; e < kOwn; ++e) {
        const int64_t at = id[e] - base;
        if (at < 0 || at >= len) continue;
        const int piece = (int)at / E, bit = piece / NT * E + (int)at % E;
        atomicOr((unsigned long long*)&masks[piece % NT], 1ull << bit);
      }
      __syncthreads();
      const uint64_t named = masks[tid];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const uint32_t mask = (uint32_t)(named >> v * E) & ((1u << E) - 1u);
        if (mask) s.drop(v, mask);
      }
    }
    const float m = block_max<NT>(s.max(), wave_max);     // synchronises
    Sums r = {};
    if (!no_distribution(m))
      r = slice_sums<T, NT, NV, false>(s, m, a.f, sums);
    r.m = m;
    if (tid == 0) a.part[w] = r;
    __syncthreads();
  }
}

// Four rows to a block, a wave each; N * 64 entries at most. Bound by latency,
// of its loads and of fp64: 4 us of 614 rows, 9 of 4096.
template <typename T, bool TAIL, int N>
__global__ __launch_bounds__(256) void distill_finish_kernel(
    const T* __restrict__ logits, const DistillArgs a) {
  __shared__ uint8_t owners[4][kSlots];
  uint8_t* slots = owners[threadIdx.x >> 6];
  const int lane = threadIdx.x & 63;
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
       row < a.rows; row += (int64_t)gridDim.x * 4) {
    const Sums* part = a.part + row * a.slices;
    const Sums mine = record_of(part, a.slices);
    Entries<N> t;
    t.load(a, row, logits + row * a.zs);
    bool live = t.id[0] >= 0;
    if constexpr (N > 1) live |= t.id[1] >= 0;
    if (!__any(live)) {
      if (lane == 0) a.loss[row] = 0.f;
      if (a.stats) {
        if (lane == 0) a.stats[row] = {0.f, 0.f, 0.f, 0.f};
        for (int i = lane; i < a.k; i += 64) a.named_out[row * a.k + i] = 0.f;
      }
      continue;
    }
    finish_distill<TAIL, N>(
        a, row, join_sums(mine, part, a.slices, a.f), t, slots);
  }
}

// ----------------------------------------------------------------- backward
// A block of 256 takes 512 vectors of one row. The last row comes first: what
// the forward pass has read last is still in the last-level cache (4096 x 30528
// bf16, 250 MB, in a pass of forward and backward: 88 us in the rows' order, 80
// in this one).
constexpr int kBwdThreads = 256;
constexpr int kBwdVectors = 2;
template <typename T>
constexpr int kBwdTokens = kBwdThreads * kBwdVectors * kVec<T>;

// Where a gradient is larger than half of the last-level cache it is written
// past the caches: 4096 x 30528 fp32, 15 % of the rows labelled, takes 86 us
// instead of 111; of 75 MB, 24 either way, and there what reads it next may
// find it in the cache.
constexpr int64_t kStreamBytes = 128 << 20;

template <bool STREAM, typename T>
__device__ __forceinline__ void store_vec(T* p, u32x4 v) {
  if constexpr (STREAM) stream16(p, v);
  else store16(p, v);
}

template <bool STREAM, typename T, typename F>
__device__ __forceinline__ void map_piece(const T* z, T* out, int len, F f) {
  constexpr int E = kVec<T>;
  u32x4 v[kBwdVectors];
#pragma unroll
  for (int p = 0; p < kBwdVectors; ++p) {
    const int i = (p * kBwdThreads + (int)threadIdx.x) * E;
    if (i + E <= len) v[p] = load16(z + i);
  }
#pragma unroll
  for (int p = 0; p < kBwdVectors; ++p) {
    const int i = (p * kBwdThreads + (int)threadIdx.x) * E;
    if (i + E <= len) {
      float r[E];
#pragma unroll
      for (int j = 0; j < E; ++j) r[j] = f(elem<T>(v[p], j));
      store_vec<STREAM>(out + i, pack<T>(r));
    } else {
      for (int j = i; j < len; ++j) out[j] = static_cast<T>(f(to_f(z[j])));
    }
  }
}

template <bool STREAM, typename T>
__device__ __forceinline__ void zero_piece(T* out, int len) {
  constexpr int E = kVec<T>;
#pragma unroll
  for (int p = 0; p < kBwdVectors; ++p) {
    const int i = (p * kBwdThreads + (int)threadIdx.x) * E;
    if (i + E <= len) store_vec<STREAM>(out + i, u32x4{0, 0, 0, 0});
    else
      for (int j = i; j < len; ++j) out[j] = static_cast<T>(0.f);
  }
}

// Bound by memory. 4096 x 30528 fp32 with 15 % of the rows labelled, 75 MB read
// and 500 written: 86 us (6.7 TB/s); all labelled 156 us (6.4 TB/s). Rows that
// were not looked at are only written.
template <typename T, bool ENT, bool STREAM>
__global__ __launch_bounds__(kBwdThreads) void logprobs_bwd_kernel(
    const T* __restrict__ logits, int64_t zs,
    const int64_t* __restrict__ tokens, const int64_t* __restrict__ top_ids,
    const RowStats* __restrict__ stats, const float* __restrict__ d_logprob,
    const float* __restrict__ d_entropy, const float* __restrict__ d_top,
    T* __restrict__ dz, int64_t rows, int V, int64_t pieces, int k, float c,
    float inv_t) {
  __shared__ int token_in_top;
  const int tid = threadIdx.x;
  for (int64_t i = blockIdx.x; i < rows * pieces; i += gridDim.x) {
    const int64_t w = rows * pieces - 1 - i, row = w / pieces;
    const int base = (int)(w - row * pieces) * kBwdTokens<T>;
    const int len = min(kBwdTokens<T>, V - base);
    const T* z = logits + row * zs + base;
    T* out = dz + row * V + base;
    const RowStats s = stats[row];
    if (s.inv_s == 0.f) {
      zero_piece<STREAM>(out, len);
      continue;
    }
    const int64_t token = d_logprob ? tokens[row] : -1;
    const float up = d_logprob ? d_logprob[row] : 0.f;
    const float dh = ENT ? d_entropy[row] : 0.f;
    float a = 0.f;
    if (d_top) {
      for (int i = tid & 63; i < k; i += 64) a += d_top[row * k + i];
      a = wave_reduce(a, Add{});
    }
    a += up;
    // a token outside of the vocabulary has no gradient that is a number
    if (d_logprob && (token < 0 || token >= V)) a = NAN;
    const float scale = -s.inv_s * inv_t;
    auto spread = [&](float v) {
      const float y = (v - s.m) * c;
      const float e = __builtin_amdgcn_exp2f(y) * scale;
      if constexpr (ENT)
        // e is 0 from -150 on: no product with it may be infinite
        return e * fmaf(dh, fmaf(fmaxf(y, -256.f), (float)kLn2, s.a), a);
      return e * a;
    };
    map_piece<STREAM>(z, out, len, spread);
    if (!d_logprob && !d_top) continue;
    // the named tokens of this piece again, with what is theirs; the token
    // itself where it is not one of the top
    if (tid == 0) token_in_top = 0;
    __syncthreads();
    if (d_top && tid < k) {
      const int64_t id = top_ids[row * k + tid];
      float g = d_top[row * k + tid];
      if (id == token) {
        g += up;
        token_in_top = 1;
      }
      if (id >= base && id - base < len) {
        const int i = (int)(id - base);
        out[i] = static_cast<T>(fmaf(g, inv_t, spread(to_f(z[i]))));
      }
    }
    __syncthreads();
    if (tid == 0 && !token_in_top && token >= base && token - base < len) {
      const int i = (int)(token - base);
      out[i] = static_cast<T>(fmaf(up, inv_t, spread(to_f(z[i]))));
    }
    __syncthreads();
  }
}

// Bound by memory: 4096 x 30528 bf16, 80 us (6.2 TB/s); 614 rows of fp32,
// 150 MB in all, 25 us (6.1 TB/s).
template <typename T, bool STREAM>
__global__ __launch_bounds__(kBwdThreads) void distill_bwd_kernel(
    const T* __restrict__ logits, int64_t zs,
    const int64_t* __restrict__ ids, const float* __restrict__ named,
    const DistillRow* __restrict__ stats, const float* __restrict__ d_loss,
    T* __restrict__ dz, int64_t rows, int V, int64_t pieces, int k, float c,
    float t) {
  const int tid = threadIdx.x;
  for (int64_t i = blockIdx.x; i < rows * pieces; i += gridDim.x) {
    const int64_t w = rows * pieces - 1 - i, row = w / pieces;
    const int base = (int)(w - row * pieces) * kBwdTokens<T>;
    const int len = min(kBwdTokens<T>, V - base);
    const T* z = logits + row * zs + base;
    T* out = dz + row * V + base;
    const DistillRow s = stats[row];
    if (s.live == 0.f) {
      zero_piece<STREAM>(out, len);
      continue;
    }
    const float g = d_loss[row] * t, outside = s.outside * g;
    // with a tail what this gives the named tokens may be anything
    map_piece<STREAM>(z, out, len, [&](float v) {
      return __builtin_amdgcn_exp2f((v - s.m) * c) * outside;
    });
    __syncthreads();
    if (tid < k) {
      const int64_t id = ids[row * k + tid];
      if (id >= base && id - base < len)
        out[(int)(id - base)] = static_cast<T>(named[row * k + tid] * g);
    }
  }
}

// ------------------------------------------------------------------ launches
int grid_for(int64_t work) {
  return (int)(work < kMaxBlocks ? work : kMaxBlocks);
}

// log2(e) / T: exp(t) is exp2 of the distance times this
Factor exp2_factor(double t) {
  const double exact = 1.4426950408889634074 / t;
  return {(float)exact, exact, (exact / (double)(float)exact - 1.0) * kLn2};
}

// Slices of a row, of up to `most` 16-byte vectors; of up to `few` where that
// would give fewer blocks than there are compute units. Smaller slices overlap
// their phases better, larger ones leave fewer lists to make and join. Of 4096
// and 2048 vectors, us: 614 of 4096 rows of 30528 fp32, no top, 28.8 and 25.0;
// 4096 rows of 30528 bf16 with a top of 32 76.0 and 79.5, of 128 123 and 197;
// distillation of the same without a tail 52.3 and 50.6. Few rows, of 4096 and
// 1024 vectors: 1 x 131072 bf16, top 8, 12.7 and 11.9, top 64 16.5 and 31.4;
// 2 x 600011 fp32, top 16, 15.7 and 20.5, top 128 46 and 130.
struct Cut {
  int64_t each, slices;      // vectors of a slice, slices of a row
};
constexpr int kLargeSlice = 4096, kSmallSlice = 2048, kFewRows = 1024;

Cut cut_row(int64_t rows, int V, int per_vector, int64_t most, int64_t few) {
  const int64_t vecs = ((int64_t)V + per_vector - 1) / per_vector;
  if (rows * ((vecs + most - 1) / most) < 256) most = few;
  const int64_t slices = (vecs + most - 1) / most;
  const int64_t each = (vecs + slices - 1) / slices;
  return {each, (vecs + each - 1) / each};             // none of them empty
}

// Log probabilities of few rows: a block to each row if it can hold that, which
// then needs no second kernel. A row of 30528 fp32 with a top of 8, us: 11.5 in
// slices, 8.3 whole; 64 such rows 13.2 and 9.7.
constexpr int kWhole = 8192;
Cut cut_logprobs(int type, int64_t rows, int V, int k) {
  const int E = type == kF32 ? 4 : 8;
  const int64_t vecs = ((int64_t)V + E - 1) / E;
  if (rows < 256 && vecs <= kWhole) return {vecs, 1};
  return k ? cut_row(rows, V, E, kLargeSlice, kLargeSlice)
           : cut_row(rows, V, E, kSmallSlice, kFewRows);
}
Cut cut_distill(int type, int64_t rows, int V) {
  return cut_row(rows, V, type == kF32 ? 4 : 8, kSmallSlice, kFewRows);
}

// Whether rows that are one slice are finished in their block: where all of
// them run at once (4 waves on each SIMD) this saves a launch, and with more
// the larger kernel's registers cost more than that. Us, apart and together:
// 4096 x 1000 fp32, top 4, 14.7 and 10.5; 300 x 30528 bf16, top 32, 16.6 and
// 12.9; 4096 x 30528 bf16, top 32, 76 and 90.
bool finish_there(const Cut& c, int64_t rows, int threads) {
  return c.slices == 1 && rows * threads <= 256 * 16 * 64;
}

// The smallest block that holds a slice. k: of how many alternatives, 0 of
// none. A wave by itself has a floor for no more than 64 of them, and ranks
// them slowly.
template <bool TOP, int MOST, typename F>
void with_cut(const Cut& c, int k, F f) {
  if (c.each <= 256 && k <= 16) {
    f(Int<64>{}, Int<4>{});
    return;
  }
  if constexpr (MOST > kLargeSlice) {
    if (c.each > kLargeSlice) {
      f(Int<1024>{}, Int<8>{});
      return;
    }
  }
  if constexpr (MOST > kSmallSlice) {
    if (c.each > kSmallSlice) {
      f(Int<512>{}, Int<8>{});
      return;
    }
  }
  if constexpr (TOP) {
    if (c.each <= 256) {
      f(Int<256>{}, Int<1>{});
      return;
    }
  }
  if (c.each <= 1024) f(Int<256>{}, Int<4>{});
  else f(Int<256>{}, Int<8>{});
}

template <typename F>
void with_type(int type, F f) {
  if (type == kF32) f(float{});
  else if (type == kBF16) f(bf16{});
  else f(f16{});
}

int per_vector(int type) { return type == kF32 ? 4 : 8; }

}  // namespace

// Bytes that a forward pass leaves for the kernel that joins the slices; 0
// where there is none.
int64_t dear_logprobs_work(int type, int64_t rows, int V, int k) {
  const Cut cut = cut_logprobs(type, rows, V, k);
  bool whole = false;
  auto ask = [&](auto nt, auto) {
    whole = finish_there(cut, rows, decltype(nt)::value);
  };
  if (k) with_cut<true, kWhole>(cut, k, ask);
  else with_cut<false, kWhole>(cut, 0, ask);
  return whole ? 0
               : rows * cut.slices *
                     (int64_t)(sizeof(Sums) + k * sizeof(uint64_t));
}
int64_t dear_distill_work(int type, int64_t rows, int V) {
  return rows * cut_distill(type, rows, V).slices * (int64_t)sizeof(Sums);
}

int dear_logprobs_fwd(hipStream_t st, int type, const void* logits, int64_t zs,
                      const int64_t* tokens, int64_t ignore, int64_t rows,
                      int V, int k, double t, float* logprob, float* entropy,
                      float* top_lp, int64_t* top_ids, void* stats,
                      void* work) {
  const Cut cut = cut_logprobs(type, rows, V, k);
  Sums* part = (Sums*)work;              // and behind the records the lists
  const LogprobArgs a = {tokens, zs, ignore, rows, V, k,
                         (int)(cut.each * per_vector(type)), cut.slices,
                         exp2_factor(t), 1.0 / t, logprob, entropy,
                         top_lp, top_ids, (RowStats*)stats, part,
                         (uint64_t*)(part + rows * cut.slices)};
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    auto launch = [&](auto nt, auto nv, auto top, auto whole) {
      constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value;
      hipLaunchKernelGGL(
          (logprobs_slice_kernel<T, NT, NV, decltype(top)::value,
                                 decltype(whole)::value>),
          dim3(grid_for(rows * cut.slices)), dim3(NT), 0, st,
          (const T*)logits, a);
    };
    auto run = [&](auto nt, auto nv, auto top) {
      if (finish_there(cut, rows, decltype(nt)::value)) {
        launch(nt, nv, top, Int<1>{});
        return;
      }
      // rows in longer slices are few, and were finished
      if constexpr (decltype(nt)::value * decltype(nv)::value <=
                    (decltype(top)::value ? kLargeSlice : kSmallSlice))
        launch(nt, nv, top, Int<0>{});
      hipLaunchKernelGGL((logprobs_finish_kernel<T>),
                         dim3(grid_for((rows + 3) / 4)), dim3(256), 0, st,
                         (const T*)logits, a);
    };
    if (k)
      with_cut<true, kWhole>(
          cut, k, [&](auto nt, auto nv) { run(nt, nv, Int<1>{}); });
    else
      with_cut<false, kWhole>(
          cut, 0, [&](auto nt, auto nv) { run(nt, nv, Int<0>{}); });
  });
  return (int)hipGetLastError();
}

int dear_logprobs_bwd(hipStream_t st, int type, const void* logits, int64_t zs,
                      const int64_t* tokens, const int64_t* top_ids,
                      const void* stats, const float* d_logprob,
                      const float* d_entropy, const float* d_top, void* dz,
                      int64_t rows, int V, int k, double t) {
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    const int64_t pieces = ((int64_t)V + kBwdTokens<T> - 1) / kBwdTokens<T>;
    const dim3 grid(grid_for(rows * pieces)), block(kBwdThreads);
    const float c = exp2_factor(t).c, inv_t = (float)(1.0 / t);
    auto launch = [&](auto ent, auto stream) {
      hipLaunchKernelGGL((logprobs_bwd_kernel<T, decltype(ent)::value,
                                              decltype(stream)::value>),
                         grid, block, 0, st, (const T*)logits, zs, tokens,
                         top_ids, (const RowStats*)stats, d_logprob, d_entropy,
                         d_top, (T*)dz, rows, V, pieces, k, c, inv_t);
    };
    const bool stream = rows * V * (int64_t)sizeof(T) > kStreamBytes;
    auto with_ent = [&](auto ent) {
      stream ? launch(ent, Int<1>{}) : launch(ent, Int<0>{});
    };
    d_entropy ? with_ent(Int<1>{}) : with_ent(Int<0>{});
  });
  return (int)hipGetLastError();
}

int dear_distill_fwd(hipStream_t st, int type, bool tail, const void* logits,
                     int64_t zs, const int64_t* ids, const float* teacher,
                     int64_t rows, int V, int k, double t, float* loss,
                     float* named, void* stats, void* work) {
  const Cut cut = cut_distill(type, rows, V);
  const DistillArgs a = {ids, teacher, zs, rows, V, k,
                         (int)(cut.each * per_vector(type)), cut.slices,
                         exp2_factor(t), t, 1.0 / t, loss, named,
                         (DistillRow*)stats, (Sums*)work};
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    with_cut<false, kSmallSlice>(cut, 0, [&](auto nt, auto nv) {
      constexpr int NT = decltype(nt)::value, NV = decltype(nv)::value;
      const dim3 grid(grid_for(rows * cut.slices)), block(NT);
      if (tail)
        hipLaunchKernelGGL((distill_slice_kernel<T, NT, NV, true>), grid,
                           block, 0, st, (const T*)logits, a);
      else
        hipLaunchKernelGGL((distill_slice_kernel<T, NT, NV, false>), grid,
                           block, 0, st, (const T*)logits, a);
    });
    const dim3 rest(grid_for((rows + 3) / 4));
    auto finish = [&](auto with_tail, auto n) {
      hipLaunchKernelGGL((distill_finish_kernel<T, decltype(with_tail)::value,
                                                decltype(n)::value>),
                         rest, dim3(256), 0, st, (const T*)logits, a);
    };
    if (k <= 64) tail ? finish(Int<1>{}, Int<1>{}) : finish(Int<0>{}, Int<1>{});
    else tail ? finish(Int<1>{}, Int<2>{}) : finish(Int<0>{}, Int<2>{});
  });
  return (int)hipGetLastError();
}

int dear_distill_bwd(hipStream_t st, int type, const void* logits, int64_t zs,
                     const int64_t* ids, const float* named, const void* stats,
                     const float* d_loss, void* dz, int64_t rows, int V, int k,
                     double t) {
  with_type(type, [&](auto zero) {
    using T = decltype(zero);
    const int64_t pieces = ((int64_t)V + kBwdTokens<T> - 1) / kBwdTokens<T>;
    auto launch = [&](auto stream) {
      hipLaunchKernelGGL((distill_bwd_kernel<T, decltype(stream)::value>),
                         dim3(grid_for(rows * pieces)), dim3(kBwdThreads), 0,
                         st, (const T*)logits, zs, ids, named,
                         (const DistillRow*)stats, d_loss, (T*)dz, rows, V,
                         pieces, k, exp2_factor(t).c, (float)t);
    };
    rows * V * (int64_t)sizeof(T) > kStreamBytes ? launch(Int<1>{})
                                                 : launch(Int<0>{});
  });
  return (int)hipGetLastError();
}
