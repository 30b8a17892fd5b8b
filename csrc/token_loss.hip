// Log-probabilities of given tokens, and the losses built on them (MI355X).
//
// For a row of logits x and a token t:
//   lp = x_t - lse,  lse = log sum_j exp(x_j)
//   d lp / d x_j = [j = t] - exp(x_j - lse)
// Every loss here is a function of the lp alone, so a step is three passes
// over memory: the forward reads the logits once (running reference and sum),
// a finishing kernel turns the row statistics into lp, the loss and each
// row's d loss / d lp, and the backward reads the logits once more and
// writes the gradient.  Rows whose target is ignored are not read, nor, in
// the backward, rows whose coefficient is zero (clipped tokens): their
// gradient is written as zeros.
//
// Exponentials are fp32; their long sums and what follows them (log,
// differences to other log-probabilities, sums over tokens) are fp64, because
// the losses take small differences of large sums.  For the same reason the
// sums must not be off the same way in every row: see Part.

#include <hip/hip_runtime.h>

#include "elem.h"

namespace {

using elem::kVec;

constexpr int kThreads = 256;

struct Shape {
  long rows, vocab;        // rows = outer * inner
  long inner;              // rows that follow each other at row_stride
  long outer_stride, row_stride;  // of the logits, in elements
};

template <typename T>
__device__ __forceinline__ const T* row_of(const T* x, const Shape& s,
                                           long row) {
  return x + (row / s.inner) * s.outer_stride +
         (row % s.inner) * s.row_stride;
}

__device__ __forceinline__ bool is_live(long t, long vocab, long ignore) {
  return t != ignore && t >= 0 && t < vocab;
}

// log2 e: rounded, what that leaves, and with 16 bits, so that its product
// with a bf16 number is exact.
constexpr float kLog2e = 1.4426950216293335f;
constexpr float kLog2eLow = 1.925963033500011e-08f;
constexpr float kLog2e16 = 47274.f / 32768.f;
constexpr double kLn2 = 0.6931471805599453;
// v_exp_f32 comes out 3.2e-9 low on the average of its arguments; given back,
// fp32 rows are within 2e-10 on average.
constexpr double kExpBias = 3.2e-9;

// exp(d)
__device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(
      __builtin_fmaf(d, kLog2e, d * kLog2eLow));
}

// A part of a row: its maximum, and  sum = sum_j 2^(x_j B - k).  Sequences add
// the lp of many tokens up, so what matters is that the sums are not off the
// same way in every row:
// * k is a whole number near max B, so parts join by exact powers of two; with
//   the maximum as the reference each joining multiplies a rounded
//   exponential in;
// * B is log2 e a share kCut short, 1.3e-8 by its rounding to fp32.  A bf16 row
//   is a few hundred values whose products with that round alike in every
//   row (1e-8 of lp): there B has 16 bits, the products are exact and kCut is
//   4.9e-6.  Both are given back by
//     log sum exp(x) = log sum exp((1 - kCut) x) + kCut E[x] + O(kCut^2 Var),
//   E[x] = moment / sum;
// * a few values are added in fp32, in pairs, and these sums in fp64; what the
//   fp32 sum with the largest term lost is added afterwards.
// At 128256 normal values lp (in fp64) is off by 2e-9 in the mean square and
// by less than 1e-9 on average, in every type; 4e-10 to 8e-10 where one token
// has most of the weight.
struct Part {
  double sum;
  float max, k, moment;
};

template <bool BF16>
constexpr float kBase = BF16 ? kLog2e16 : kLog2e;
template <bool BF16>
constexpr double kCut = 1. - (double)kBase<BF16> * kLn2;

// From these maxima on the next smaller value of the type lies 32 or more
// below: only the values equal to the maximum count, and sum is their number.
// It keeps x B within what fp32 resolves, and kCut E[x] small.
template <bool BF16>
constexpr float kHuge = BF16 ? 8192.f : 536870912.f;
constexpr float kLeast = -1e9f;  // first k

__device__ __forceinline__ Part nothing() {
  return Part{0., -__builtin_huge_valf(), kLeast, 0.f};
}

template <bool BF16>
__device__ __forceinline__ bool is_huge(float m) {
  return fabsf(m) >= kHuge<BF16> && fabsf(m) <= 3.402823466e38f;
}

__device__ __forceinline__ float shifted(float v, float by) {
  return __builtin_ldexpf(v, (int)fmaxf(by, -2000.f));
}
__device__ __forceinline__ double shifted(double v, float by) {
  return __builtin_ldexp(v, (int)fmaxf(by, -2000.f));
}

template <bool BF16>
__device__ __forceinline__ void join(Part& p, const Part& q) {
  if (is_huge<BF16>(p.max) || is_huge<BF16>(q.max)) {
    // the larger maximum takes all; NaN stays
    const double seen = p.sum + q.sum;
    if (seen != seen) p.sum = seen;
    else if (p.max == q.max) p.sum = seen;
    else if (q.max > p.max) p = q;
    p.max = fmaxf(p.max, q.max);
    return;
  }
  const float k = fmaxf(p.k, q.k);
  p.sum = shifted(p.sum, p.k - k) + shifted(q.sum, q.k - k);
  p.moment = shifted(p.moment, p.k - k) + shifted(q.moment, q.k - k);
  p.k = k;
  p.max = fmaxf(p.max, q.max);
}

__device__ __forceinline__ Part from_lane(const Part& p, int off) {
  return Part{__shfl_xor(p.sum, off), __shfl_xor(p.max, off),
              __shfl_xor(p.k, off), __shfl_xor(p.moment, off)};
}

// Elements of `row` up to the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T* p) {
  return (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) /
         (int)sizeof(T);
}

// 2^(x B - k)
template <bool BF16>
__device__ __forceinline__ float term(float x, float k) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(x, kBase<BF16>, -k));
}

// The terms of a few values and their sum in pairs.
template <bool BF16, int N>
__device__ __forceinline__ float sum_of(const float (&v)[N], float k,
                                        float (&x)[N]) {
  float sum[N];
  #pragma unroll
  for (int e = 0; e < N; ++e) sum[e] = x[e] = term<BF16>(v[e], k);
  #pragma unroll
  for (int half = N / 2; half > 0; half /= 2)
    #pragma unroll
    for (int e = 0; e < half; ++e) sum[e] += sum[e + half];
  return sum[0];
}

// One value, or a few at once, into a thread's part, where `here` becomes the
// place of its maximum.  -inf adds 0; +inf and NaN make the sum NaN.
template <bool BF16, int N>
__device__ __forceinline__ void take(const float (&v)[N], Part& p, int at,
                                     int& here) {
  float top = v[0];
  #pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, v[e]);
  if (top > p.max) {
    p.max = top;
    here = at;
  }
  const float k = ceilf(top * kLog2e);
  if (k > p.k) {
    p.sum = shifted(p.sum, p.k - k);
    p.moment = shifted(p.moment, p.k - k);
    p.k = k;
  }
  float x[N], moment = 0.f;
  p.sum += (double)sum_of<BF16>(v, p.k, x);
  #pragma unroll
  for (int e = 0; e < N; ++e)  // a masked value must not meet 0 * inf
    moment = __builtin_fmaf(x[e], fmaxf(v[e], -1e30f), moment);
  p.moment += moment;
}

// What the fp32 sum of a few values lost.
template <bool BF16, int N>
__device__ __forceinline__ double lost_of(const float (&v)[N], float k) {
  float x[N];
  const float sum = sum_of<BF16>(v, k, x);
  double exact = 0.;
  #pragma unroll
  for (int e = 0; e < N; ++e) exact += (double)x[e];
  return exact - (double)sum;
}

template <typename T, int N>
__device__ __forceinline__ void widen(const T* x, int step,
                                      float (&v)[N * kVec<T>]) {
  constexpr int V = kVec<T>;
  elem::vec<T, V> w[N];
  #pragma unroll
  for (int u = 0; u < N; ++u) w[u] = elem::load<false, V>(x + u * step);
  #pragma unroll
  for (int e = 0; e < N * V; ++e) v[e] = (float)w[e / V][e % V];
}

// What the backward needs of a row is saved as four floats: its maximum R,
// exp(R - lse), lp and the row's coefficient.
struct RowLp {
  float ref, inv;
  double lp;
};

template <bool BF16>
__device__ __forceinline__ RowLp finish(const Part& p, float xt) {
  RowLp r;
  if (is_huge<BF16>(p.max)) {
    // the difference first: a sum would lose the logarithm
    r.ref = p.max;
    r.inv = (float)(1. / p.sum);
    r.lp = ((double)xt - (double)p.max) - log(p.sum);
    return r;
  }
  // lse - max, from the largest term in fp64 and what the others add to it: a
  // token that is almost certain keeps its lp, and the bias is the others'
  const double top =
      exp2((double)p.max * (double)kBase<BF16> - (double)p.k);
  const double rest = p.sum - (double)term<BF16>(p.max, p.k);
  double over = log1p(rest * (1. + kExpBias) / top);
  if (rest > 0.)
    over += kCut<BF16> * ((double)p.moment / p.sum - (double)p.max);
  r.ref = p.max;
  r.inv = (float)exp(-over);
  r.lp = ((double)xt - (double)p.max) - over;
  return r;
}

// One block for each (row, piece of the vocabulary): stats[row, piece].
// A row starts at any element (odd vocabularies): the few up to a 16-byte
// boundary and behind the last whole 16 bytes are taken one by one.
// The target's logit goes along: the row's page is at hand here, while the
// finishing kernels would meet another one for each row.  With FINISH (one
// piece a row) a row's lp is written here.
//
// Bound by memory: 8192 rows of 128256 bf16, 65 % of them read, take 237 us
// (1.37 GB, 5.8 TB/s), all of them 376 us.  A thread takes 32 values between two
// looks at its maximum; the loads stay in the caches for the backward.
template <typename T, int THREADS, bool FINISH>
__global__ __launch_bounds__(THREADS) void row_stats_kernel(
    const T* __restrict__ logits, const long* __restrict__ target,
    Part* __restrict__ stats, float* __restrict__ picked,
    unsigned* __restrict__ ticket, Shape s, long ignore, int pieces,
    long piece, float4* __restrict__ saved, float* __restrict__ lp) {
  constexpr int V = kVec<T>;
  constexpr bool kBf16 = std::is_same_v<T, __bf16>;
  const long row = blockIdx.x;
  const int part = blockIdx.y;
  if (row == 0 && part == 0 && threadIdx.x == 0 && ticket) *ticket = 0;
  const long t = target[row];
  if (!is_live(t, s.vocab, ignore)) {
    if (FINISH && threadIdx.x == 0) {
      lp[row] = 0.f;
      if (saved) saved[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  const long begin = part * piece;
  const T* x = row_of(logits, s, row) + begin;
  const int n = (int)(min(s.vocab, begin + piece) - begin);
  const int head = min(head_of(x), n);
  const int body = (n - head) / V;
  const bool mine = threadIdx.x == 0 && t >= begin && t < begin + n;
  const float xt = mine ? (float)x[t - begin] : 0.f;
  Part p = nothing();
  int here = -1;
  const T* xv = x + head;
  int i = threadIdx.x;
  for (; i + 3 * THREADS < body; i += 4 * THREADS) {
    float v[4 * V];
    widen<T, 4>(xv + i * V, THREADS * V, v);
    take<kBf16>(v, p, i, here);
  }
  for (; i < body; i += THREADS) {
    float v[V];
    widen<T, 1>(xv + i * V, 0, v);
    take<kBf16>(v, p, i, here);
  }
  const int rest = n - body * V;  // head and tail
  if ((int)threadIdx.x < rest) {
    const int at = (int)threadIdx.x < head ? (int)threadIdx.x
                                           : (int)threadIdx.x + body * V;
    const float v[1] = {(float)x[at]};
    take<kBf16>(v, p, -1, here);
  }
  // one reference for the block, then plain sums
  __shared__ float tops[THREADS / 64], moments[THREADS / 64];
  __shared__ double sums[THREADS / 64];
  float top = p.max;
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1)
    top = fmaxf(top, __shfl_xor(top, off));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  #pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, tops[w]);
  const float k = fmaxf(ceilf(top * kLog2e), kLeast);
  if (is_huge<kBf16>(top)) {
    p = nothing();
    for (int at = threadIdx.x; at < n; at += THREADS) {
      const float v = (float)x[at];
      p.sum += v != v ? v : v == top ? 1.f : 0.f;
    }
  } else {
    if (p.max == top && here >= 0) {
      // next to the largest term the fp32 sum lost most: 2e-8 of the row
      // where one token has most of the weight
      if (here + 3 * THREADS < body) {
        float v[4 * V];
        widen<T, 4>(xv + here * V, THREADS * V, v);
        p.sum += lost_of<kBf16>(v, p.k);
      } else {
        float v[V];
        widen<T, 1>(xv + here * V, 0, v);
        p.sum += lost_of<kBf16>(v, p.k);
      }
    }
    p.sum = shifted(p.sum, p.k - k);
    p.moment = shifted(p.moment, p.k - k);
  }
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    p.sum += __shfl_xor(p.sum, off);
    p.moment += __shfl_xor(p.moment, off);
  }
  if ((threadIdx.x & 63) == 0) {
    sums[threadIdx.x >> 6] = p.sum;
    moments[threadIdx.x >> 6] = p.moment;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    #pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) {
      p.sum += sums[w];
      p.moment += moments[w];
    }
    p.max = top;
    p.k = k;
    if (!FINISH) {
      stats[row * pieces + part] = p;
      if (mine) picked[row] = xt;
      return;
    }
    const RowLp r = finish<kBf16>(p, xt);
    lp[row] = (float)r.lp;
    if (saved) saved[row] = make_float4(r.ref, r.inv, (float)r.lp, 1.f);
  }
}

// Joins the pieces of a row in their order.
template <bool BF16>
__device__ __forceinline__ RowLp row_lp(const Part* __restrict__ stats,
                                        const float* __restrict__ picked,
                                        long row, int pieces) {
  Part a = stats[row * pieces];
  #pragma unroll 4
  for (int p = 1; p < pieces; ++p) join<BF16>(a, stats[row * pieces + p]);
  return finish<BF16>(a, picked[row]);
}

// A wave for each row, of which there are few and the pieces many.
template <bool BF16>
__global__ __launch_bounds__(64) void lp_finish_kernel(
    const long* __restrict__ target, const Part* __restrict__ stats,
    const float* __restrict__ picked, float4* __restrict__ saved,
    float* __restrict__ lp, Shape s, long ignore, int pieces) {
  const long row = blockIdx.x;
  const int lane = threadIdx.x;
  if (!is_live(target[row], s.vocab, ignore)) {
    if (lane == 0) {
      lp[row] = 0.f;
      if (saved) saved[row] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    return;
  }
  Part p = nothing();
  for (int i = lane; i < pieces; i += 64)
    join<BF16>(p, stats[row * pieces + i]);
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) join<BF16>(p, from_lane(p, off));
  if (lane == 0) {
    const RowLp r = finish<BF16>(p, picked[row]);
    lp[row] = (float)r.lp;
    if (saved) saved[row] = make_float4(r.ref, r.inv, (float)r.lp, 1.f);
  }
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
  __shared__ double sums[THREADS / 64];
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.;
  #pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) v += sums[w];
  return v;
}

// True in the block that arrives last, once it can read what the thread 0 of
// the others stored before.  Only thread 0 orders memory: a fence writes an
// L2 back, and one for each wave took longer than the kernel's own work.
__device__ __forceinline__ bool last_block(unsigned* ticket) {
  __shared__ bool last;
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL,
                                  __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  __syncthreads();
  return last;
}

// Values of another block: past the caches that may hold older ones.
__device__ __forceinline__ double from_block(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct PolicyArgs {
  double low, high;  // bounds of the ratio
  double kl;
};

// rho = exp(lp - old);  token loss = -min(rho A, clip(rho) A)
//                                    + kl (e^d - d - 1),  d = ref - lp
// The partial sums of the blocks are added in their order by the last one.
template <bool BF16>
__global__ __launch_bounds__(kThreads) void policy_finish_kernel(
    const long* __restrict__ target, const Part* __restrict__ stats,
    const float* __restrict__ picked, const float* __restrict__ old_lp,
    const float* __restrict__ adv, const float* __restrict__ ref_lp,
    float4* __restrict__ saved, double* __restrict__ partial,
    unsigned* __restrict__ ticket, float* __restrict__ loss,
    float* __restrict__ inv_count, Shape s, long ignore, int pieces,
    PolicyArgs a) {
  const long row = (long)blockIdx.x * kThreads + threadIdx.x;
  double tok = 0., count = 0.;
  if (row < s.rows) {
    const long t = target[row];
    float4 keep = make_float4(0.f, 0.f, 0.f, 0.f);
    if (is_live(t, s.vocab, ignore)) {
      const RowLp r = row_lp<BF16>(stats, picked, row, pieces);
      const double rho = exp(r.lp - (double)old_lp[row]);
      const double A = (double)adv[row];
      const double free = rho * A;
      const double held = fmin(fmax(rho, a.low), a.high) * A;
      // the gradient flows where the free term is the smaller one or both
      // are the same; NaN takes this side as well and stays NaN
      const bool clipped = free > held;
      tok = clipped ? -held : -free;
      double coef = clipped ? 0. : -free;
      if (ref_lp) {
        const double d = (double)ref_lp[row] - r.lp;
        const double e = exp(d);
        // a token that the policy rules out: not inf - inf
        tok += a.kl * (d == __builtin_huge_val() ? e : e - d - 1.);
        coef += a.kl * (1. - e);
      }
      count = 1.;
      keep = make_float4(r.ref, r.inv, (float)r.lp, (float)coef);
    }
    saved[row] = keep;
  }
  tok = block_sum<kThreads>(tok);
  count = block_sum<kThreads>(count);
  if (threadIdx.x == 0) {
    partial[2 * blockIdx.x] = tok;
    partial[2 * blockIdx.x + 1] = count;
  }
  if (!last_block(ticket)) return;
  tok = count = 0.;
  for (unsigned b = threadIdx.x; b < gridDim.x; b += kThreads) {
    tok += from_block(partial + 2 * b);
    count += from_block(partial + 2 * b + 1);
  }
  tok = block_sum<kThreads>(tok);
  count = block_sum<kThreads>(count);
  if (threadIdx.x == 0) {
    const double n = count > 0. ? count : 1.;
    *loss = (float)(tok / n);
    *inv_count = (float)(1. / n);
  }
}

constexpr int kPairThreads = 512;

// One block for each pair: the rewards beta * sum(lp - ref) of its two
// sequences, h = their difference, and the pair's
//   loss = (1 - eps) softplus(-h) + eps softplus(h).
// One long pair leaves the chip idle: 2 x 8192 tokens take 56 us, 510 rows a
// pair 6 us.
// Rows of the chosen sequence get d loss / d lp = slope[pair], of the rejected
// one its negative; the mean over the pairs is in it.
template <bool BF16>
__global__ __launch_bounds__(kPairThreads) void prefer_finish_kernel(
    const long* __restrict__ target, const Part* __restrict__ stats,
    const float* __restrict__ picked, const float* __restrict__ ref_lp,
    float4* __restrict__ saved, double* __restrict__ partial,
    unsigned* __restrict__ ticket, float* __restrict__ loss,
    float* __restrict__ rewards, float* __restrict__ slope, Shape s,
    long ignore, int pieces, long seq, double beta, double eps) {
  const long pairs = gridDim.x, pair = blockIdx.x;
  double sums[2] = {0., 0.};
  #pragma unroll 2
  for (long i = threadIdx.x; i < 2 * seq; i += kPairThreads) {
    const int side = i >= seq;
    const long row = side ? (pair + pairs - 1) * seq + i : pair * seq + i;
    float4 keep = make_float4(0.f, 0.f, 0.f, 0.f);
    if (is_live(target[row], s.vocab, ignore)) {
      const RowLp r = row_lp<BF16>(stats, picked, row, pieces);
      const double d = r.lp - (double)ref_lp[row];
      sums[0] += side ? 0. : d;
      sums[1] += side ? d : 0.;
      keep = make_float4(r.ref, r.inv, (float)r.lp, side ? -1.f : 1.f);
    }
    saved[row] = keep;
  }
  const double gain[2] = {beta * block_sum<kPairThreads>(sums[0]),
                          beta * block_sum<kPairThreads>(sums[1])};
  const double h = gain[0] - gain[1];
  const double tail = log1p(exp(-fabs(h)));
  const double e = exp(-h);  // sigmoid(-h) = e / (1 + e)
  const double down = h > 0. ? e / (1. + e) : 1. / (1. + exp(h));
  const double dh = eps - down;  // d loss / d h
  if (threadIdx.x == 0) {
    slope[pair] = (float)(beta * dh / (double)pairs);
    rewards[pair] = (float)gain[0];
    rewards[pair + pairs] = (float)gain[1];
    // without smoothing a margin of +inf costs nothing: not 0 * inf
    partial[pair] = (1. - eps) * (fmax(-h, 0.) + tail) +
                    (eps > 0. ? eps * (fmax(h, 0.) + tail) : 0.);
  }
  if (!last_block(ticket)) return;
  double sum = 0.;
  for (long p = threadIdx.x; p < pairs; p += kPairThreads)
    sum += from_block(partial + p);
  sum = block_sum<kPairThreads>(sum);
  if (threadIdx.x == 0) *loss = (float)(sum / (double)pairs);
}

// A factor for groups of `rows` rows, starting again after `groups` of them;
// none where `at` is null.
struct Scale {
  const float* at;
  long rows, groups;
};

// dx_j = c ([j = t] - exp(x_j - R) exp(R - lse)),  c = coef * up * scale.
//
// Bound by memory: 8192 rows of 128256 bf16, 65 % of them read, take 600 us
// (3.47 GB, 5.8 TB/s).  Blocks of 1024 threads with four accesses each beat
// 256 threads by 8 %.
template <typename T, int THREADS, bool NT>
__global__ __launch_bounds__(THREADS) void lp_bwd_kernel(
    const T* __restrict__ logits, const long* __restrict__ target,
    const float4* __restrict__ saved, const float* __restrict__ up,
    int up_step, Scale scale, T* __restrict__ dlogits, Shape s, long ignore,
    long piece) {
  constexpr int V = kVec<T>;
  using Vec = elem::vec<T, V>;
  const long row = blockIdx.x;
  const long begin = blockIdx.y * piece;
  const int n = (int)(min(s.vocab, begin + piece) - begin);
  T* dx = dlogits + row * s.vocab + begin;
  const long t = target[row];
  const float4 r = saved[row];
  float c = 0.f;
  if (is_live(t, s.vocab, ignore)) {
    c = r.w * up[row * up_step];
    if (scale.at) c *= scale.at[row / scale.rows % scale.groups];
  }
  const int head = min(head_of(dx), n);
  const int body = (n - head) / V;
  const int rest = n - body * V;
  const int lone = (int)threadIdx.x < head ? (int)threadIdx.x
                                           : (int)threadIdx.x + body * V;
  T* dv = dx + head;
  if (c == 0.f) {
    const Vec zero = (Vec)(T)0.f;
    for (int i = threadIdx.x; i < body; i += THREADS)
      elem::store<NT, V>(dv + i * V, zero);
    if ((int)threadIdx.x < rest) dx[lone] = (T)0.f;
    return;
  }
  const T* x = row_of(logits, s, row) + begin;
  const T* xv = x + head;  // of another row stride: on other boundaries
  const float k = -c * r.y;
  // 1 - p of a token that is almost certain loses its digits
  const T at_target = (T)(-c * expm1f(r.z));
  const long at = t - begin;  // may lie in another piece
  const auto slope = [&](const Vec& w) {
    Vec o;
    #pragma unroll
    for (int e = 0; e < V; ++e) o[e] = (T)(k * exp_of((float)w[e] - r.x));
    return o;
  };
  int i = threadIdx.x;
  for (; i + 3 * THREADS < body; i += 4 * THREADS) {
    Vec w[4];
    #pragma unroll
    for (int u = 0; u < 4; ++u)
      w[u] = elem::load<NT, V>(xv + (i + u * THREADS) * V);
    #pragma unroll
    for (int u = 0; u < 4; ++u)
      elem::store<NT, V>(dv + (i + u * THREADS) * V, slope(w[u]));
  }
  for (; i < body; i += THREADS)
    elem::store<NT, V>(dv + i * V, slope(elem::load<NT, V>(xv + i * V)));
  if ((int)threadIdx.x < rest)
    dx[lone] = (T)(k * exp_of((float)x[lone] - r.x));
  __syncthreads();  // the target's own value last
  if (threadIdx.x == 0 && at >= 0 && at < n) dx[at] = at_target;
}

// How a call reads the logits.
struct Call {
  Shape s;
  long ignore;
  int pieces;
  long piece;
};

// Few rows are split over the vocabulary so that the whole chip reads.
void split(long rows, long vocab, int& pieces, long& piece) {
  long want = (1024 + rows - 1) / rows;
  want = std::max<long>(1, std::min<long>(want, (vocab + 4095) / 4096));
  // whole 16 bytes, so that all pieces of a row are aligned alike
  piece = (vocab + want - 1) / want;
  piece = (piece + 7) / 8 * 8;
  pieces = (int)((vocab + piece - 1) / piece);
}

// logits [rows, V] or [outer, inner, V] with a unit last stride.
Call plan(const at::Tensor& logits, long ignore) {
  const bool flat = logits.dim() == 2;
  Call c;
  c.s.vocab = logits.size(-1);
  c.s.inner = std::max<long>(1, logits.size(-2));
  c.s.rows = flat ? logits.size(0) : logits.size(0) * logits.size(1);
  c.s.row_stride = logits.stride(-2);
  c.s.outer_stride = flat ? 0 : logits.stride(0);
  // a launch has fewer than 2^32 threads along x
  TORCH_CHECK_VALUE(c.s.rows < (1L << 22) && c.s.vocab < (1L << 30),
                    "Stoke -- losses on logits take fewer than 2^22 "
                    "positions of fewer than 2^30 logits");
  c.ignore = ignore;
  c.pieces = 1;
  c.piece = c.s.vocab;
  if (c.s.rows > 0) split(c.s.rows, c.s.vocab, c.pieces, c.piece);
  return c;
}

void check(const at::Tensor& logits, const at::Tensor& target,
           const char* what) {
  TORCH_CHECK_VALUE(
      logits.is_cuda() && logits.dim() >= 2 && logits.size(-1) >= 1 &&
          (logits.scalar_type() == at::kBFloat16 ||
           logits.scalar_type() == at::kHalf ||
           logits.scalar_type() == at::kFloat),
      "Stoke -- ", what, " takes floating logits [..., V], got ",
      logits.scalar_type(), " ", logits.sizes());
  TORCH_CHECK_VALUE(
      target.scalar_type() == at::kLong &&
          target.device() == logits.device() &&
          target.sizes() == logits.sizes().slice(0, logits.dim() - 1),
      "Stoke -- ", what, " takes int64 targets of the logits' shape without "
      "the vocabulary on their device, got ", target.scalar_type(), " ",
      target.sizes(), " for logits ", logits.sizes());
}

// The kernels' layout: 2-D logits, or 3-D with any two leading strides.
at::Tensor rows_of(const at::Tensor& logits) {
  at::Tensor x = logits;
  if (x.dim() > 3) x = x.flatten(0, -3);
  if (x.size(-1) > 1 && x.stride(-1) != 1) x = x.contiguous();
  return x;
}

// Constant values for each token in contiguous fp32.
at::Tensor per_token(const at::Tensor& v, const at::Tensor& target,
                     const char* what) {
  TORCH_CHECK_VALUE(!v.requires_grad(), "Stoke -- ", what,
                    " is a constant of the loss; detach() it");
  bool fits = v.is_floating_point() && v.device() == target.device() &&
              v.dim() == target.dim();
  for (int64_t i = 0; fits && i < v.dim(); ++i)
    fits = v.size(i) == target.size(i) || v.size(i) == 1;
  TORCH_CHECK_VALUE(fits, "Stoke -- ", what,
                    " must hold floating values for targets ",
                    target.sizes(), " (sizes of 1 broadcast) on their "
                    "device, got ", v.scalar_type(), " ", v.sizes());
  at::Tensor x = v;
  if (x.scalar_type() != at::kFloat) x = x.to(at::kFloat);
  if (x.sizes() != target.sizes()) x = x.expand(target.sizes());
  return x.contiguous();
}

// Of the logits as they were given: a copy of a leaf is not a leaf.
bool wants_grad(const at::Tensor& logits) {
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) return false;
  elem::check_capture({logits});
  return true;
}

// Temporary memory of a forward call: the blocks' partial sums in fp64, the
// ticket of the last block and the row statistics, in one allocation.
struct Scratch {
  at::Tensor store;
  double* partial;
  unsigned* ticket;
  Part* stats;
  float* picked;
  Scratch(const at::Tensor& like, long partials, const Call& c) {
    const long n = partials + 1;
    store = at::empty({n * 8 + c.s.rows * (c.pieces * (long)sizeof(Part) + 4)},
                      like.options().dtype(at::kByte));
    partial = (double*)store.data_ptr();
    ticket = (unsigned*)(partial + partials);
    stats = (Part*)(partial + n);
    picked = (float*)(stats + c.s.rows * c.pieces);
  }
};

template <typename T>
void launch_stats(const at::Tensor& logits, const at::Tensor& target,
                  const Call& c, const Scratch& tmp) {
  hipLaunchKernelGGL((row_stats_kernel<T, kThreads, false>),
                     dim3((unsigned)c.s.rows, (unsigned)c.pieces),
                     dim3(kThreads), 0, elem::stream(),
                     (const T*)logits.data_ptr(), target.data_ptr<long>(),
                     tmp.stats, tmp.picked, tmp.ticket, c.s, c.ignore,
                     c.pieces, c.piece, nullptr, nullptr);
}

// dlogits of a loss with `saved` row statistics.  up: one value for each row
// (token_logprobs) or one for all (the losses).
at::Tensor backward_of(const at::Tensor& logits, const at::Tensor& target,
                       const float4* saved, const at::Tensor& grad,
                       const Scale& scale, long ignore) {
  const c10::DeviceGuard guard(logits.device());
  const Call c = plan(logits, ignore);
  auto dlogits = at::empty(logits.sizes(), logits.options());
  const auto up = grad.to(at::kFloat).contiguous();
  STOKE_ELEM_SWITCH(logits.scalar_type(), "token_loss", {
    const auto launch = [&](auto threads, auto past_caches) {
      hipLaunchKernelGGL(
          (lp_bwd_kernel<T, threads, past_caches>),
          dim3((unsigned)c.s.rows, (unsigned)c.pieces), dim3(threads), 0,
          elem::stream(), (const T*)logits.data_ptr(),
          target.data_ptr<long>(), saved, up.data_ptr<float>(),
          up.numel() == 1 ? 0 : 1, scale, (T*)dlogits.data_ptr(), c.s,
          ignore, c.piece);
    };
    const auto sized = [&](auto past_caches) {
      if (c.piece >= 4 * 1024 * kVec<T>)
        launch(std::integral_constant<int, 1024>{}, past_caches);
      else
        launch(std::integral_constant<int, kThreads>{}, past_caches);
    };
    if (c.s.rows > 0) {
      // the next product reads the gradient: where it fits, it stays in the
      // last-level cache.  Past it the backward leaves there what the
      // forward read last: 8192 x 128256 bf16, about 60 % of the rows read,
      // forward and backward 790 us against 900 us through the caches; at
      // 512 rows (131 MB) 52 against 50 us.
      if (c.s.rows * c.s.vocab * (long)sizeof(T) > elem::kCached)
        sized(std::true_type{});
      else
        sized(std::false_type{});
    }
  });
  return dlogits;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Four values for each row, and `scales` behind them.
at::Tensor saved_for(const at::Tensor& logits, long rows, long scales) {
  return at::empty({4 * rows + scales}, logits.options().dtype(at::kFloat));
}

// Calls of few rows whose rows one block of 1024 takes whole, which saves the
// second launch: short rows (50257 bf16: 6.0 against 7.6 us, while one row of
// 128256 is faster split, 7.3 against 9.9 us), and rows that fill half the
// chip without a split (200 of 128256: 12.6 against 15.0 us).
bool takes_whole_rows(long rows, long bytes) {
  return bytes <= (160L << 10) || rows >= 128;
}

// (lp [...] fp32); saved may be undefined.
at::Tensor logprobs_forward(const at::Tensor& logits,
                            const at::Tensor& target, long ignore,
                            const at::Tensor& saved) {
  const c10::DeviceGuard guard(logits.device());
  const Call c = plan(logits, ignore);
  auto lp = at::empty(target.sizes(), logits.options().dtype(at::kFloat));
  if (c.s.rows == 0) return lp;
  float4* keep = saved.defined() ? (float4*)saved.data_ptr() : nullptr;
  STOKE_ELEM_SWITCH(logits.scalar_type(), "token_logprobs", {
    const auto whole_rows = [&](auto threads) {
      hipLaunchKernelGGL((row_stats_kernel<T, threads, true>),
                         dim3((unsigned)c.s.rows), dim3(threads), 0,
                         elem::stream(), (const T*)logits.data_ptr(),
                         target.data_ptr<long>(), nullptr, nullptr, nullptr,
                         c.s, ignore, 1, c.s.vocab, keep,
                         lp.data_ptr<float>());
    };
    if (c.pieces == 1) {
      whole_rows(std::integral_constant<int, kThreads>{});
    } else if (takes_whole_rows(c.s.rows, c.s.vocab * (long)sizeof(T))) {
      whole_rows(std::integral_constant<int, 1024>{});
    } else {
      const Scratch tmp(logits, 0, c);
      launch_stats<T>(logits, target, c, tmp);
      hipLaunchKernelGGL(
          (lp_finish_kernel<std::is_same_v<T, __bf16>>),
          dim3((unsigned)c.s.rows), dim3(64), 0,
          elem::stream(), target.data_ptr<long>(), tmp.stats, tmp.picked,
          keep, lp.data_ptr<float>(), c.s, ignore, c.pieces);
    }
  });
  return lp;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits,
                            const at::Tensor& target, int64_t ignore) {
    auto saved = saved_for(logits, target.numel(), 0);
    auto lp = logprobs_forward(logits, target, ignore, saved);
    ctx->save_for_backward({logits, target, saved});
    ctx->saved_data["ignore"] = ignore;
    return lp;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto v = ctx->get_saved_variables();
    auto d = backward_of(v[0], v[1], (const float4*)v[2].data_ptr(), up[0],
                         Scale{}, ctx->saved_data["ignore"].toInt());
    return elem::once_differentiable({d, at::Tensor(), at::Tensor()});
  }
};

// Behind the saved rows: 1 / (number of tokens).
at::Tensor policy_forward(const at::Tensor& logits, const at::Tensor& target,
                          const at::Tensor& old_lp, const at::Tensor& adv,
                          const at::Tensor& ref_lp, const PolicyArgs& a,
                          long ignore, at::Tensor& saved) {
  const c10::DeviceGuard guard(logits.device());
  const Call c = plan(logits, ignore);
  const auto f32 = logits.options().dtype(at::kFloat);
  saved = saved_for(logits, c.s.rows, 1);
  if (c.s.rows == 0) return at::zeros({}, f32);
  auto loss = at::empty({}, f32);
  const long blocks = (c.s.rows + kThreads - 1) / kThreads;
  const Scratch tmp(logits, 2 * blocks, c);
  STOKE_ELEM_SWITCH(logits.scalar_type(), "policy_loss", {
    launch_stats<T>(logits, target, c, tmp);
    hipLaunchKernelGGL(
        (policy_finish_kernel<std::is_same_v<T, __bf16>>),
        dim3((unsigned)blocks), dim3(kThreads), 0,
        elem::stream(), target.data_ptr<long>(), tmp.stats, tmp.picked,
        old_lp.data_ptr<float>(),
        adv.data_ptr<float>(),
        ref_lp.defined() ? ref_lp.data_ptr<float>() : nullptr,
        (float4*)saved.data_ptr(), tmp.partial, tmp.ticket,
        loss.data_ptr<float>(), saved.data_ptr<float>() + 4 * c.s.rows, c.s,
        ignore, c.pieces, a);
  });
  return loss;
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits,
                            const at::Tensor& target,
                            const at::Tensor& old_lp, const at::Tensor& adv,
                            const std::optional<at::Tensor>& ref_lp,
                            double low, double high, double kl,
                            int64_t ignore) {
    at::Tensor saved;
    auto loss = policy_forward(logits, target, old_lp, adv,
                               ref_lp.value_or(at::Tensor()),
                               PolicyArgs{low, high, kl}, ignore, saved);
    ctx->save_for_backward({logits, target, saved});
    ctx->saved_data["ignore"] = ignore;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto v = ctx->get_saved_variables();
    const float* saved = v[2].data_ptr<float>();
    auto d = backward_of(v[0], v[1], (const float4*)saved, up[0],
                         Scale{saved + 4 * v[1].numel(), 1, 1},
                         ctx->saved_data["ignore"].toInt());
    variable_list out(9);
    out[0] = d;
    return elem::once_differentiable(std::move(out));
  }
};

// Behind the saved rows: the slope of each pair.
variable_list preference_forward(const at::Tensor& logits,
                                 const at::Tensor& target,
                                 const at::Tensor& ref_lp, double beta,
                                 double eps, long ignore, at::Tensor& saved) {
  const c10::DeviceGuard guard(logits.device());
  const Call c = plan(logits, ignore);
  const auto f32 = logits.options().dtype(at::kFloat);
  const long pairs = target.size(0) / 2, seq = target.size(1);
  saved = saved_for(logits, c.s.rows, pairs);
  auto loss = at::empty({}, f32), rewards = at::empty({2 * pairs}, f32);
  if (c.s.rows == 0) {
    loss.fill_(0.6931471805599453);
    rewards.zero_();
    return {loss, rewards};
  }
  const Scratch tmp(logits, pairs, c);
  STOKE_ELEM_SWITCH(logits.scalar_type(), "preference_loss", {
    launch_stats<T>(logits, target, c, tmp);
    hipLaunchKernelGGL(
        (prefer_finish_kernel<std::is_same_v<T, __bf16>>),
        dim3((unsigned)pairs), dim3(kPairThreads), 0,
        elem::stream(), target.data_ptr<long>(), tmp.stats, tmp.picked,
        ref_lp.data_ptr<float>(),
        (float4*)saved.data_ptr(), tmp.partial, tmp.ticket,
        loss.data_ptr<float>(), rewards.data_ptr<float>(),
        saved.data_ptr<float>() + 4 * c.s.rows, c.s, ignore, c.pieces, seq,
        beta, eps);
  });
  return {loss, rewards};
}

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits,
                               const at::Tensor& target,
                               const at::Tensor& ref_lp, double beta,
                               double eps, int64_t ignore) {
    at::Tensor saved;
    auto out = preference_forward(logits, target, ref_lp, beta, eps, ignore,
                                  saved);
    ctx->save_for_backward({logits, target, saved});
    ctx->mark_non_differentiable({out[1]});
    ctx->saved_data["ignore"] = ignore;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const auto v = ctx->get_saved_variables();
    const float* saved = v[2].data_ptr<float>();
    const long pairs = v[1].size(0) / 2;
    auto d = backward_of(v[0], v[1], (const float4*)saved, up[0],
                         Scale{saved + 4 * v[1].numel(),
                               std::max<long>(1, v[1].size(1)), pairs},
                         ctx->saved_data["ignore"].toInt());
    variable_list out(6);
    out[0] = d;
    return elem::once_differentiable(std::move(out));
  }
};

}  // namespace

// The entry points check their arguments and have gradients for the logits.
at::Tensor token_logprobs(at::Tensor logits, at::Tensor target,
                          int64_t ignore) {
  elem::refuse_tangents("token_logprobs", logits);
  check(logits, target, "token_logprobs");
  const auto x = rows_of(logits), t = target.contiguous();
  if (!wants_grad(logits)) return logprobs_forward(x, t, ignore, at::Tensor());
  return TokenLogprobs::apply(x, t, ignore);
}

at::Tensor policy_loss(at::Tensor logits, at::Tensor target,
                       at::Tensor old_lp, at::Tensor adv,
                       std::optional<at::Tensor> ref_lp, double clip_low,
                       double clip_high, double kl, int64_t ignore) {
  elem::refuse_tangents("fused_policy_loss", logits, old_lp, adv, ref_lp);
  check(logits, target, "fused_policy_loss");
  TORCH_CHECK_VALUE(
      clip_low >= 0 && clip_low <= 1 && clip_high >= 0 && kl >= 0,
      "Stoke -- fused_policy_loss takes 0 <= clip_low <= 1, clip_high >= 0 "
      "and kl_coef >= 0, got ", clip_low, ", ", clip_high, ", ", kl);
  TORCH_CHECK_VALUE(kl == 0 || ref_lp, "Stoke -- kl_coef needs ref_logprobs");
  const auto x = rows_of(logits), t = target.contiguous();
  const auto old_rows = per_token(old_lp, target, "old_logprobs");
  const auto adv_rows = per_token(adv, target, "advantages");
  std::optional<at::Tensor> ref;
  if (kl != 0) ref = per_token(*ref_lp, target, "ref_logprobs");
  if (wants_grad(logits))
    return PolicyLoss::apply(x, t, old_rows, adv_rows, ref, 1. - clip_low,
                             1. + clip_high, kl, ignore);
  at::Tensor saved;
  return policy_forward(x, t, old_rows, adv_rows, ref.value_or(at::Tensor()),
                        PolicyArgs{1. - clip_low, 1. + clip_high, kl},
                        ignore, saved);
}

// (loss, rewards)
std::vector<at::Tensor> preference_loss(at::Tensor logits, at::Tensor target,
                                        at::Tensor ref_lp, double beta,
                                        double eps, int64_t ignore) {
  elem::refuse_tangents("fused_preference_loss", logits, ref_lp);
  check(logits, target, "fused_preference_loss");
  TORCH_CHECK_VALUE(
      logits.dim() == 3 && logits.size(0) > 0 && logits.size(0) % 2 == 0,
      "Stoke -- fused_preference_loss takes logits [2P, S, V] (chosen, then "
      "rejected), got ", logits.sizes());
  TORCH_CHECK_VALUE(beta > 0 && eps >= 0 && eps <= 0.5,
                    "Stoke -- fused_preference_loss takes beta > 0 and "
                    "0 <= label_smoothing <= 0.5, got ", beta, ", ", eps);
  const auto x = rows_of(logits), t = target.contiguous();
  const auto ref = per_token(ref_lp, target, "ref_logprobs");
  if (wants_grad(logits))
    return PreferenceLoss::apply(x, t, ref, beta, eps, ignore);
  at::Tensor saved;
  return preference_forward(x, t, ref, beta, eps, ignore, saved);
}
