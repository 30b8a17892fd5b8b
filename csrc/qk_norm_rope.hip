// Per-head RMS norm of queries and keys and the rotary rotation in one pass.
//
// For a head's row x of D values, weight w and angle row (c, s):
//   r = 1 / sqrt(mean(x^2) + eps),  n = x r w
//   pair (a, b):  y_a = n_a c - n_b s,  y_b = n_b c + n_a s
// The first R = 2 * half values are rotated, pairs (2i, 2i+1) or
// (i, i + half); the rest only normalised.  Pair p of token (b, s) takes row
// positions[axis(p), b, s] of the tables, axis(p) from the sections.
// Backward, with dn the rotation of dy by the opposite angle and g = dn w:
//   dx = r (g - x r^2 mean(g x)),   dw = sum over rows of dn x r
// r is computed again: x is read anyway.
//
// A position outside the tables reads nothing and gives NaN.

#include <hip/hip_runtime.h>

#include "elem.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxAxes = 4;
constexpr int kMaxDim = 1024;

// Queries or keys.
struct Side {
  const void* x;
  const void* dy;  // backward; contiguous
  void* y;         // forward output or dx; contiguous [B, S, H, D]
  const void* w;   // null: ones
  long sb, ss, sh;  // strides of x in elements
  int heads;
};

struct Args {
  Side side[2];
  const float *cosines, *sines;
  const long* pos;  // [axes, tokens], null: the index in the sequence
  long tokens, seq, table;
  int dim, half, axes;
  int ends[kMaxAxes];  // section ends in pairs
  bool w_fp32, interleaved;
  float eps;
};

template <typename T>
__device__ __forceinline__ float weight(const Side& s, bool fp32, int e) {
  if (!s.w) return 1.f;
  return fp32 ? ((const float*)s.w)[e] : (float)((const T*)s.w)[e];
}

// Cosine and sine of pair p at a token.
__device__ __forceinline__ float2 angle(const Args& a, long token, int p) {
  int axis = 0;
  while (axis + 1 < a.axes && p >= a.ends[axis]) ++axis;
  const long at = a.pos ? a.pos[axis * a.tokens + token] : token % a.seq;
  if (at < 0 || at >= a.table) {
    const float nan = __uint_as_float(0x7fc00000);
    return make_float2(nan, nan);
  }
  return make_float2(a.cosines[at * a.half + p], a.sines[at * a.half + p]);
}

__device__ __forceinline__ float wave_sum(float v) {
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const Args& a, const Side& s,
                                           long row) {
  const long token = row / s.heads;
  return (const T*)s.x + (token / a.seq) * s.sb + (token % a.seq) * s.ss +
         (row % s.heads) * s.sh;
}

// The other value of e's pair.
__device__ __forceinline__ int partner(const Args& a, int e) {
  if (a.interleaved) return e ^ 1;
  return e < a.half ? e + a.half : e - a.half;
}
__device__ __forceinline__ int pair_of(const Args& a, int e) {
  if (a.interleaved) return e >> 1;
  return e < a.half ? e : e - a.half;
}
__device__ __forceinline__ bool is_first(const Args& a, int e) {
  return a.interleaved ? (e & 1) == 0 : e < a.half;
}

// A wave for each row, the row in shared memory: any dim, stride and
// alignment.
template <typename T>
__global__ __launch_bounds__(kThreads) void fwd_any_kernel(Args a,
                                                           int q_blocks) {
  extern __shared__ float rows[];
  const int which = (int)blockIdx.x >= q_blocks;
  const Side& s = a.side[which];
  const long block = blockIdx.x - (which ? q_blocks : 0);
  const long blocks = which ? gridDim.x - q_blocks : q_blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float* mine = rows + wave * a.dim;
  const long total = a.tokens * s.heads;
  for (long base = block * kWaves; base < total; base += blocks * kWaves) {
    const long row = base + wave;
    const bool live = row < total;
    float r = 0.f;
    if (live) {
      const T* x = row_of<T>(a, s, row);
      float sum = 0.f;
      for (int e = lane; e < a.dim; e += 64) {
        const float v = (float)x[e];
        sum += v * v;
        mine[e] = v * weight<T>(s, a.w_fp32, e);
      }
      r = 1.f / sqrtf(wave_sum(sum) / (float)a.dim + a.eps);
    }
    __syncthreads();
    if (live) {
      T* y = (T*)s.y + row * a.dim;
      for (int e = lane; e < a.dim; e += 64) {
        float v = mine[e] * r;
        if (e < 2 * a.half) {
          const float2 cs = angle(a, row / s.heads, pair_of(a, e));
          const float o = mine[partner(a, e)] * r;
          v = v * cs.x + (is_first(a, e) ? -o : o) * cs.y;
        }
        y[e] = (T)v;
      }
    }
    __syncthreads();
  }
}

// dw of a block's rows goes to partial[block]; the blocks of the queries
// come first.
template <typename T>
__global__ __launch_bounds__(kThreads) void bwd_any_kernel(
    Args a, int q_blocks, float* __restrict__ partial) {
  extern __shared__ float rows[];
  const int which = (int)blockIdx.x >= q_blocks;
  const Side& s = a.side[which];
  const long block = blockIdx.x - (which ? q_blocks : 0);
  const long blocks = which ? gridDim.x - q_blocks : q_blocks;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float* mine = rows + wave * a.dim;
  float* dw = rows + (kWaves + wave) * a.dim;
  for (int e = lane; e < a.dim; e += 64) dw[e] = 0.f;
  const long total = a.tokens * s.heads;
  for (long base = block * kWaves; base < total; base += blocks * kWaves) {
    const long row = base + wave;
    const bool live = row < total;
    const T* dy = (const T*)s.dy + row * a.dim;
    if (live)
      for (int e = lane; e < a.dim; e += 64) mine[e] = (float)dy[e];
    __syncthreads();
    if (live) {
      const T* x = row_of<T>(a, s, row);
      T* dx = (T*)s.y + row * a.dim;
      float dn[kMaxDim / 64];
      float sum = 0.f, dot = 0.f;
      #pragma unroll
      for (int i = 0; i < kMaxDim / 64; ++i) {
        const int e = lane + 64 * i;
        if (e >= a.dim) continue;
        float v = mine[e];
        if (e < 2 * a.half) {
          const float2 cs = angle(a, row / s.heads, pair_of(a, e));
          const float o = mine[partner(a, e)];
          v = v * cs.x + (is_first(a, e) ? o : -o) * cs.y;
        }
        dn[i] = v;
        const float xv = (float)x[e];
        sum += xv * xv;
        dot += v * weight<T>(s, a.w_fp32, e) * xv;
      }
      const float r = 1.f / sqrtf(wave_sum(sum) / (float)a.dim + a.eps);
      const float k = wave_sum(dot) / (float)a.dim * r * r;
      #pragma unroll
      for (int i = 0; i < kMaxDim / 64; ++i) {
        const int e = lane + 64 * i;
        if (e >= a.dim) continue;
        const float xv = (float)x[e];
        dx[e] = (T)(r * (dn[i] * weight<T>(s, a.w_fp32, e) - xv * k));
        dw[e] += dn[i] * xv * r;
      }
    }
    __syncthreads();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.dim; e += kThreads) {
    float v = 0.f;
    for (int w = 0; w < kWaves; ++w) v += rows[(kWaves + w) * a.dim + e];
    partial[(long)blockIdx.x * a.dim + e] = v;
  }
}

// dw of one side from the blocks' sums, added in their order.
template <typename T>
__global__ __launch_bounds__(kThreads) void dw_kernel(
    const float* __restrict__ partial, void* dwq, void* dwk, int q_blocks,
    int blocks, int dim, bool fp32) {
  __shared__ double sums[kThreads];
  const int which = blockIdx.y;
  const int col = blockIdx.x * 16 + (threadIdx.x & 15);
  const int first = which ? q_blocks : 0, last = which ? blocks : q_blocks;
  double v = 0.;
  if (col < dim)
    for (int b = first + (threadIdx.x >> 4); b < last; b += kThreads / 16)
      v += (double)partial[(long)b * dim + col];
  sums[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x >= 16 || col >= dim) return;
  for (int i = 1; i < kThreads / 16; ++i) v += sums[threadIdx.x + 16 * i];
  void* out = which ? dwk : dwq;
  if (!out) return;
  if (fp32) ((float*)out)[col] = (float)v;
  else ((T*)out)[col] = (T)(float)v;
}

void check_side(const at::Tensor& x, const at::Tensor& like,
                const c10::optional<at::Tensor>& w, const char* what) {
  TORCH_CHECK(x.is_cuda() && x.device() == like.device() && x.dim() == 4 &&
                  x.scalar_type() == like.scalar_type() &&
                  x.size(0) == like.size(0) && x.size(1) == like.size(1) &&
                  x.size(3) == like.size(3) &&
                  (x.size(3) <= 1 || x.stride(3) == 1),
              "qk_norm_rope: ", what,
              " must be [B, S, H, D] with a unit last stride");
  TORCH_CHECK(!w || (w->device() == x.device() && w->dim() == 1 &&
                     w->size(0) == x.size(3) && w->is_contiguous() &&
                     (w->scalar_type() == at::kFloat ||
                      w->scalar_type() == x.scalar_type())),
              "qk_norm_rope: contiguous weights [D] in fp32 or the heads' "
              "dtype required");
}

void fill_side(Side& s, const at::Tensor& x,
               const c10::optional<at::Tensor>& w, at::Tensor& y) {
  s.x = x.data_ptr();
  s.dy = nullptr;
  s.y = y.data_ptr();
  s.w = w ? w->data_ptr() : nullptr;
  s.sb = x.stride(0);
  s.ss = x.stride(1);
  s.sh = x.stride(2);
  s.heads = (int)x.size(2);
}

Args make_args(const at::Tensor& q, const at::Tensor& k,
               const c10::optional<at::Tensor>& wq,
               const c10::optional<at::Tensor>& wk, const at::Tensor& cosines,
               const at::Tensor& sines, const c10::optional<at::Tensor>& pos,
               const std::vector<int64_t>& sections, double eps,
               bool interleaved, at::Tensor& yq, at::Tensor& yk) {
  check_side(q, q, wq, "q");
  check_side(k, q, wk, "k");
  TORCH_CHECK(!wq || !wk || wq->scalar_type() == wk->scalar_type(),
              "qk_norm_rope: weights of one dtype required");
  Args a;
  a.tokens = q.size(0) * q.size(1);
  a.seq = std::max<long>(1, q.size(1));
  a.dim = (int)q.size(3);
  TORCH_CHECK(a.dim >= 1 && a.dim <= kMaxDim,
              "qk_norm_rope: head dim of 1 to ", kMaxDim, " required");
  TORCH_CHECK(cosines.device() == q.device() && cosines.dim() == 2 &&
                  cosines.scalar_type() == at::kFloat &&
                  cosines.is_contiguous() && sines.device() == q.device() &&
                  sines.sizes() == cosines.sizes() &&
                  sines.scalar_type() == at::kFloat && sines.is_contiguous() &&
                  2 * cosines.size(1) <= a.dim,
              "qk_norm_rope: contiguous fp32 tables [P, <= D / 2] required");
  a.table = cosines.size(0);
  a.half = (int)cosines.size(1);
  a.cosines = cosines.data_ptr<float>();
  a.sines = sines.data_ptr<float>();
  a.axes = std::max<int>(1, (int)sections.size());
  TORCH_CHECK(a.axes <= kMaxAxes, "qk_norm_rope: at most ", kMaxAxes, " axes");
  int end = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    if (i < (int)sections.size()) end += (int)sections[i];
    else end = a.half;
    a.ends[i] = end;
  }
  a.pos = nullptr;
  if (pos) {
    TORCH_CHECK(pos->device() == q.device() && pos->is_contiguous() &&
                    pos->scalar_type() == at::kLong &&
                    pos->numel() == a.axes * a.tokens,
                "qk_norm_rope: contiguous int64 positions [axes, B, S] "
                "required");
    a.pos = pos->data_ptr<long>();
  } else {
    TORCH_CHECK(a.axes == 1 && a.table >= a.seq,
                "qk_norm_rope: tables shorter than the sequence");
  }
  a.w_fp32 = (wq && wq->scalar_type() == at::kFloat) ||
             (wk && wk->scalar_type() == at::kFloat);
  a.interleaved = interleaved;
  a.eps = (float)eps;
  fill_side(a.side[0], q, wq, yq);
  fill_side(a.side[1], k, wk, yk);
  return a;
}

// Blocks of the queries and of the keys, by their share of the rows.
void share(const Args& a, long most, int& q_blocks, int& blocks) {
  const long rq = a.tokens * a.side[0].heads, rk = a.tokens * a.side[1].heads;
  auto part = [&](long rows) {
    const long all = std::max<long>(1, rq + rk);
    const long want = std::max<long>(1, most * rows / all);
    return rows == 0 ? 0L : std::min<long>(want, (rows + kWaves - 1) / kWaves);
  };
  q_blocks = (int)part(rq);
  blocks = q_blocks + (int)part(rk);
}

}  // namespace

std::vector<at::Tensor> qk_norm_rope_fwd(
    at::Tensor q, at::Tensor k, c10::optional<at::Tensor> wq,
    c10::optional<at::Tensor> wk, at::Tensor cosines, at::Tensor sines,
    c10::optional<at::Tensor> pos, std::vector<int64_t> sections, double eps,
    bool interleaved) {
  const c10::DeviceGuard guard(q.device());
  auto yq = at::empty(q.sizes(), q.options());
  auto yk = at::empty(k.sizes(), k.options());
  const Args a = make_args(q, k, wq, wk, cosines, sines, pos, sections, eps,
                           interleaved, yq, yk);
  int q_blocks, blocks;
  share(a, 65536, q_blocks, blocks);
  STOKE_ELEM_SWITCH(q.scalar_type(), "qk_norm_rope", {
    if (blocks > 0)
      hipLaunchKernelGGL((fwd_any_kernel<T>), dim3((unsigned)blocks),
                         dim3(kThreads), kWaves * a.dim * sizeof(float),
                         elem::stream(), a, q_blocks);
  });
  return {yq, yk};
}

// (dq, dk, dwq, dwk); the last two empty where there is no weight.
std::vector<at::Tensor> qk_norm_rope_bwd(
    at::Tensor dyq, at::Tensor dyk, at::Tensor q, at::Tensor k,
    c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk,
    at::Tensor cosines, at::Tensor sines, c10::optional<at::Tensor> pos,
    std::vector<int64_t> sections, double eps, bool interleaved) {
  const c10::DeviceGuard guard(q.device());
  auto dq = at::empty(q.sizes(), q.options());
  auto dk = at::empty(k.sizes(), k.options());
  Args a = make_args(q, k, wq, wk, cosines, sines, pos, sections, eps,
                     interleaved, dq, dk);
  TORCH_CHECK(dyq.sizes() == q.sizes() && dyk.sizes() == k.sizes() &&
                  dyq.scalar_type() == q.scalar_type() &&
                  dyk.scalar_type() == q.scalar_type() &&
                  dyq.is_contiguous() && dyk.is_contiguous(),
              "qk_norm_rope: contiguous gradients of the outputs' shape");
  a.side[0].dy = dyq.data_ptr();
  a.side[1].dy = dyk.data_ptr();
  int q_blocks, blocks;
  share(a, 2048, q_blocks, blocks);
  auto partial = at::empty({blocks, a.dim}, q.options().dtype(at::kFloat));
  at::Tensor dwq, dwk;
  if (wq) dwq = at::empty(wq->sizes(), wq->options());
  if (wk) dwk = at::empty(wk->sizes(), wk->options());
  STOKE_ELEM_SWITCH(q.scalar_type(), "qk_norm_rope", {
    if (blocks > 0)
      hipLaunchKernelGGL((bwd_any_kernel<T>), dim3((unsigned)blocks),
                         dim3(kThreads), 2 * kWaves * a.dim * sizeof(float),
                         elem::stream(), a, q_blocks,
                         partial.data_ptr<float>());
    if (wq || wk)
      hipLaunchKernelGGL((dw_kernel<T>), dim3((a.dim + 15) / 16, 2),
                         dim3(kThreads), 0, elem::stream(),
                         partial.data_ptr<float>(),
                         wq ? dwq.data_ptr() : nullptr,
                         wk ? dwk.data_ptr() : nullptr, q_blocks, blocks,
                         a.dim, a.w_fp32);
  });
  return {dq, dk, dwq, dwk};
}
