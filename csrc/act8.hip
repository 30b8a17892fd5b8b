// Activations held in 8 bits: 32 values share a power of two.
//
// A block of 32 consecutive values of the flattened tensor keeps one byte
// E and 32 signed bytes q with  value = q * 2^(E - 127),  |q| <= 127.
// E is the least exponent from 1 up at which the block's largest value still
// rounds into 127, so a value is off by at most half of 2^(E-127), that is
// 1/127 of the block's largest (2^-127 where that is below 2^-120 and E stays
// at 1).  Scaling by a power of two is exact: the one rounding is the
// conversion to a whole number (half to even).  E = 255
// marks a block with an infinity or NaN; all of it reads back as NaN, so an
// overflow in the forward pass still reaches the gradients.

#include <hip/hip_runtime.h>

#include "elem.h"

namespace {

// E for a block whose largest magnitude has these fp32 bits.
__device__ __forceinline__ unsigned block_exponent(unsigned top) {
  const int be = (int)(top >> 23);
  if (be == 255) return 255;
  // top * 2^(127-E) lies in [64, 128); from 127.5 up it rounds to 128
  const int e = be - 6 + ((top & 0x7fffff) >= 0x7f0000 ? 1 : 0);
  return (unsigned)max(e, 1);
}

__device__ __forceinline__ float pow2_bits(unsigned biased) {
  return __uint_as_float(biased << 23);
}

__device__ __forceinline__ int quantize(float x, unsigned e) {
  return e == 255 ? 0 : (int)rintf(x * pow2_bits(254 - e));
}

template <typename T>
__device__ __forceinline__ float largest() {
  return sizeof(T) == 4 ? 3.402823466e38f : 3.389531390e38f;
}
template <>
__device__ __forceinline__ float largest<_Float16>() { return 65504.f; }

// q * 2^(E-127).  The value next to the type's largest rounds up to a power
// of two past its range: it comes back as the largest.
template <typename T>
__device__ __forceinline__ float restored(int q, unsigned e) {
  const float v = (float)q * pow2_bits(e);
  if (e == 255) return __uint_as_float(0x7fc00000);
  return fminf(fmaxf(v, -largest<T>()), largest<T>());
}

// The 32 lanes of a half wave hold one block, a value each.
__device__ __forceinline__ unsigned half_wave_max(unsigned v) {
  #pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    v = max(v, (unsigned)__shfl_xor((int)v, off));
  return v;
}

constexpr int kThreads = 256;
constexpr int kRun = 8;  // values of a thread: 4 threads hold a block of 32

template <typename T>
using Run = elem::vec<T, kRun>;
using Bytes = elem::vec<signed char, kRun>;

// Largest over the 4 lanes of a quad, which hold one block.
__device__ __forceinline__ unsigned quad_max(unsigned v) {
  v = max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 15, 15, true));
  return max(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 15, 15,
                                                   true));
}

// A quad's block: its exponent, and the thread's 8 values in 8 bits.
__device__ __forceinline__ unsigned pack_run(const float (&v)[kRun],
                                             Bytes& q) {
  unsigned top = 0;
  #pragma unroll
  for (int e = 0; e < kRun; ++e)
    top = max(top, __float_as_uint(v[e]) & 0x7fffffff);
  const unsigned exp = block_exponent(quad_max(top));
  // adding 1.5 * 2^23 leaves the whole number, half to even, in the low
  // bits: its lowest byte is the signed byte
  const float inv = pow2_bits(254 - exp);
  #pragma unroll
  for (int e = 0; e < kRun; ++e)
    q[e] = (signed char)__float_as_uint(
        __builtin_fmaf(v[e], inv, 12582912.f));
  if (exp == 255) q = (Bytes)(signed char)0;
  return exp;
}

template <typename T>
__device__ __forceinline__ void unpack_run(const Bytes q, unsigned exp,
                                           float (&v)[kRun]) {
  const float step = pow2_bits(exp);  // inf for 255: 0 * inf = NaN
  #pragma unroll
  for (int e = 0; e < kRun; ++e) v[e] = (float)q[e] * step;
  // only the topmost exponents can pass the largest value
  constexpr unsigned kTop = sizeof(T) == 2 && std::is_same_v<T, _Float16>
                                ? 127 + 10 : 127 + 122;
  if (exp >= kTop) {
    #pragma unroll
    for (int e = 0; e < kRun; ++e) v[e] = restored<T>(q[e], exp);
  }
}

template <bool NT, typename T>
__device__ __forceinline__ void load_run(const T* __restrict__ p, long i,
                                         float (&v)[kRun]) {
  const Run<T> w = elem::load<NT, kRun>(p + i);
  #pragma unroll
  for (int e = 0; e < kRun; ++e) v[e] = (float)w[e];
}

template <bool NT, typename T>
__device__ __forceinline__ void store_run(T* __restrict__ p, long i,
                                          const float (&v)[kRun]) {
  Run<T> w;
  #pragma unroll
  for (int e = 0; e < kRun; ++e) w[e] = (T)v[e];
  elem::store<NT, kRun>(p + i, w);
}

__device__ __forceinline__ float sigmoid(float a) {
  return 1.f / (1.f + __expf(-a));
}

// y = silu(g) u
__device__ __forceinline__ float swiglu(float a, float b) {
  return a / (1.f + __expf(-a)) * b;
}

// dg = dy u s (1 + g (1 - s)),  du = dy g s,  s = 1 / (1 + e^-g)
__device__ __forceinline__ void swiglu_grad(float d, float a, float b,
                                            float& da, float& db) {
  const float s = sigmoid(a);
  da = d * b * s * (1.f + a * (1.f - s));
  db = d * a * s;
}

// Every kernel takes 8 values a thread, with 16-byte (or two 16-byte)
// accesses, for the whole blocks of 32, and one value a thread for the last,
// partial block, which begins at `first`.
// NT: tensors over elem::kCached are read past the caches (and, in the
// backward, written).  What the forward writes is read by the next product:
// it goes through them.
//
// All are bound by memory.  Two runs of 134M bf16 values packed in 68 and 74 us
// and unpacked in 59 and 64 us (407 MB each, 5.5 to 6.9 TB/s); SwiGLU at 8192 x
// 14336 took 156 and 168 us forward (947 MB, 5.6 to 6.1 TB/s; 109 us and 705 MB
// without a backward to come) and 154 and 166 us backward.  Through the caches
// they took 7 to 13 % longer.  One value a thread took 389 and 659 us for both
// directions, against 133 and 309 us.
template <typename T, bool NT>
__global__ __launch_bounds__(kThreads) void pack_kernel(
    const T* __restrict__ x, signed char* __restrict__ q,
    unsigned char* __restrict__ scale, long n, long first) {
  const long step = (long)gridDim.x * kThreads;
  const long me = (long)blockIdx.x * kThreads + threadIdx.x;
  for (long i = me * kRun; i < first; i += step * kRun) {
    float v[kRun];
    Bytes b;
    load_run<NT>(x, i, v);
    const unsigned e = pack_run(v, b);
    *(Bytes*)(q + i) = b;
    if ((threadIdx.x & 3) == 0) scale[i >> 5] = (unsigned char)e;
  }
  const long n32 = (n + 31) / 32 * 32;
  for (long i = first + me; i < n32; i += step) {
    const float v = i < n ? (float)x[i] : 0.f;
    const unsigned e =
        block_exponent(half_wave_max(__float_as_uint(v) & 0x7fffffff));
    if (i < n) q[i] = (signed char)quantize(v, e);
    if ((threadIdx.x & 31) == 0) scale[i >> 5] = (unsigned char)e;
  }
}

template <typename T, bool NT>
__global__ __launch_bounds__(kThreads) void unpack_kernel(
    const signed char* __restrict__ q,
    const unsigned char* __restrict__ scale, T* __restrict__ x, long n,
    long first) {
  const long step = (long)gridDim.x * kThreads;
  const long me = (long)blockIdx.x * kThreads + threadIdx.x;
  for (long i = me * kRun; i < first; i += step * kRun) {
    float v[kRun];
    unpack_run<T>(elem::load<NT, kRun>(q + i), scale[i >> 5], v);
    store_run<false>(x, i, v);
  }
  for (long i = first + me; i < n; i += step)
    x[i] = (T)restored<T>(q[i], scale[i >> 5]);
}

// Where the values of g and u lie: rows of `cols` values `g` and `u` elements
// apart, as the halves of one projection are; contiguous where cols is 0.
// Rows hold whole runs, and there are fewer than 2^31 values.
struct Rows {
  unsigned cols;
  long g, u;
};

// y = silu(g) * u from the values as they come; with KEEP g and u stay in 8
// bits.  Without a backward to come nothing else is computed or written.
template <typename T, bool NT, bool KEEP>
__global__ __launch_bounds__(kThreads) void swiglu8_fwd_kernel(
    const T* __restrict__ g, const T* __restrict__ u, T* __restrict__ y,
    signed char* __restrict__ qg, signed char* __restrict__ qu,
    unsigned char* __restrict__ sg, unsigned char* __restrict__ su, long n,
    long first, Rows rows) {
  const long step = (long)gridDim.x * kThreads;
  const long me = (long)blockIdx.x * kThreads + threadIdx.x;
  const auto place = [&](long i, long& ig, long& iu) {
    ig = iu = i;
    if (!rows.cols) return;
    const unsigned row = (unsigned)i / rows.cols;
    const long col = (unsigned)i - row * rows.cols;
    ig = row * rows.g + col;
    iu = row * rows.u + col;
  };
  for (long i = me * kRun; i < first; i += step * kRun) {
    float a[kRun], b[kRun], o[kRun];
    long ig, iu;
    place(i, ig, iu);
    load_run<NT>(g, ig, a);
    load_run<NT>(u, iu, b);
    #pragma unroll
    for (int e = 0; e < kRun; ++e) o[e] = swiglu(a[e], b[e]);
    store_run<false>(y, i, o);
    if (!KEEP) continue;
    Bytes qa, qb;
    const unsigned ea = pack_run(a, qa), eb = pack_run(b, qb);
    *(Bytes*)(qg + i) = qa;
    *(Bytes*)(qu + i) = qb;
    if ((threadIdx.x & 3) == 0) {
      sg[i >> 5] = (unsigned char)ea;
      su[i >> 5] = (unsigned char)eb;
    }
  }
  const long n32 = (n + 31) / 32 * 32;
  for (long i = first + me; i < n32; i += step) {
    long ig, iu;
    place(i, ig, iu);
    const float a = i < n ? (float)g[ig] : 0.f;
    const float b = i < n ? (float)u[iu] : 0.f;
    if (i < n) y[i] = (T)swiglu(a, b);
    if (!KEEP) continue;
    const unsigned eg =
        block_exponent(half_wave_max(__float_as_uint(a) & 0x7fffffff));
    const unsigned eu =
        block_exponent(half_wave_max(__float_as_uint(b) & 0x7fffffff));
    if (i < n) {
      qg[i] = (signed char)quantize(a, eg);
      qu[i] = (signed char)quantize(b, eu);
    }
    if ((threadIdx.x & 31) == 0) {
      sg[i >> 5] = (unsigned char)eg;
      su[i >> 5] = (unsigned char)eu;
    }
  }
}

template <typename T, bool NT>
__global__ __launch_bounds__(kThreads) void swiglu8_bwd_kernel(
    const T* __restrict__ dy, const signed char* __restrict__ qg,
    const signed char* __restrict__ qu, const unsigned char* __restrict__ sg,
    const unsigned char* __restrict__ su, T* __restrict__ dg,
    T* __restrict__ du, long n, long first) {
  const long step = (long)gridDim.x * kThreads;
  const long me = (long)blockIdx.x * kThreads + threadIdx.x;
  for (long i = me * kRun; i < first; i += step * kRun) {
    float d[kRun], a[kRun], b[kRun], da[kRun], db[kRun];
    load_run<NT>(dy, i, d);
    unpack_run<T>(elem::load<NT, kRun>(qg + i), sg[i >> 5], a);
    unpack_run<T>(elem::load<NT, kRun>(qu + i), su[i >> 5], b);
    #pragma unroll
    for (int e = 0; e < kRun; ++e)
      swiglu_grad(d[e], a[e], b[e], da[e], db[e]);
    store_run<NT>(dg, i, da);
    store_run<NT>(du, i, db);
  }
  for (long i = first + me; i < n; i += step) {
    float da, db;
    swiglu_grad((float)dy[i], restored<T>(qg[i], sg[i >> 5]),
                restored<T>(qu[i], su[i >> 5]), da, db);
    dg[i] = (T)da;
    du[i] = (T)db;
  }
}

// Where the last, partial block begins.
inline long first_of(long n) { return n / 32 * 32; }

inline dim3 grid_for(long n, long first, int runs = 1) {
  const long threads = std::max(first / kRun / runs, n - first);
  return dim3((unsigned)std::min<long>((threads + kThreads - 1) / kThreads,
                                       1 << 20));
}

// Calls f with whether the accesses go past the caches as a constant.
template <typename F>
void with_caching(long bytes, F f) {
  if (bytes > elem::kCached) f(std::true_type{});
  else f(std::false_type{});
}

// Pieces of the byte buffer that holds g and u: both values, then both
// exponents; each piece starts on 16 bytes.
struct Held {
  signed char *qg, *qu;
  unsigned char *sg, *su;
  long bytes;
  Held(void* base, long n) {
    const long q = (n + 15) / 16 * 16;
    const long s = ((n + 31) / 32 + 15) / 16 * 16;
    char* p = (char*)base;
    qg = (signed char*)p;
    qu = (signed char*)(p + q);
    sg = (unsigned char*)(p + 2 * q);
    su = (unsigned char*)(p + 2 * q + s);
    bytes = 2 * q + 2 * s;
  }
};

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The distance of x's rows where it is rows of contiguous values at one
// positive distance from another, else 0.
long row_step(const at::Tensor& x) {
  const long d = x.dim();
  if (d < 2 || x.stride(d - 1) != 1) return 0;
  long step = 0, next = 0;
  for (long i = d - 2; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (x.stride(i) <= 0 || (step && x.stride(i) != next)) return 0;
    if (!step) step = x.stride(i);
    next = x.stride(i) * x.size(i);
  }
  return step;
}

// held: what the backward needs, null where there is none.
at::Tensor swiglu8_forward(const at::Tensor& gate, const at::Tensor& up,
                           at::Tensor* held) {
  const c10::DeviceGuard guard(gate.device());
  const long n = gate.numel();
  Rows rows{0, 0, 0};
  if (!gate.is_contiguous() || !up.is_contiguous()) {
    rows = Rows{(unsigned)gate.size(-1), row_step(gate), row_step(up)};
    if (n >= (1L << 31) || gate.size(-1) % kRun || !rows.g || !rows.u)
      rows.cols = 0;
  }
  const at::Tensor g = rows.cols ? gate : gate.contiguous();
  const at::Tensor u = rows.cols ? up : up.contiguous();
  auto y = at::empty(g.sizes(), g.options());
  if (held)
    *held = at::empty({Held(nullptr, n).bytes}, g.options().dtype(at::kByte));
  if (n == 0) return y;
  const Held h(held ? held->data_ptr() : nullptr, n);
  STOKE_ELEM_SWITCH(g.scalar_type(), "swiglu8", {
    const long first = first_of(n);
    with_caching(n * (long)sizeof(T), [&](auto nt) {
      const auto launch = [&](auto keep) {
        hipLaunchKernelGGL((swiglu8_fwd_kernel<T, nt, keep>),
                           grid_for(n, first), dim3(kThreads), 0,
                           elem::stream(), (const T*)g.data_ptr(),
                           (const T*)u.data_ptr(), (T*)y.data_ptr(), h.qg,
                           h.qu, h.sg, h.su, n, first, rows);
      };
      if (held) launch(std::true_type{});
      else launch(std::false_type{});
    });
  });
  return y;
}

variable_list swiglu8_backward(const at::Tensor& dy, const at::Tensor& held) {
  const c10::DeviceGuard guard(dy.device());
  const long n = dy.numel();
  auto dg = at::empty(dy.sizes(), dy.options());
  auto du = at::empty(dy.sizes(), dy.options());
  if (n == 0) return {dg, du};
  const Held h(held.data_ptr(), n);
  STOKE_ELEM_SWITCH(dy.scalar_type(), "swiglu8", {
    const long first = first_of(n);
    with_caching(n * (long)sizeof(T), [&](auto nt) {
      hipLaunchKernelGGL((swiglu8_bwd_kernel<T, nt>), grid_for(n, first),
                         dim3(kThreads), 0, elem::stream(),
                         (const T*)dy.data_ptr(), h.qg, h.qu, h.sg, h.su,
                         (T*)dg.data_ptr(), (T*)du.data_ptr(), n, first);
    });
  });
  return {dg, du};
}

struct SwiGLU8 : torch::autograd::Function<SwiGLU8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& g,
                            const at::Tensor& u) {
    at::Tensor held;
    auto y = swiglu8_forward(g, u, &held);
    ctx->save_for_backward({held});
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    return elem::once_differentiable(swiglu8_backward(
        dy[0].contiguous(), ctx->get_saved_variables()[0]));
  }
};

}  // namespace

// (values, exponents)
std::vector<at::Tensor> act8_pack(at::Tensor act) {
  TORCH_CHECK_VALUE(act.is_cuda() && (act.scalar_type() == at::kBFloat16 ||
                                      act.scalar_type() == at::kHalf ||
                                      act.scalar_type() == at::kFloat),
                    "Stoke -- compress_activation takes bf16, fp16 or fp32, "
                    "got ", act.scalar_type());
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(act.device());
  const at::Tensor x = act.contiguous();
  const long n = x.numel();
  auto q = at::empty(x.sizes(), x.options().dtype(at::kChar));
  auto scale = at::empty({(n + 31) / 32}, x.options().dtype(at::kByte));
  STOKE_ELEM_SWITCH(x.scalar_type(), "act8_pack", {
    const long first = first_of(n);
    // past the caches a thread takes two runs: 134M values in 6 % less time
    if (n > 0)
      with_caching(n * (long)sizeof(T), [&](auto nt) {
        hipLaunchKernelGGL((pack_kernel<T, nt>),
                           grid_for(n, first, nt ? 2 : 1), dim3(kThreads), 0,
                           elem::stream(), (const T*)x.data_ptr(),
                           (signed char*)q.data_ptr(),
                           (unsigned char*)scale.data_ptr(), n, first);
      });
  });
  return {q, scale};
}

at::Tensor act8_unpack(at::Tensor values, at::Tensor scales,
                       at::ScalarType dtype) {
  const long n = values.numel();
  TORCH_CHECK_VALUE(
      values.is_cuda() && values.scalar_type() == at::kChar &&
          scales.device() == values.device() &&
          scales.scalar_type() == at::kByte &&
          scales.numel() == (n + 31) / 32 &&
          (dtype == at::kBFloat16 || dtype == at::kHalf ||
           dtype == at::kFloat),
      "Stoke -- restore_activation takes what compress_activation returned: "
      "int8 values and one uint8 exponent for every 32");
  const c10::DeviceGuard guard(values.device());
  const at::Tensor q = values.contiguous(), scale = scales.contiguous();
  auto x = at::empty(q.sizes(), q.options().dtype(dtype));
  STOKE_ELEM_SWITCH(dtype, "act8_unpack", {
    const long first = first_of(n);
    if (n > 0)
      with_caching(n * (long)sizeof(T), [&](auto nt) {
        hipLaunchKernelGGL((unpack_kernel<T, nt>),
                           grid_for(n, first, nt ? 2 : 1), dim3(kThreads), 0,
                           elem::stream(), (const signed char*)q.data_ptr(),
                           (const unsigned char*)scale.data_ptr(),
                           (T*)x.data_ptr(), n, first);
      });
  });
  return x;
}

// The entry point: checks its arguments, and has gradients for both.
at::Tensor swiglu8(at::Tensor g, at::Tensor u) {
  elem::refuse_tangents("swiglu(save_bits=8)", g, u);
  TORCH_CHECK_VALUE(
      g.is_cuda() && g.sizes() == u.sizes() && g.device() == u.device() &&
          g.scalar_type() == u.scalar_type() &&
          (g.scalar_type() == at::kBFloat16 ||
           g.scalar_type() == at::kHalf || g.scalar_type() == at::kFloat),
      "Stoke -- swiglu(save_bits=8) takes gate and up of one shape, device "
      "and dtype (bf16, fp16, fp32), got ", g.sizes(), " ", g.scalar_type(),
      " and ", u.sizes(), " ", u.scalar_type());
  if (!at::GradMode::is_enabled() || !(g.requires_grad() || u.requires_grad()))
    return swiglu8_forward(g, u, nullptr);
  elem::check_capture({g, u});
  return SwiGLU8::apply(g, u);
}
