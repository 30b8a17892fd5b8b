// Activations held in 8 bits (MXINT8: 32 values share a power of two).
//
// A block of 32 consecutive values of the flattened tensor keeps one byte
// E and 32 signed bytes q with  value = q * 2^(E - 127),  |q| <= 127.
// E is the least exponent from 1 up at which the block's largest value still
// rounds into 127, so a value is off by at most half of 2^(E-127), that is
// 1/127 of the block's largest.  Scaling by a power of two is exact: the one
// rounding is the conversion to a whole number (half to even).  E = 255
// marks a block with an infinity or NaN; all of it reads back as NaN, so an
// overflow in the forward pass still reaches the gradients.

#include <hip/hip_runtime.h>

#include "elem.h"

namespace {

using elem::kVec;

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

// One value per lane: any length.
template <typename T>
__global__ __launch_bounds__(kThreads) void pack_kernel(
    const T* __restrict__ x, signed char* __restrict__ q,
    unsigned char* __restrict__ scale, long n) {
  const long step = (long)gridDim.x * kThreads;
  const long n32 = (n + 31) / 32 * 32;
  for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < n32;
       i += step) {
    const float v = i < n ? (float)x[i] : 0.f;
    const unsigned e =
        block_exponent(half_wave_max(__float_as_uint(v) & 0x7fffffff));
    if (i < n) q[i] = (signed char)quantize(v, e);
    if ((threadIdx.x & 31) == 0) scale[i >> 5] = (unsigned char)e;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void unpack_kernel(
    const signed char* __restrict__ q,
    const unsigned char* __restrict__ scale, T* __restrict__ x, long n) {
  const long step = (long)gridDim.x * kThreads;
  for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < n; i += step)
    x[i] = (T)restored<T>(q[i], scale[i >> 5]);
}

// y = silu(g) * u from the values as they come; g and u stay in 8 bits.
template <typename T>
__global__ __launch_bounds__(kThreads) void swiglu8_fwd_kernel(
    const T* __restrict__ g, const T* __restrict__ u, T* __restrict__ y,
    signed char* __restrict__ qg, signed char* __restrict__ qu,
    unsigned char* __restrict__ sg, unsigned char* __restrict__ su, long n) {
  const long step = (long)gridDim.x * kThreads;
  const long n32 = (n + 31) / 32 * 32;
  for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < n32;
       i += step) {
    const float a = i < n ? (float)g[i] : 0.f;
    const float b = i < n ? (float)u[i] : 0.f;
    const unsigned eg =
        block_exponent(half_wave_max(__float_as_uint(a) & 0x7fffffff));
    const unsigned eu =
        block_exponent(half_wave_max(__float_as_uint(b) & 0x7fffffff));
    if (i < n) {
      y[i] = (T)(a / (1.f + __expf(-a)) * b);
      qg[i] = (signed char)quantize(a, eg);
      qu[i] = (signed char)quantize(b, eu);
    }
    if ((threadIdx.x & 31) == 0) {
      sg[i >> 5] = (unsigned char)eg;
      su[i >> 5] = (unsigned char)eu;
    }
  }
}

// dg = dy u s (1 + g (1 - s)),  du = dy g s,  s = 1 / (1 + e^-g)
template <typename T>
__global__ __launch_bounds__(kThreads) void swiglu8_bwd_kernel(
    const T* __restrict__ dy, const signed char* __restrict__ qg,
    const signed char* __restrict__ qu, const unsigned char* __restrict__ sg,
    const unsigned char* __restrict__ su, T* __restrict__ dg,
    T* __restrict__ du, long n) {
  const long step = (long)gridDim.x * kThreads;
  for (long i = (long)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) {
    const float a = restored<T>(qg[i], sg[i >> 5]);
    const float b = restored<T>(qu[i], su[i >> 5]);
    const float d = (float)dy[i];
    const float s = 1.f / (1.f + __expf(-a));
    dg[i] = (T)(d * b * s * (1.f + a * (1.f - s)));
    du[i] = (T)(d * a * s);
  }
}

inline dim3 grid_for(long items) {
  return dim3((unsigned)std::min<long>((items + kThreads - 1) / kThreads,
                                       65536));
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

}  // namespace

std::vector<at::Tensor> act8_pack(at::Tensor x) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous(),
              "act8_pack: contiguous GPU tensor required");
  const c10::DeviceGuard guard(x.device());
  const long n = x.numel();
  auto q = at::empty(x.sizes(), x.options().dtype(at::kChar));
  auto scale = at::empty({(n + 31) / 32}, x.options().dtype(at::kByte));
  STOKE_ELEM_SWITCH(x.scalar_type(), "act8_pack", {
    if (n > 0)
      hipLaunchKernelGGL((pack_kernel<T>), grid_for(n), dim3(kThreads), 0,
                         elem::stream(), (const T*)x.data_ptr(),
                         (signed char*)q.data_ptr(),
                         (unsigned char*)scale.data_ptr(), n);
  });
  return {q, scale};
}

at::Tensor act8_unpack(at::Tensor q, at::Tensor scale, at::ScalarType dtype) {
  const long n = q.numel();
  TORCH_CHECK(q.is_cuda() && q.is_contiguous() &&
                  q.scalar_type() == at::kChar,
              "act8_unpack: contiguous int8 GPU values required");
  TORCH_CHECK(scale.device() == q.device() && scale.is_contiguous() &&
                  scale.scalar_type() == at::kByte &&
                  scale.numel() == (n + 31) / 32,
              "act8_unpack: one uint8 exponent for every 32 values required");
  const c10::DeviceGuard guard(q.device());
  auto x = at::empty(q.sizes(), q.options().dtype(dtype));
  STOKE_ELEM_SWITCH(dtype, "act8_unpack", {
    if (n > 0)
      hipLaunchKernelGGL((unpack_kernel<T>), grid_for(n), dim3(kThreads), 0,
                         elem::stream(), (const signed char*)q.data_ptr(),
                         (const unsigned char*)scale.data_ptr(),
                         (T*)x.data_ptr(), n);
  });
  return x;
}

std::vector<at::Tensor> swiglu8_fwd(at::Tensor g, at::Tensor u) {
  TORCH_CHECK(g.is_cuda() && u.device() == g.device() &&
                  g.is_contiguous() && u.is_contiguous() &&
                  g.sizes() == u.sizes() &&
                  g.scalar_type() == u.scalar_type(),
              "swiglu8: gate and up must be contiguous GPU tensors of one "
              "shape and dtype");
  const c10::DeviceGuard guard(g.device());
  const long n = g.numel();
  auto y = at::empty_like(g);
  auto held = at::empty({Held(nullptr, n).bytes},
                        g.options().dtype(at::kByte));
  const Held h(held.data_ptr(), n);
  STOKE_ELEM_SWITCH(g.scalar_type(), "swiglu8", {
    if (n > 0)
      hipLaunchKernelGGL((swiglu8_fwd_kernel<T>), grid_for(n),
                         dim3(kThreads), 0, elem::stream(),
                         (const T*)g.data_ptr(), (const T*)u.data_ptr(),
                         (T*)y.data_ptr(), h.qg, h.qu, h.sg, h.su, n);
  });
  return {y, held};
}

std::vector<at::Tensor> swiglu8_bwd(at::Tensor dy, at::Tensor held) {
  const long n = dy.numel();
  const Held h(held.data_ptr(), n);
  TORCH_CHECK(dy.is_cuda() && dy.is_contiguous() &&
                  held.device() == dy.device() && held.numel() == h.bytes,
              "swiglu8: gradient must be a contiguous GPU tensor of the "
              "output's shape");
  const c10::DeviceGuard guard(dy.device());
  auto dg = at::empty_like(dy);
  auto du = at::empty_like(dy);
  STOKE_ELEM_SWITCH(dy.scalar_type(), "swiglu8", {
    if (n > 0)
      hipLaunchKernelGGL((swiglu8_bwd_kernel<T>), grid_for(n),
                         dim3(kThreads), 0, elem::stream(),
                         (const T*)dy.data_ptr(), h.qg, h.qu, h.sg, h.su,
                         (T*)dg.data_ptr(), (T*)du.data_ptr(), n);
  });
  return {dg, du};
}
