// stoke-amd native HIP kernels for MI355X (gfx950, CDNA4).
//
// These replace the CUDA kernels the reference implicitly relied on through
// its dependencies:
//   * torch.cuda.amp GradScaler ops (_amp_foreach_non_finite_check_and_unscale_,
//     _amp_update_scale_)            -> multi_tensor_unscale / amp_update_scale
//   * apex/fairscale FusedAdam      -> multi_tensor_adamw (+ bf16-param variant)
//   * torch clip_grad_norm_ / _value_ reductions -> multi_tensor_l2norm / clamp
//
// Design notes (per /opt/skills/guides/cdna_hip_programming.md):
//   * wavefront = 64; BLOCK = 256 threads (multiple of 64).
//   * All ops here are HBM-bandwidth-bound elementwise/reduction work: the
//     lever is vectorized 16 B/lane access (float4), not MFMA.
//   * Multi-tensor-apply: one launch covers many tensors via a by-value
//     kernarg struct of chunk descriptors (no per-tensor launches, no device
//     metadata allocations).
//   * Reductions do wave-level __shfl_down then one LDS step, one atomic per
//     block (Guideline 12).

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <vector>

#define BLOCK 256
#define CHUNK (1 << 16)  // elements per block-chunk
#define MAX_TENSORS 24
#define MAX_BLOCKS 256

namespace {

// ---------------------------------------------------------------------------
// Multi-tensor-apply plumbing: chunk descriptors passed by value in kernarg.
// ---------------------------------------------------------------------------
template <int DEPTH>
struct ChunkMeta {
  const void* addr[DEPTH][MAX_TENSORS];
  int sizes[MAX_TENSORS];
  unsigned char block_to_tensor[MAX_BLOCKS];
  int block_to_chunk[MAX_BLOCKS];
  int nblocks;
};

template <int DEPTH, typename Functor, typename... Args>
__global__ __launch_bounds__(BLOCK) void mta_kernel(ChunkMeta<DEPTH> meta,
                                                    Functor fn, Args... args) {
  const int bid = blockIdx.x;
  if (bid >= meta.nblocks) return;
  const int t = meta.block_to_tensor[bid];
  const int chunk = meta.block_to_chunk[bid];
  const int n = meta.sizes[t];
  const int start = chunk * CHUNK;
  const int len = min(CHUNK, n - start);
  fn(meta, t, start, len, args...);
}

template <int DEPTH, typename Functor, typename... Args>
void multi_tensor_apply(const std::vector<std::vector<at::Tensor>>& lists,
                        Functor fn, Args... args) {
  TORCH_CHECK(lists.size() == DEPTH, "depth mismatch");
  const int ntensors = lists[0].size();
  if (ntensors == 0) return;
  auto stream = at::hip::getCurrentHIPStream();
  ChunkMeta<DEPTH> meta;
  // Find the last non-empty tensor so the final launch triggers in-loop.
  int last_idx = -1;
  for (int i = 0; i < ntensors; ++i)
    if (lists[0][i].numel() > 0) last_idx = i;
  if (last_idx < 0) return;
  int ti = -1;  // tensor slot within meta
  int bi = 0;   // block slot within meta
  for (int i = 0; i < ntensors; ++i) {
    const int n = lists[0][i].numel();
    if (n == 0) continue;
    ++ti;
    meta.sizes[ti] = n;
    for (int d = 0; d < DEPTH; ++d) meta.addr[d][ti] = lists[d][i].data_ptr();
    const int nchunks = (n + CHUNK - 1) / CHUNK;
    for (int c = 0; c < nchunks; ++c) {
      meta.block_to_tensor[bi] = ti;
      meta.block_to_chunk[bi] = c;
      ++bi;
      const bool tensors_full = (ti == MAX_TENSORS - 1 && c == nchunks - 1);
      const bool blocks_full = (bi == MAX_BLOCKS);
      const bool is_last = (i == last_idx && c == nchunks - 1);
      if (tensors_full || blocks_full || is_last) {
        meta.nblocks = bi;
        hipLaunchKernelGGL((mta_kernel<DEPTH, Functor, Args...>), dim3(bi),
                           dim3(BLOCK), 0, stream.stream(), meta, fn, args...);
        bi = 0;
        if (c == nchunks - 1) {
          ti = -1;  // next tensor starts a fresh meta
        } else {
          // Mid-tensor flush: keep this tensor in slot 0 for remaining chunks.
          meta.sizes[0] = n;
          for (int d = 0; d < DEPTH; ++d) meta.addr[d][0] = meta.addr[d][ti];
          ti = 0;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Helpers
// ---------------------------------------------------------------------------
__device__ __forceinline__ float warp_reduce_sum(float v) {
  #pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off);
  return v;
}

__device__ __forceinline__ float block_reduce_sum(float v) {
  __shared__ float smem[BLOCK / 64];
  const int lane = threadIdx.x & 63;
  const int wid = threadIdx.x >> 6;
  v = warp_reduce_sum(v);
  if (lane == 0) smem[wid] = v;
  __syncthreads();
  v = (threadIdx.x < BLOCK / 64) ? smem[threadIdx.x] : 0.f;
  if (wid == 0) {
    #pragma unroll
    for (int off = BLOCK / 128; off > 0; off >>= 1) v += __shfl_down(v, off);
  }
  return v;
}

typedef float float4v __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Functors
// ---------------------------------------------------------------------------

// grads *= inv_scale; found_inf = 1.0 if any non-finite (fused unscale+check).
struct UnscaleFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             const float* inv_scale, float* found_inf) const {
    float* g = ((float*)meta.addr[0][t]) + start;
    const float inv = *inv_scale;
    bool bad = false;
    // float4 path only for 16-B-aligned chunk bases (grad views may be offset)
    const int n4 = ((reinterpret_cast<uintptr_t>(g) & 15) == 0) ? (len & ~3) : 0;
    for (int i = threadIdx.x * 4; i < n4; i += BLOCK * 4) {
      float4v v = *(const float4v*)(g + i);
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x = v[k] * inv;
        bad |= !isfinite(x);
        v[k] = x;
      }
      *(float4v*)(g + i) = v;
    }
    for (int i = n4 + threadIdx.x; i < len; i += BLOCK) {
      float x = g[i] * inv;
      bad |= !isfinite(x);
      g[i] = x;
    }
    if (__any(bad) && (threadIdx.x & 63) == 0) *found_inf = 1.0f;
  }
};

// 2-byte-dtype variant (fp16/bf16 grads): same fused unscale + finite check,
// vectorized 8 elements (16 B) per lane.  Exists so the scaler never falls
// back to foreach + per-tensor host isfinite syncs in fp16 AMP mode
//
typedef __attribute__((ext_vector_type(8))) short short8v;

// __HIP_NO_HALF_CONVERSIONS__ is set by the torch build: use explicit
// intrinsics instead of C-style casts for fp16<->fp32.
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__hip_bfloat16 v) {
  return __bfloat162float(v);
}
__device__ __forceinline__ void from_f32(__half& d, float x) {
  d = __float2half(x);
}
__device__ __forceinline__ void from_f32(__hip_bfloat16& d, float x) {
  d = __float2bfloat16(x);
}

template <typename T>
struct UnscaleHalfFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             const float* inv_scale, float* found_inf) const {
    T* g = ((T*)meta.addr[0][t]) + start;
    const float inv = *inv_scale;
    bool bad = false;
    const int n8 = ((reinterpret_cast<uintptr_t>(g) & 15) == 0) ? (len & ~7) : 0;
    for (int i = threadIdx.x * 8; i < n8; i += BLOCK * 8) {
      short8v v = *(const short8v*)(g + i);
      T* e = reinterpret_cast<T*>(&v);
      #pragma unroll
      for (int k = 0; k < 8; ++k) {
        float x = to_f32(e[k]) * inv;
        bad |= !isfinite(x);
        from_f32(e[k], x);
      }
      *(short8v*)(g + i) = v;
    }
    for (int i = n8 + threadIdx.x; i < len; i += BLOCK) {
      float x = to_f32(g[i]) * inv;
      bad |= !isfinite(x);
      from_f32(g[i], x);
    }
    if (__any(bad) && (threadIdx.x & 63) == 0) *found_inf = 1.0f;
  }
};

// out[0] += sum(x*x) over all chunks (fp32 or bf16 input)
template <typename T>
struct L2NormFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             float* out) const {
    const T* g = ((const T*)meta.addr[0][t]) + start;
    float acc = 0.f;
    for (int i = threadIdx.x; i < len; i += BLOCK) {
      float x = (float)g[i];
      acc += x * x;
    }
    acc = block_reduce_sum(acc);
    if (threadIdx.x == 0) atomicAdd(out, acc);
  }
};

// x *= scale (by pointer so it composes with device-side clip coefficients)
struct ScalePtrFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             const float* scale) const {
    float* g = ((float*)meta.addr[0][t]) + start;
    const float s = *scale;
    const int n4 = ((reinterpret_cast<uintptr_t>(g) & 15) == 0) ? (len & ~3) : 0;
    for (int i = threadIdx.x * 4; i < n4; i += BLOCK * 4) {
      float4v v = *(const float4v*)(g + i);
      #pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= s;
      *(float4v*)(g + i) = v;
    }
    for (int i = n4 + threadIdx.x; i < len; i += BLOCK) g[i] *= s;
  }
};

// clamp to [-limit, limit]
struct ClampFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             float limit) const {
    float* g = ((float*)meta.addr[0][t]) + start;
    const int n4 = ((reinterpret_cast<uintptr_t>(g) & 15) == 0) ? (len & ~3) : 0;
    for (int i = threadIdx.x * 4; i < n4; i += BLOCK * 4) {
      float4v v = *(const float4v*)(g + i);
      #pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = fminf(fmaxf(v[k], -limit), limit);
      *(float4v*)(g + i) = v;
    }
    for (int i = n4 + threadIdx.x; i < len; i += BLOCK)
      g[i] = fminf(fmaxf(g[i], -limit), limit);
  }
};

// AdamW, fp32 params/grads/state, decoupled weight decay, bias correction.
// Optionally skips the whole update when *found_inf != 0 (scaler-integrated),
// and unscales the gradient in-register (grad_scale = 1/loss_scale).
struct AdamWFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             float lr, float beta1, float beta2, float eps,
                             float weight_decay, float bc1, float bc2,
                             const float* found_inf, const float* inv_scale) const {
    if (found_inf && *found_inf != 0.f) return;
    float* p = ((float*)meta.addr[0][t]) + start;
    float* g = ((float*)meta.addr[1][t]) + start;
    float* m = ((float*)meta.addr[2][t]) + start;
    float* v = ((float*)meta.addr[3][t]) + start;
    const float inv = inv_scale ? *inv_scale : 1.f;
    const int n4 = ((reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(g) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(m) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(v) & 15) == 0)
                       ? (len & ~3) : 0;
    for (int i = threadIdx.x * 4; i < n4; i += BLOCK * 4) {
      float4v pv = *(const float4v*)(p + i);
      float4v gv = *(const float4v*)(g + i);
      float4v mv = *(const float4v*)(m + i);
      float4v vv = *(const float4v*)(v + i);
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        float gg = gv[k] * inv;
        float mm = beta1 * mv[k] + (1.f - beta1) * gg;
        float vn = beta2 * vv[k] + (1.f - beta2) * gg * gg;
        float denom = sqrtf(vn / bc2) + eps;
        float update = (mm / bc1) / denom + weight_decay * pv[k];
        pv[k] = pv[k] - lr * update;
        mv[k] = mm;
        vv[k] = vn;
      }
      *(float4v*)(p + i) = pv;
      *(float4v*)(m + i) = mv;
      *(float4v*)(v + i) = vv;
    }
    for (int i = n4 + threadIdx.x; i < len; i += BLOCK) {
      float gg = g[i] * inv;
      float mm = beta1 * m[i] + (1.f - beta1) * gg;
      float vn = beta2 * v[i] + (1.f - beta2) * gg * gg;
      float denom = sqrtf(vn / bc2) + eps;
      float update = (mm / bc1) / denom + weight_decay * p[i];
      p[i] = p[i] - lr * update;
      m[i] = mm;
      v[i] = vn;
    }
  }
};

// AdamW with bf16 model params + fp32 master params/state, bf16 grads
// (the FSDP bf16 flat-shard path: depth 5 = [bf16 p, bf16 g, fp32 m, fp32 v,
// fp32 master]).  Vectorized 8-wide: bf16x8 (16 B) for p/g, 2x float4 for
// m/v/w — the scalar version measured 19% of a Llama-8B step (2-byte loads).
union adam_bf16x8 {
  uint4 u4;
  unsigned short h[8];
};

struct AdamWBF16Functor {
  __device__ __forceinline__ float upd(float gg, float& mm, float& vn,
                                       float pw, float lr, float beta1,
                                       float beta2, float eps, float wd,
                                       float bc1, float bc2) const {
    mm = beta1 * mm + (1.f - beta1) * gg;
    vn = beta2 * vn + (1.f - beta2) * gg * gg;
    float denom = sqrtf(vn / bc2) + eps;
    return pw - lr * ((mm / bc1) / denom + wd * pw);
  }

  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             float lr, float beta1, float beta2, float eps,
                             float weight_decay, float bc1, float bc2,
                             const float* found_inf, const float* inv_scale) const {
    if (found_inf && *found_inf != 0.f) return;
    __hip_bfloat16* p = ((__hip_bfloat16*)meta.addr[0][t]) + start;
    const __hip_bfloat16* g = ((const __hip_bfloat16*)meta.addr[1][t]) + start;
    float* m = ((float*)meta.addr[2][t]) + start;
    float* v = ((float*)meta.addr[3][t]) + start;
    float* w = ((float*)meta.addr[4][t]) + start;  // fp32 master copy
    const float inv = inv_scale ? *inv_scale : 1.f;
    const bool aligned = ((reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
                          (reinterpret_cast<uintptr_t>(g) & 15) == 0 &&
                          (reinterpret_cast<uintptr_t>(m) & 15) == 0 &&
                          (reinterpret_cast<uintptr_t>(v) & 15) == 0 &&
                          (reinterpret_cast<uintptr_t>(w) & 15) == 0);
    const int n8 = aligned ? (len & ~7) : 0;
    for (int i = threadIdx.x * 8; i < n8; i += BLOCK * 8) {
      adam_bf16x8 gv;
      gv.u4 = *(const uint4*)(g + i);
      float4v m0 = *(const float4v*)(m + i);
      float4v m1 = *(const float4v*)(m + i + 4);
      float4v v0 = *(const float4v*)(v + i);
      float4v v1 = *(const float4v*)(v + i + 4);
      float4v w0 = *(const float4v*)(w + i);
      float4v w1 = *(const float4v*)(w + i + 4);
      adam_bf16x8 pv;
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        __hip_bfloat16_raw r;
        r.x = gv.h[k];
        float gg = __bfloat162float(*reinterpret_cast<__hip_bfloat16*>(&r)) * inv;
        float mm = m0[k], vn = v0[k];
        float pw = upd(gg, mm, vn, w0[k], lr, beta1, beta2, eps,
                       weight_decay, bc1, bc2);
        m0[k] = mm;
        v0[k] = vn;
        w0[k] = pw;
        __hip_bfloat16 hb = __float2bfloat16(pw);
        pv.h[k] = *reinterpret_cast<unsigned short*>(&hb);
      }
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        __hip_bfloat16_raw r;
        r.x = gv.h[4 + k];
        float gg = __bfloat162float(*reinterpret_cast<__hip_bfloat16*>(&r)) * inv;
        float mm = m1[k], vn = v1[k];
        float pw = upd(gg, mm, vn, w1[k], lr, beta1, beta2, eps,
                       weight_decay, bc1, bc2);
        m1[k] = mm;
        v1[k] = vn;
        w1[k] = pw;
        __hip_bfloat16 hb = __float2bfloat16(pw);
        pv.h[4 + k] = *reinterpret_cast<unsigned short*>(&hb);
      }
      *(uint4*)(p + i) = pv.u4;
      *(float4v*)(m + i) = m0;
      *(float4v*)(m + i + 4) = m1;
      *(float4v*)(v + i) = v0;
      *(float4v*)(v + i + 4) = v1;
      *(float4v*)(w + i) = w0;
      *(float4v*)(w + i + 4) = w1;
    }
    for (int i = n8 + threadIdx.x; i < len; i += BLOCK) {
      float gg = __bfloat162float(g[i]) * inv;
      float mm = m[i], vn = v[i];
      float pw = upd(gg, mm, vn, w[i], lr, beta1, beta2, eps, weight_decay,
                     bc1, bc2);
      w[i] = pw;
      p[i] = __float2bfloat16(pw);
      m[i] = mm;
      v[i] = vn;
    }
  }
};

// SGD with momentum (torch.optim.SGD semantics incl. first-step buf = g),
// fp32 params/grads/buf, depth 3.  found_inf/inv_scale integrate with the
// scaler exactly like AdamWFunctor (device-side skip, in-register unscale).
struct SGDFunctor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             float lr, float momentum, float dampening,
                             float weight_decay, int nesterov, int first_step,
                             const float* found_inf,
                             const float* inv_scale) const {
    if (found_inf && *found_inf != 0.f) return;
    float* p = ((float*)meta.addr[0][t]) + start;
    float* g = ((float*)meta.addr[1][t]) + start;
    float* b = ((float*)meta.addr[2][t]) + start;
    const float inv = inv_scale ? *inv_scale : 1.f;
    const int n4 = ((reinterpret_cast<uintptr_t>(p) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(g) & 15) == 0 &&
                    (reinterpret_cast<uintptr_t>(b) & 15) == 0)
                       ? (len & ~3) : 0;
    for (int i = threadIdx.x * 4; i < n4; i += BLOCK * 4) {
      float4v pv = *(const float4v*)(p + i);
      float4v gv = *(const float4v*)(g + i);
      float4v bv = *(const float4v*)(b + i);
      #pragma unroll
      for (int k = 0; k < 4; ++k) {
        float gg = gv[k] * inv + weight_decay * pv[k];
        if (momentum != 0.f) {
          float bb = first_step ? gg
                                : momentum * bv[k] + (1.f - dampening) * gg;
          bv[k] = bb;
          gg = nesterov ? gg + momentum * bb : bb;
        }
        pv[k] -= lr * gg;
      }
      *(float4v*)(p + i) = pv;
      if (momentum != 0.f) *(float4v*)(b + i) = bv;
    }
    for (int i = n4 + threadIdx.x; i < len; i += BLOCK) {
      float gg = g[i] * inv + weight_decay * p[i];
      if (momentum != 0.f) {
        float bb = first_step ? gg : momentum * b[i] + (1.f - dampening) * gg;
        b[i] = bb;
        gg = nesterov ? gg + momentum * bb : bb;
      }
      p[i] -= lr * gg;
    }
  }
};

// bf16 params/grads + fp32 momentum buf + fp32 master (depth 4) — the
// pure-bf16-weights LM training path, mirroring AdamWBF16Functor.
struct SGDBF16Functor {
  template <typename Meta>
  __device__ void operator()(const Meta& meta, int t, int start, int len,
                             float lr, float momentum, float dampening,
                             float weight_decay, int nesterov, int first_step,
                             const float* found_inf,
                             const float* inv_scale) const {
    if (found_inf && *found_inf != 0.f) return;
    __hip_bfloat16* p = ((__hip_bfloat16*)meta.addr[0][t]) + start;
    const __hip_bfloat16* g = ((const __hip_bfloat16*)meta.addr[1][t]) + start;
    float* b = ((float*)meta.addr[2][t]) + start;
    float* w = ((float*)meta.addr[3][t]) + start;
    const float inv = inv_scale ? *inv_scale : 1.f;
    for (int i = threadIdx.x; i < len; i += BLOCK) {
      float pw = w[i];
      float gg = __bfloat162float(g[i]) * inv + weight_decay * pw;
      if (momentum != 0.f) {
        float bb = first_step ? gg : momentum * b[i] + (1.f - dampening) * gg;
        b[i] = bb;
        gg = nesterov ? gg + momentum * bb : bb;
      }
      pw -= lr * gg;
      w[i] = pw;
      p[i] = __float2bfloat16(pw);
    }
  }
};

// Dynamic loss-scale update with hysteresis (replaces _amp_update_scale_).
__global__ void amp_update_scale_kernel(float* scale, int* growth_tracker,
                                        const float* found_inf,
                                        float growth_factor,
                                        float backoff_factor,
                                        int growth_interval) {
  if (*found_inf != 0.f) {
    *scale *= backoff_factor;
    *growth_tracker = 0;
  } else {
    int g = *growth_tracker + 1;
    if (g >= growth_interval) {
      *scale *= growth_factor;
      g = 0;
    }
    *growth_tracker = g;
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Python-visible entry points
// ---------------------------------------------------------------------------

void multi_tensor_unscale_(std::vector<at::Tensor> grads, at::Tensor inv_scale,
                           at::Tensor found_inf) {
  const auto dt = grads[0].scalar_type();
  if (dt == at::kHalf) {
    multi_tensor_apply<1>({grads}, UnscaleHalfFunctor<__half>{},
                          inv_scale.data_ptr<float>(),
                          found_inf.data_ptr<float>());
  } else if (dt == at::kBFloat16) {
    multi_tensor_apply<1>({grads}, UnscaleHalfFunctor<__hip_bfloat16>{},
                          inv_scale.data_ptr<float>(),
                          found_inf.data_ptr<float>());
  } else {
    multi_tensor_apply<1>({grads}, UnscaleFunctor{},
                          inv_scale.data_ptr<float>(),
                          found_inf.data_ptr<float>());
  }
}

at::Tensor multi_tensor_l2norm_sq(std::vector<at::Tensor> tensors) {
  auto out = at::zeros({1}, tensors[0].options().dtype(at::kFloat));
  if (tensors[0].scalar_type() == at::kBFloat16) {
    multi_tensor_apply<1>({tensors}, L2NormFunctor<__hip_bfloat16>{},
                          out.data_ptr<float>());
  } else {
    multi_tensor_apply<1>({tensors}, L2NormFunctor<float>{},
                          out.data_ptr<float>());
  }
  return out;
}

void multi_tensor_scale_(std::vector<at::Tensor> tensors, at::Tensor scale) {
  multi_tensor_apply<1>({tensors}, ScalePtrFunctor{}, scale.data_ptr<float>());
}

void multi_tensor_clamp_(std::vector<at::Tensor> tensors, double limit) {
  multi_tensor_apply<1>({tensors}, ClampFunctor{}, (float)limit);
}

void multi_tensor_adamw_(std::vector<at::Tensor> params,
                         std::vector<at::Tensor> grads,
                         std::vector<at::Tensor> exp_avgs,
                         std::vector<at::Tensor> exp_avg_sqs,
                         int64_t step, double lr, double beta1, double beta2,
                         double eps, double weight_decay,
                         c10::optional<at::Tensor> found_inf,
                         c10::optional<at::Tensor> inv_scale) {
  const float bc1 = 1.f - powf((float)beta1, (float)step);
  const float bc2 = 1.f - powf((float)beta2, (float)step);
  const float* fi = found_inf ? found_inf->data_ptr<float>() : nullptr;
  const float* is = inv_scale ? inv_scale->data_ptr<float>() : nullptr;
  multi_tensor_apply<4>({params, grads, exp_avgs, exp_avg_sqs}, AdamWFunctor{},
                        (float)lr, (float)beta1, (float)beta2, (float)eps,
                        (float)weight_decay, bc1, bc2, fi, is);
}

void multi_tensor_adamw_bf16_(std::vector<at::Tensor> params,
                              std::vector<at::Tensor> grads,
                              std::vector<at::Tensor> exp_avgs,
                              std::vector<at::Tensor> exp_avg_sqs,
                              std::vector<at::Tensor> masters,
                              int64_t step, double lr, double beta1,
                              double beta2, double eps, double weight_decay,
                              c10::optional<at::Tensor> found_inf,
                              c10::optional<at::Tensor> inv_scale) {
  const float bc1 = 1.f - powf((float)beta1, (float)step);
  const float bc2 = 1.f - powf((float)beta2, (float)step);
  const float* fi = found_inf ? found_inf->data_ptr<float>() : nullptr;
  const float* is = inv_scale ? inv_scale->data_ptr<float>() : nullptr;
  multi_tensor_apply<5>({params, grads, exp_avgs, exp_avg_sqs, masters},
                        AdamWBF16Functor{}, (float)lr, (float)beta1,
                        (float)beta2, (float)eps, (float)weight_decay, bc1,
                        bc2, fi, is);
}

void multi_tensor_sgd_(std::vector<at::Tensor> params,
                       std::vector<at::Tensor> grads,
                       std::vector<at::Tensor> momentum_bufs,
                       double lr, double momentum, double dampening,
                       double weight_decay, bool nesterov, bool first_step,
                       c10::optional<at::Tensor> found_inf,
                       c10::optional<at::Tensor> inv_scale) {
  const float* fi = found_inf ? found_inf->data_ptr<float>() : nullptr;
  const float* is = inv_scale ? inv_scale->data_ptr<float>() : nullptr;
  multi_tensor_apply<3>({params, grads, momentum_bufs}, SGDFunctor{},
                        (float)lr, (float)momentum, (float)dampening,
                        (float)weight_decay, nesterov ? 1 : 0,
                        first_step ? 1 : 0, fi, is);
}

void multi_tensor_sgd_bf16_(std::vector<at::Tensor> params,
                            std::vector<at::Tensor> grads,
                            std::vector<at::Tensor> momentum_bufs,
                            std::vector<at::Tensor> masters,
                            double lr, double momentum, double dampening,
                            double weight_decay, bool nesterov,
                            bool first_step,
                            c10::optional<at::Tensor> found_inf,
                            c10::optional<at::Tensor> inv_scale) {
  const float* fi = found_inf ? found_inf->data_ptr<float>() : nullptr;
  const float* is = inv_scale ? inv_scale->data_ptr<float>() : nullptr;
  multi_tensor_apply<4>({params, grads, momentum_bufs, masters},
                        SGDBF16Functor{}, (float)lr, (float)momentum,
                        (float)dampening, (float)weight_decay,
                        nesterov ? 1 : 0, first_step ? 1 : 0, fi, is);
}

void amp_update_scale_(at::Tensor scale, at::Tensor growth_tracker,
                       at::Tensor found_inf, double growth_factor,
                       double backoff_factor, int64_t growth_interval) {
  auto stream = at::hip::getCurrentHIPStream();
  hipLaunchKernelGGL(amp_update_scale_kernel, dim3(1), dim3(1), 0,
                     stream.stream(), scale.data_ptr<float>(),
                     growth_tracker.data_ptr<int>(),
                     found_inf.data_ptr<float>(), (float)growth_factor,
                     (float)backoff_factor, (int)growth_interval);
}

// Fused cross-entropy (csrc/fused_ce.hip)
std::vector<at::Tensor> ce_fwd(at::Tensor logits, at::Tensor target,
                               int64_t ignore_index);
at::Tensor ce_bwd(at::Tensor logits, at::Tensor target, at::Tensor lse,
                  at::Tensor gscale, int64_t ignore_index);

// Fused NHWC BatchNorm kernels (csrc/fused_bn.hip)
std::vector<at::Tensor> bn_fwd_train(
    at::Tensor x, c10::optional<at::Tensor> residual, at::Tensor gamma,
    at::Tensor beta, c10::optional<at::Tensor> running_mean,
    c10::optional<at::Tensor> running_var, double eps, double momentum,
    bool relu);
at::Tensor bn_fwd_eval(at::Tensor x, c10::optional<at::Tensor> residual,
                       at::Tensor gamma, at::Tensor beta,
                       at::Tensor running_mean, at::Tensor running_var,
                       double eps, bool relu);
std::vector<at::Tensor> bn_bwd(at::Tensor x, at::Tensor dy, at::Tensor y,
                               at::Tensor mean, at::Tensor invstd,
                               at::Tensor gamma, bool relu, bool needs_dres);

// Fused RMSNorm kernels (csrc/fused_rmsnorm.hip)
std::vector<at::Tensor> rmsnorm_fwd(at::Tensor x, at::Tensor w, double eps);
std::vector<at::Tensor> rmsnorm_bwd(at::Tensor x, at::Tensor dy, at::Tensor w,
                                    at::Tensor invr);

// Fused RoPE kernel (csrc/fused_rope.hip)
at::Tensor rope_apply(at::Tensor x, at::Tensor cosc, at::Tensor sinc,
                      bool conj);

// Fused SwiGLU kernels (csrc/fused_swiglu.hip)
at::Tensor swiglu_fwd(at::Tensor g, at::Tensor u);
std::vector<at::Tensor> swiglu_bwd(at::Tensor dy, at::Tensor g, at::Tensor u);

// Fused LayerNorm kernels (csrc/fused_layernorm.hip)
std::vector<at::Tensor> layernorm_fwd(at::Tensor x, at::Tensor w, at::Tensor b,
                                      double eps);
std::vector<at::Tensor> layernorm_bwd(at::Tensor x, at::Tensor dy,
                                      at::Tensor w, at::Tensor mean,
                                      at::Tensor invstd);

// Flash-attention forward (csrc/fa_fwd.hip)
void mfma_probe(at::Tensor A, at::Tensor B, at::Tensor D);
void mfma_probe32(at::Tensor A, at::Tensor B, at::Tensor D);
std::vector<at::Tensor> fa_fwd(at::Tensor q, at::Tensor k, at::Tensor v,
                               bool causal);
std::vector<at::Tensor> fa_bwd(at::Tensor q, at::Tensor k, at::Tensor v,
                               at::Tensor out, at::Tensor dout,
                               at::Tensor lse, bool causal);

// fp8 fused quantizers (csrc/fp8_quant.hip)
at::Tensor fp8_quant(at::Tensor x, at::Tensor scale, at::Tensor amax_next,
                     int64_t kind);
std::vector<at::Tensor> fp8_quant_t(at::Tensor x, at::Tensor scale,
                                    at::Tensor amax_next, int64_t kind);

// Activations held in 8 bits (csrc/act8.hip)
std::vector<at::Tensor> act8_pack(at::Tensor act);
at::Tensor act8_unpack(at::Tensor values, at::Tensor scales,
                       at::ScalarType dtype);
at::Tensor swiglu8(at::Tensor g, at::Tensor u);

// Token log-probabilities and the losses on them (csrc/token_loss.hip)
at::Tensor token_logprobs(at::Tensor logits, at::Tensor target,
                          int64_t ignore);
at::Tensor policy_loss(at::Tensor logits, at::Tensor target,
                       at::Tensor old_lp, at::Tensor adv,
                       std::optional<at::Tensor> ref_lp, double clip_low,
                       double clip_high, double kl, int64_t ignore);
std::vector<at::Tensor> preference_loss(at::Tensor logits, at::Tensor target,
                                        at::Tensor ref_lp, double beta,
                                        double eps, int64_t ignore);

// Norm and rotation of query and key heads (csrc/qk_norm_rope.hip)
std::vector<at::Tensor> qk_norm_rope(
    at::Tensor q, at::Tensor k, std::optional<at::Tensor> wq,
    std::optional<at::Tensor> wk, at::Tensor cosines, at::Tensor sines,
    std::optional<at::Tensor> pos,
    std::optional<std::vector<int64_t>> sections, double eps,
    bool interleaved);

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("ce_fwd", &ce_fwd, "fused bf16 cross-entropy forward (online lse)");
  m.def("ce_bwd", &ce_bwd, "fused bf16 cross-entropy backward");
  m.def("bn_fwd_train", &bn_fwd_train,
        "fused NHWC bf16 BN forward (train): stats + scale/shift(+res)+relu");
  m.def("bn_fwd_eval", &bn_fwd_eval, "fused NHWC bf16 BN forward (eval)");
  m.def("bn_bwd", &bn_bwd,
        "fused NHWC bf16 BN backward: reduce(+relu mask) + dx(+dres)");
  m.def("rmsnorm_fwd", &rmsnorm_fwd,
        "fused bf16 RMSNorm forward: y = x*rsqrt(mean(x^2)+eps)*w");
  m.def("rmsnorm_bwd", &rmsnorm_bwd, "fused bf16 RMSNorm backward");
  m.def("rope_apply", &rope_apply,
        "fused bf16 rotary embedding (conj=true for the backward rotation)");
  m.def("swiglu_fwd", &swiglu_fwd, "fused bf16 silu(g)*u");
  m.def("swiglu_bwd", &swiglu_bwd, "fused bf16 SwiGLU backward");
  m.def("layernorm_fwd", &layernorm_fwd, "fused bf16 LayerNorm forward");
  m.def("layernorm_bwd", &layernorm_bwd, "fused bf16 LayerNorm backward");
  m.def("mfma_probe32", &mfma_probe32,
        "layout probe: one v_mfma_f32_32x32x16_bf16 (A[32,16] x B[16,32])");
  m.def("mfma_probe", &mfma_probe,
        "16x16x32 bf16 MFMA fragment-layout probe");
  m.def("fa_fwd", &fa_fwd,
        "CDNA4 flash-attention forward (strip-paired FA-2, strided views)");
  m.def("fa_bwd", &fa_bwd,
        "CDNA4 flash-attention backward (dkv + dq + delta)");
  m.def("fp8_quant", &fp8_quant,
        "fused bf16->fp8 quantize + next-amax byproduct");
  m.def("fp8_quant_t", &fp8_quant_t,
        "fused bf16->fp8 quantize emitting row-major AND transposed layouts");
  m.def("multi_tensor_unscale_", &multi_tensor_unscale_,
        "fused grad unscale + inf/nan check (HIP)");
  m.def("multi_tensor_l2norm_sq", &multi_tensor_l2norm_sq,
        "sum of squares over tensor list (HIP)");
  m.def("multi_tensor_scale_", &multi_tensor_scale_,
        "in-place scale by device scalar (HIP)");
  m.def("multi_tensor_clamp_", &multi_tensor_clamp_,
        "in-place clamp to [-limit, limit] (HIP)");
  m.def("multi_tensor_adamw_", &multi_tensor_adamw_,
        "fused AdamW, fp32 (HIP)");
  m.def("multi_tensor_sgd_", &multi_tensor_sgd_,
        "fused multi-tensor SGD-momentum step (HIP)");
  m.def("multi_tensor_sgd_bf16_", &multi_tensor_sgd_bf16_,
        "fused SGD for bf16 params with fp32 masters (HIP)");
  m.def("multi_tensor_adamw_bf16_", &multi_tensor_adamw_bf16_,
        "fused AdamW, bf16 params + fp32 master (HIP)");
  m.def("amp_update_scale_", &amp_update_scale_,
        "dynamic loss scale update (HIP)");
  m.def("act8_pack", &act8_pack, "activation to 8 bits");
  m.def("act8_unpack", &act8_unpack, "activation back from 8 bits");
  m.def("swiglu8", &swiglu8,
        "silu(g)*u, keeping g and u in 8 bits for the backward");
  m.def("token_logprobs", &token_logprobs,
        "log-probabilities of given tokens");
  m.def("policy_loss", &policy_loss, "clipped policy loss with a KL term");
  m.def("preference_loss", &preference_loss, "paired preference loss");
  m.def("qk_norm_rope", &qk_norm_rope,
        "per-head RMS norm and rotation of queries and keys");
  m.attr("_built_for") = "gfx950";
}
