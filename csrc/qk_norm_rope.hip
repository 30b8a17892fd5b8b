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
  const void* dy;  // backward
  void* y;         // forward output or dx; contiguous [B, S, H, D]
  const void* w;   // null: ones
  long sb, ss, sh;  // strides of x in elements
  long db, ds, dh;  // and of dy: attention hands back [B, H, S, D]
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
__device__ __forceinline__ float2 angle(const Args& a, long token,
                                        long in_seq, int p) {
  int axis = 0;
  while (axis + 1 < a.axes && p >= a.ends[axis]) ++axis;
  const long at = a.pos ? a.pos[axis * a.tokens + token] : in_seq;
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

// Where a row lies.
struct Row {
  long token, in_seq, x, dy;  // offsets of x and dy
};

__device__ __forceinline__ Row row_of(const Args& a, const Side& s,
                                      long row) {
  Row r;
  r.token = row / s.heads;
  const long no = r.token / a.seq;
  r.in_seq = r.token - no * a.seq;
  const long head = row - r.token * s.heads;
  r.x = no * s.sb + r.in_seq * s.ss + head * s.sh;
  r.dy = no * s.db + r.in_seq * s.ds + head * s.dh;
  return r;
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

// A wave for each row, the row in shared memory: any dim and any number of
// pairs.  Bound by instructions, not by memory: every value finds its own
// position and angle, and a row waits for its block twice.  16384 tokens of 32 +
// 8 heads of 80 bf16 with 20 values rotated take 253 us forward (210 MB) and
// 591 + 28 us backward (315 MB).
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
    const Row at = row_of(a, s, live ? row : 0);
    float r = 0.f;
    if (live) {
      const T* x = (const T*)s.x + at.x;
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
          const float2 cs = angle(a, at.token, at.in_seq, pair_of(a, e));
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
    const Row at = row_of(a, s, live ? row : 0);
    const T* dy = (const T*)s.dy + at.dy;
    if (live)
      for (int e = lane; e < a.dim; e += 64) mine[e] = (float)dy[e];
    __syncthreads();
    if (live) {
      const T* x = (const T*)s.x + at.x;
      T* dx = (T*)s.y + row * a.dim;
      float dn[kMaxDim / 64];
      float sum = 0.f, dot = 0.f;
      #pragma unroll
      for (int i = 0; i < kMaxDim / 64; ++i) {
        const int e = lane + 64 * i;
        if (e >= a.dim) continue;
        float v = mine[e];
        if (e < 2 * a.half) {
          const float2 cs = angle(a, at.token, at.in_seq, pair_of(a, e));
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

// ---------------------------------------------------------------------------
// Rows in registers: G lanes hold a row, 8 values each, so a wave works on
// 64 / G heads of one token at a time and goes through the token's heads of
// queries, then keys.  The angles and positions of a token are read once.
// Needs D in eights and pairs in fours (see fits()), but no alignment.
//
// Bound by memory: 16384 tokens of 32 + 8 heads of 128 in bf16 take 58 us
// forward (336 MB, 5.8 TB/s) and 86 + 5 us backward (503 MB, 5.8 TB/s), with
// halves 59 and 90 + 5 us.
// Heads of more than elem::kCached are written past the caches (NT): through
// them 66 against 58 us and 110 against 90 us.  The backward keeps dw in
// registers over all rows of a wave; 1024 blocks hide its latency (512: 126
// against 90 us), more of them only lengthen the sum over blocks (4096: 10
// us), and reading a head ahead gained nothing.
constexpr int kRun = 8;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(
      __builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 15, 15, true));
}

// Sum over the G lanes of a row; every lane gets it.
template <int G>
__device__ __forceinline__ float row_sum(float v) {
  v += dpp<0xB1>(v);                // lane ^ 1
  v += dpp<0x4E>(v);                // lane ^ 2
  v += dpp<0x141>(v);               // mirror in 8: the other quad
  if (G >= 16) v += dpp<0x140>(v);  // mirror in 16: the other 8
  if (G >= 32) v += __shfl_xor(v, 16);
  if (G >= 64) v += __shfl_xor(v, 32);
  return v;
}

// What a lane holds of every row: four pairs from p on, or, behind the
// rotated part, eight values that do not turn.  Interleaved pairs are the 8
// values from `a` on; with halves the first values of the pairs are the 4
// from `a` on and the second those from `b` on, so that no lane needs
// another's values.
struct Lane {
  int a, b, p;
  bool on, turns;
};

template <int G, bool INTER>
__device__ __forceinline__ Lane lane_of(const Args& args) {
  const int sub = threadIdx.x % G, turning = args.half / 4;
  Lane l;
  l.turns = sub < turning;
  l.p = 4 * sub;
  l.a = kRun * sub;
  l.b = l.a + 4;
  if (!INTER && l.turns) {
    l.a = l.p;
    l.b = l.p + args.half;
  }
  l.on = kRun * sub < args.dim;
  return l;
}

// The first and second values of a lane's pairs.
struct Pairs {
  float a[4], b[4];
};

template <typename T, bool INTER>
__device__ __forceinline__ Pairs load(const Lane& l, const T* row) {
  Pairs v;
  if (INTER) {
    const auto w = elem::load<false, kRun>(row + l.a);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.a[i] = (float)w[2 * i];
      v.b[i] = (float)w[2 * i + 1];
    }
  } else {
    const auto wa = elem::load<false, 4>(row + l.a);
    const auto wb = elem::load<false, 4>(row + l.b);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.a[i] = (float)wa[i];
      v.b[i] = (float)wb[i];
    }
  }
  return v;
}

template <typename T, bool INTER, bool NT>
__device__ __forceinline__ void store(const Lane& l, T* row, const Pairs& v) {
  if (INTER) {
    elem::vec<T, kRun> w;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[2 * i] = (T)v.a[i];
      w[2 * i + 1] = (T)v.b[i];
    }
    elem::store<NT, kRun>(row + l.a, w);
  } else {
    elem::vec<T, 4> wa, wb;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      wa[i] = (T)v.a[i];
      wb[i] = (T)v.b[i];
    }
    elem::store<NT, 4>(row + l.a, wa);
    elem::store<NT, 4>(row + l.b, wb);
  }
}

// Place of a lane's i-th pair in the row.
template <bool INTER>
__device__ __forceinline__ int first_at(const Lane& l, int i) {
  return INTER ? l.a + 2 * i : l.a + i;
}
template <bool INTER>
__device__ __forceinline__ int second_at(const Lane& l, int i) {
  return INTER ? l.a + 2 * i + 1 : l.b + i;
}

// Where the rows of the tables that a token's axes take begin; negative
// outside the tables.  The same for all lanes of a wave.
struct Starts {
  long at[kMaxAxes];
};

__device__ __forceinline__ Starts starts(const Args& a, long token,
                                         long in_seq) {
  Starts r;
  #pragma unroll
  for (int i = 0; i < kMaxAxes; ++i) {
    r.at[i] = -1;
    if (i >= a.axes) continue;
    const long at = a.pos ? a.pos[i * a.tokens + token] : in_seq;
    r.at[i] = at >= 0 && at < a.table ? at * a.half : -1;
  }
  return r;
}

// Sections of pairs follow each other.
__device__ __forceinline__ int axis_of(const Args& a, int p) {
  int axis = 0;
  #pragma unroll
  for (int i = 0; i + 1 < kMaxAxes; ++i)
    axis += i + 1 < a.axes && p >= a.ends[i];
  return axis;
}

// Chosen by the pair, not by the axis' number: an array indexed by a register
// would be laid out in shared memory (72 instead of 58 us at the size above).
__device__ __forceinline__ long start_of(const Args& a, const Starts& t,
                                         int p) {
  long at = t.at[0];
  #pragma unroll
  for (int i = 1; i < kMaxAxes; ++i)
    if (i < a.axes && p >= a.ends[i - 1]) at = t.at[i];
  return at;
}

// Cosines and sines of a lane's pairs; the identity where nothing turns.
struct Angles {
  float c[4], s[4];
};

__device__ __forceinline__ Angles angles(const Args& a, const Lane& l,
                                         const Starts& t) {
  const float nan = __uint_as_float(0x7fc00000);
  Angles r;
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.c[i] = 1.f;
    r.s[i] = 0.f;
  }
  if (!l.turns) return r;
  if (axis_of(a, l.p) == axis_of(a, l.p + 3)) {
    const long at = start_of(a, t, l.p);
    if (at < 0) {
      #pragma unroll
      for (int i = 0; i < 4; ++i) r.c[i] = r.s[i] = nan;
      return r;
    }
    const auto c = elem::load<false, 4>(a.cosines + at + l.p);
    const auto s = elem::load<false, 4>(a.sines + at + l.p);
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.c[i] = c[i];
      r.s[i] = s[i];
    }
    return r;
  }
  // on more than one axis
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long from = start_of(a, t, l.p + i);
    r.c[i] = from < 0 ? nan : a.cosines[from + l.p + i];
    r.s[i] = from < 0 ? nan : a.sines[from + l.p + i];
  }
  return r;
}

// Weights of a lane's values, zeros for a lane behind the row.
template <typename T, bool INTER>
__device__ __forceinline__ Pairs weights(const Args& a, const Side& s,
                                         const Lane& l) {
  if (l.on && s.w)
    return a.w_fp32 ? load<float, INTER>(l, (const float*)s.w)
                    : load<T, INTER>(l, (const T*)s.w);
  Pairs w;
  #pragma unroll
  for (int i = 0; i < 4; ++i) w.a[i] = w.b[i] = l.on ? 1.f : 0.f;
  return w;
}

// The wave's number, known to be the same for its lanes: what follows from it
// is computed and loaded once.
__device__ __forceinline__ int wave_no() {
  return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
}

// Work of a wave: the heads [h0, h1) of a token, queries before keys.
struct Item {
  long token, seq_no, in_seq;
  int h0, h1;
};

__device__ __forceinline__ Item item_of(const Args& a, long item, int chunks,
                                        int per) {
  Item it;
  it.token = item / chunks;
  it.h0 = (int)(item % chunks) * per;
  it.h1 = min(it.h0 + per, a.side[0].heads + a.side[1].heads);
  it.seq_no = it.token / a.seq;
  it.in_seq = it.token % a.seq;
  return it;
}

template <typename T, int G, bool INTER, bool NT>
__device__ __forceinline__ void fwd_side(const Args& a, const Side& s,
                                         const Lane& l, const Item& it,
                                         int h0, int h1, const Pairs& w,
                                         const Angles& t) {
  const int group = (threadIdx.x & 63) / G;
  const T* x = (const T*)s.x + it.seq_no * s.sb + it.in_seq * s.ss;
  T* y = (T*)s.y + it.token * s.heads * a.dim;
  const float inv_dim = 1.f / (float)a.dim;
  for (int h = h0 + group; h < h1; h += 64 / G) {
    Pairs v = {};
    if (l.on) v = load<T, INTER>(l, x + h * s.sh);
    float sum = 0.f;
    #pragma unroll
    for (int i = 0; i < 4; ++i) sum += v.a[i] * v.a[i] + v.b[i] * v.b[i];
    const float r =
        __builtin_amdgcn_rsqf(row_sum<G>(sum) * inv_dim + a.eps);
    Pairs o;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = v.a[i] * r * w.a[i], q = v.b[i] * r * w.b[i];
      o.a[i] = p * t.c[i] - q * t.s[i];
      o.b[i] = q * t.c[i] + p * t.s[i];
    }
    if (l.on) store<T, INTER, NT>(l, y + (long)h * a.dim, o);
  }
}

template <typename T, int G, bool INTER, bool NT>
__global__ __launch_bounds__(kThreads) void fwd_rows_kernel(Args a,
                                                            int chunks,
                                                            int per) {
  const Lane l = lane_of<G, INTER>(a);
  const int hq = a.side[0].heads;
  const Pairs wq = weights<T, INTER>(a, a.side[0], l);
  const Pairs wk = weights<T, INTER>(a, a.side[1], l);
  const long items = a.tokens * chunks;
  for (long i = (long)blockIdx.x * kWaves + wave_no(); i < items;
       i += (long)gridDim.x * kWaves) {
    const Item it = item_of(a, i, chunks, per);
    const Angles t = angles(a, l, starts(a, it.token, it.in_seq));
    fwd_side<T, G, INTER, NT>(a, a.side[0], l, it, it.h0, min(it.h1, hq), wq,
                              t);
    fwd_side<T, G, INTER, NT>(a, a.side[1], l, it, max(it.h0 - hq, 0),
                              it.h1 - hq, wk, t);
  }
}

template <typename T, int G, bool INTER, bool NT>
__device__ __forceinline__ void bwd_side(const Args& a, const Side& s,
                                         const Lane& l, const Item& it,
                                         int h0, int h1, const Pairs& w,
                                         Pairs& dw, const Angles& t) {
  const int group = (threadIdx.x & 63) / G;
  const T* x = (const T*)s.x + it.seq_no * s.sb + it.in_seq * s.ss;
  const T* dy = (const T*)s.dy + it.seq_no * s.db + it.in_seq * s.ds;
  T* dx = (T*)s.y + it.token * s.heads * a.dim;
  const float inv_dim = 1.f / (float)a.dim;
  for (int h = h0 + group; h < h1; h += 64 / G) {
    Pairs v = {}, d = {}, n;
    if (l.on) {
      v = load<T, INTER>(l, x + h * s.sh);
      d = load<T, INTER>(l, dy + h * s.dh);
    }
    float sum = 0.f, dot = 0.f;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      n.a[i] = d.a[i] * t.c[i] + d.b[i] * t.s[i];
      n.b[i] = d.b[i] * t.c[i] - d.a[i] * t.s[i];
      sum += v.a[i] * v.a[i] + v.b[i] * v.b[i];
      dot += n.a[i] * w.a[i] * v.a[i] + n.b[i] * w.b[i] * v.b[i];
    }
    const float r =
        __builtin_amdgcn_rsqf(row_sum<G>(sum) * inv_dim + a.eps);
    const float k = row_sum<G>(dot) * inv_dim * r * r;
    Pairs o;
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      o.a[i] = r * (n.a[i] * w.a[i] - v.a[i] * k);
      o.b[i] = r * (n.b[i] * w.b[i] - v.b[i] * k);
      dw.a[i] += n.a[i] * v.a[i] * r;
      dw.b[i] += n.b[i] * v.b[i] * r;
    }
    if (l.on) store<T, INTER, NT>(l, dx + (long)h * a.dim, o);
  }
}

// partial[block]: dw of the queries, then of the keys.
template <typename T, int G, bool INTER, bool NT>
__global__ __launch_bounds__(kThreads) void bwd_rows_kernel(
    Args a, int chunks, int per, float* __restrict__ partial) {
  const Lane l = lane_of<G, INTER>(a);
  const int hq = a.side[0].heads, wave = wave_no();
  const Pairs wq = weights<T, INTER>(a, a.side[0], l);
  const Pairs wk = weights<T, INTER>(a, a.side[1], l);
  Pairs dw[2] = {};
  const long items = a.tokens * chunks;
  for (long i = (long)blockIdx.x * kWaves + wave; i < items;
       i += (long)gridDim.x * kWaves) {
    const Item it = item_of(a, i, chunks, per);
    const Angles t = angles(a, l, starts(a, it.token, it.in_seq));
    bwd_side<T, G, INTER, NT>(a, a.side[0], l, it, it.h0, min(it.h1, hq), wq,
                              dw[0], t);
    bwd_side<T, G, INTER, NT>(a, a.side[1], l, it, max(it.h0 - hq, 0),
                              it.h1 - hq, wk, dw[1], t);
  }
  if (!partial) return;
  // over the wave's groups, then over the block's waves
  __shared__ float sums[kWaves][2][G * kRun];
  #pragma unroll
  for (int side = 0; side < 2; ++side)
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      float va = dw[side].a[i], vb = dw[side].b[i];
      #pragma unroll
      for (int off = G; off < 64; off *= 2) {
        va += __shfl_xor(va, off);
        vb += __shfl_xor(vb, off);
      }
      if ((threadIdx.x & 63) < G) {
        sums[wave][side][first_at<INTER>(l, i)] = va;
        sums[wave][side][second_at<INTER>(l, i)] = vb;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * a.dim; i += kThreads) {
    const int side = i >= a.dim, e = side ? i - a.dim : i;
    float v = 0.f;
    #pragma unroll
    for (int wv = 0; wv < kWaves; ++wv) v += sums[wv][side][e];
    partial[(long)blockIdx.x * 2 * a.dim + i] = v;
  }
}

// dw of both sides from the blocks' sums, added in a fixed order: a block
// for 8 columns, 32 threads a column.
template <typename T>
__global__ __launch_bounds__(kThreads) void dw_rows_kernel(
    const float* __restrict__ partial, void* dwq, void* dwk, int blocks,
    int dim, bool fp32) {
  __shared__ double sums[kThreads];
  const int col = blockIdx.x * 8 + (threadIdx.x & 7);
  double v = 0.;
  if (col < 2 * dim) {
    #pragma unroll 8
    for (int b = threadIdx.x >> 3; b < blocks; b += kThreads / 8)
      v += (double)partial[(long)b * 2 * dim + col];
  }
  sums[threadIdx.x] = v;
  for (int half = kThreads / 2; half >= 8; half /= 2) {
    __syncthreads();
    if ((int)threadIdx.x < half)
      sums[threadIdx.x] += sums[threadIdx.x + half];
  }
  if (threadIdx.x >= 8 || col >= 2 * dim) return;
  const int e = col < dim ? col : col - dim;
  void* out = col < dim ? dwq : dwk;
  if (!out) return;
  const float sum = (float)sums[threadIdx.x];
  if (fp32) ((float*)out)[e] = sum;
  else ((T*)out)[e] = (T)sum;
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

void fill_side(Side& s, const at::Tensor& x,
               const at::Tensor& w, at::Tensor& y) {
  s.x = x.data_ptr();
  s.dy = nullptr;
  s.db = s.ds = s.dh = 0;
  s.y = y.data_ptr();
  s.w = w.defined() ? w.data_ptr() : nullptr;
  s.sb = x.stride(0);
  s.ss = x.stride(1);
  s.sh = x.stride(2);
  s.heads = (int)x.size(2);
}

// What a call does besides its tensors.
struct Mode {
  std::vector<int64_t> sections;  // empty: one axis
  double eps;
  bool interleaved;
};

// The tensors of a call as the kernels take them: heads with a unit last
// stride, weights, tables and positions contiguous.
struct Tensors {
  at::Tensor q, k, wq, wk, cosines, sines, pos;  // undefined where absent
};

Args make_args(const Tensors& t, const Mode& m, at::Tensor& yq,
               at::Tensor& yk) {
  Args a;
  a.tokens = t.q.size(0) * t.q.size(1);
  a.seq = std::max<long>(1, t.q.size(1));
  a.dim = (int)t.q.size(3);
  a.table = t.cosines.size(0);
  a.half = (int)t.cosines.size(1);
  a.cosines = t.cosines.data_ptr<float>();
  a.sines = t.sines.data_ptr<float>();
  a.axes = std::max<int>(1, (int)m.sections.size());
  int end = 0;
  for (int i = 0; i < kMaxAxes; ++i) {
    if (i < (int)m.sections.size()) end += (int)m.sections[i];
    else end = a.half;
    a.ends[i] = end;
  }
  a.pos = t.pos.defined() ? t.pos.data_ptr<long>() : nullptr;
  a.w_fp32 = (t.wq.defined() && t.wq.scalar_type() == at::kFloat) ||
             (t.wk.defined() && t.wk.scalar_type() == at::kFloat);
  a.interleaved = m.interleaved;
  a.eps = (float)m.eps;
  fill_side(a.side[0], t.q, t.wq, yq);
  fill_side(a.side[1], t.k, t.wk, yk);
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

// Whether the kernels with rows in registers take the call.
bool fits(const Args& a) {
  return a.dim % kRun == 0 && a.dim <= 64 * kRun && a.half % 4 == 0;
}

// Heads of a wave: all of a token's where the tokens alone fill the chip,
// else so few that the waves do.
void divide(const Args& a, int lanes, int& chunks, int& per) {
  const int at_once = 64 / lanes;
  const long heads = a.side[0].heads + a.side[1].heads;
  const long most = (heads + at_once - 1) / at_once;
  const long want = (8192 + a.tokens - 1) / a.tokens;
  const long n = std::min(want, most);
  per = (int)((most + n - 1) / n * at_once);
  chunks = (int)((heads + per - 1) / per);
}

// Calls f with the lanes of a row, the pair layout and the way to memory as
// constants.
template <typename F>
void with_layout(const Args& a, size_t size, F f) {
  const long bytes = a.tokens * (a.side[0].heads + a.side[1].heads) * a.dim *
                     (long)size;
  const auto cached = [&](auto lanes, auto inter) {
    if (bytes > elem::kCached) f(lanes, inter, std::true_type{});
    else f(lanes, inter, std::false_type{});
  };
  const auto layout = [&](auto lanes) {
    if (a.interleaved) cached(lanes, std::true_type{});
    else cached(lanes, std::false_type{});
  };
  if (a.dim <= 8 * kRun) layout(std::integral_constant<int, 8>{});
  else if (a.dim <= 16 * kRun) layout(std::integral_constant<int, 16>{});
  else if (a.dim <= 32 * kRun) layout(std::integral_constant<int, 32>{});
  else layout(std::integral_constant<int, 64>{});
}

// Rows with a unit stride inside, whatever the strides between them.
at::Tensor unit_stride(const at::Tensor& x) {
  return x.size(3) > 1 && x.stride(3) != 1 ? x.contiguous() : x;
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

variable_list forward_of(const Tensors& t, const Mode& m) {
  const c10::DeviceGuard guard(t.q.device());
  auto yq = at::empty(t.q.sizes(), t.q.options());
  auto yk = at::empty(t.k.sizes(), t.k.options());
  const Args a = make_args(t, m, yq, yk);
  if (a.tokens * (a.side[0].heads + a.side[1].heads) == 0) return {yq, yk};
  STOKE_ELEM_SWITCH(t.q.scalar_type(), "qk_norm_rope", {
    if (fits(a)) {
      with_layout(a, sizeof(T), [&](auto lanes, auto inter, auto nt) {
        int chunks, per;
        divide(a, lanes, chunks, per);
        const long blocks = (a.tokens * chunks + kWaves - 1) / kWaves;
        hipLaunchKernelGGL((fwd_rows_kernel<T, lanes, inter, nt>),
                           dim3((unsigned)std::min(blocks, 1L << 20)),
                           dim3(kThreads), 0, elem::stream(), a, chunks, per);
      });
    } else {
      int q_blocks, blocks;
      share(a, 65536, q_blocks, blocks);
      hipLaunchKernelGGL((fwd_any_kernel<T>), dim3((unsigned)blocks),
                         dim3(kThreads), kWaves * a.dim * sizeof(float),
                         elem::stream(), a, q_blocks);
    }
  });
  return {yq, yk};
}

// (dq, dk, dwq, dwk); the last two undefined where there is no weight.
variable_list backward_of(const Tensors& t, const Mode& m,
                          const at::Tensor& dyq, const at::Tensor& dyk) {
  const c10::DeviceGuard guard(t.q.device());
  auto dq = at::empty(t.q.sizes(), t.q.options());
  auto dk = at::empty(t.k.sizes(), t.k.options());
  Args a = make_args(t, m, dq, dk);
  for (const int i : {0, 1}) {
    const at::Tensor& dy = i ? dyk : dyq;
    Side& s = a.side[i];
    s.dy = dy.data_ptr();
    s.db = dy.stride(0);
    s.ds = dy.stride(1);
    s.dh = dy.stride(2);
  }
  at::Tensor dwq, dwk;
  if (t.wq.defined()) dwq = at::empty(t.wq.sizes(), t.wq.options());
  if (t.wk.defined()) dwk = at::empty(t.wk.sizes(), t.wk.options());
  if (a.tokens * (a.side[0].heads + a.side[1].heads) == 0) {
    if (dwq.defined()) dwq.zero_();
    if (dwk.defined()) dwk.zero_();
    return {dq, dk, dwq, dwk};
  }
  void* out_q = dwq.defined() ? dwq.data_ptr() : nullptr;
  void* out_k = dwk.defined() ? dwk.data_ptr() : nullptr;
  const bool sums = dwq.defined() || dwk.defined();
  const auto f32 = t.q.options().dtype(at::kFloat);
  STOKE_ELEM_SWITCH(t.q.scalar_type(), "qk_norm_rope", {
    if (fits(a)) {
      with_layout(a, sizeof(T), [&](auto lanes, auto inter, auto nt) {
        int chunks, per;
        divide(a, lanes, chunks, per);
        const long blocks =
            std::min((a.tokens * chunks + kWaves - 1) / kWaves, 1024L);
        at::Tensor partial;
        if (sums) partial = at::empty({blocks, 2 * a.dim}, f32);
        hipLaunchKernelGGL((bwd_rows_kernel<T, lanes, inter, nt>),
                           dim3((unsigned)blocks), dim3(kThreads), 0,
                           elem::stream(), a, chunks, per,
                           sums ? partial.data_ptr<float>() : nullptr);
        if (sums)
          hipLaunchKernelGGL((dw_rows_kernel<T>),
                             dim3((unsigned)(2 * a.dim + 7) / 8),
                             dim3(kThreads), 0, elem::stream(),
                             partial.data_ptr<float>(), out_q, out_k,
                             (int)blocks, a.dim, a.w_fp32);
      });
    } else {
      int q_blocks, blocks;
      share(a, 2048, q_blocks, blocks);
      auto partial = at::empty({blocks, a.dim}, f32);
      hipLaunchKernelGGL((bwd_any_kernel<T>), dim3((unsigned)blocks),
                         dim3(kThreads), 2 * kWaves * a.dim * sizeof(float),
                         elem::stream(), a, q_blocks,
                         partial.data_ptr<float>());
      if (sums)
        hipLaunchKernelGGL((dw_kernel<T>), dim3((a.dim + 15) / 16, 2),
                           dim3(kThreads), 0, elem::stream(),
                           partial.data_ptr<float>(), out_q, out_k, q_blocks,
                           blocks, a.dim, a.w_fp32);
    }
  });
  return {dq, dk, dwq, dwk};
}

struct QKNormRope : torch::autograd::Function<QKNormRope> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q,
                               const at::Tensor& k,
                               const std::optional<at::Tensor>& wq,
                               const std::optional<at::Tensor>& wk,
                               const Tensors& t, const Mode& m) {
    ctx->save_for_backward({q, k, wq.value_or(at::Tensor()),
                            wk.value_or(at::Tensor()), t.cosines, t.sines,
                            t.pos});
    ctx->saved_data["sections"] = m.sections;
    ctx->saved_data["eps"] = m.eps;
    ctx->saved_data["interleaved"] = m.interleaved;
    return forward_of(t, m);
  }

  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto v = ctx->get_saved_variables();
    const Tensors t{v[0], v[1], v[2], v[3], v[4], v[5], v[6]};
    const Mode m{ctx->saved_data["sections"].toIntVector(),
                 ctx->saved_data["eps"].toDouble(),
                 ctx->saved_data["interleaved"].toBool()};
    const auto d = backward_of(t, m, unit_stride(dy[0]), unit_stride(dy[1]));
    variable_list out(6);
    std::copy(d.begin(), d.end(), out.begin());
    return elem::once_differentiable(std::move(out));
  }
};

void check(const at::Tensor& q, const at::Tensor& k, const at::Tensor& wq,
           const at::Tensor& wk, const at::Tensor& cosines,
           const at::Tensor& sines, const std::optional<at::Tensor>& pos,
           const std::optional<std::vector<int64_t>>& sections) {
  TORCH_CHECK_VALUE(
      q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) &&
          q.size(1) == k.size(1) && q.size(3) == k.size(3) &&
          q.scalar_type() == k.scalar_type() && q.is_cuda() &&
          q.device() == k.device() &&
          (q.scalar_type() == at::kBFloat16 ||
           q.scalar_type() == at::kHalf || q.scalar_type() == at::kFloat) &&
          q.size(3) >= 1 && q.size(3) <= kMaxDim,
      "Stoke -- qk_norm_rope takes q [B, S, H, D] and k [B, S, Hk, D] of one "
      "floating dtype and device, D up to ", kMaxDim, ", got ", q.sizes(),
      " ", q.scalar_type(), " and ", k.sizes(), " ", k.scalar_type());
  for (const at::Tensor& w : {wq, wk})
    TORCH_CHECK_VALUE(
        !w.defined() ||
            (w.dim() == 1 && w.size(0) == q.size(3) &&
             w.device() == q.device() &&
             (w.scalar_type() == at::kFloat ||
              w.scalar_type() == q.scalar_type())),
        "Stoke -- qk_norm_rope weights are [", q.size(3), "] in fp32 or ",
        q.scalar_type());
  TORCH_CHECK_VALUE(!wq.defined() || !wk.defined() ||
                        wq.scalar_type() == wk.scalar_type(),
                    "Stoke -- qk_norm_rope weights have one dtype");
  TORCH_CHECK_VALUE(
      cosines.dim() == 2 && cosines.sizes() == sines.sizes() &&
          cosines.device() == q.device() && sines.device() == q.device() &&
          cosines.is_floating_point() && sines.is_floating_point() &&
          2 * cosines.size(1) <= q.size(3) && !cosines.requires_grad() &&
          !sines.requires_grad(),
      "Stoke -- qk_norm_rope takes constant tables cos, sin [P, <= D / 2], "
      "got ", cosines.sizes(), " and ", sines.sizes());
  int64_t axes = 1;
  if (sections) {
    axes = (int64_t)sections->size();
    int64_t sum = 0;
    bool fine = axes >= 1 && axes <= kMaxAxes;
    for (const int64_t n : *sections) {
      fine = fine && n >= 0 && n <= cosines.size(1);
      sum += fine ? n : 0;
    }
    TORCH_CHECK_VALUE(fine && sum == cosines.size(1),
                      "Stoke -- sections are 1 to ", kMaxAxes,
                      " numbers of pairs that add up to ", cosines.size(1),
                      ", got ", *sections);
  }
  if (!pos) {
    TORCH_CHECK_VALUE(axes == 1 && cosines.size(0) >= q.size(1),
                      "Stoke -- without positions there is one axis and the "
                      "tables cover the sequence (", cosines.size(0),
                      " rows for ", q.size(1), ")");
    return;
  }
  const int64_t lead = sections ? 1 : 0;
  bool fine = (pos->scalar_type() == at::kLong ||
               pos->scalar_type() == at::kInt) &&
              pos->device() == q.device() && pos->dim() == lead + 2 &&
              (!lead || pos->size(0) == axes);
  for (int64_t i = 0; fine && i < 2; ++i)
    fine = pos->size(lead + i) == 1 || pos->size(lead + i) == q.size(i);
  TORCH_CHECK_VALUE(fine,
                    "Stoke -- positions are whole numbers [axes with "
                    "sections, B, S] (B and S of 1 broadcast) on the heads' "
                    "device, got ", pos->sizes(), " ", pos->scalar_type());
}

at::Tensor table32(const at::Tensor& x) {
  return x.scalar_type() == at::kFloat ? x.contiguous()
                                       : x.to(at::kFloat).contiguous();
}

}  // namespace

// The entry point: checks its arguments, and has gradients for the heads and
// the weights.
std::vector<at::Tensor> qk_norm_rope(
    at::Tensor q, at::Tensor k, std::optional<at::Tensor> wq,
    std::optional<at::Tensor> wk, at::Tensor cosines, at::Tensor sines,
    std::optional<at::Tensor> pos,
    std::optional<std::vector<int64_t>> sections, double eps,
    bool interleaved) {
  elem::refuse_tangents("qk_norm_rope", q, k, wq, wk, cosines, sines);
  Tensors t;
  if (wq) t.wq = wq->contiguous();
  if (wk) t.wk = wk->contiguous();
  check(q, k, t.wq, t.wk, cosines, sines, pos, sections);
  t.q = unit_stride(q);
  t.k = unit_stride(k);
  t.cosines = table32(cosines);
  t.sines = table32(sines);
  if (pos) {
    t.pos = pos->scalar_type() == at::kLong ? *pos : pos->to(at::kLong);
    std::vector<int64_t> want = t.pos.sizes().vec();
    want[want.size() - 2] = q.size(0);
    want[want.size() - 1] = q.size(1);
    if (t.pos.sizes() != at::IntArrayRef(want)) t.pos = t.pos.expand(want);
    t.pos = t.pos.contiguous();
  }
  const Mode m{sections.value_or(std::vector<int64_t>()), eps, interleaved};
  const bool grad =
      at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() ||
       (t.wq.defined() && t.wq.requires_grad()) ||
       (t.wk.defined() && t.wk.requires_grad()));
  if (!grad) return forward_of(t, m);
  elem::check_capture({q, k, wq.value_or(at::Tensor()),
                       wk.value_or(at::Tensor())});
  // variables among the arguments are found as tensors of their own
  return QKNormRope::apply(
      t.q, t.k, wq ? std::optional<at::Tensor>(t.wq) : std::nullopt,
      wk ? std::optional<at::Tensor>(t.wk) : std::nullopt, t, m);
}
