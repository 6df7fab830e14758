// Root-mean-square norm of every head of q and k with the position rotation of the result, in
// one pass over both tensors, and its gradient.
//
//   r = (mean(x^2) + eps)^(-1/2),  n = x r w,  y = n with its first R elements turned by the
//   token's angles: (a, b) -> (a cos - b sin, a sin + b cos) on the pairs (2i, 2i + 1)
//   (interleaved) or (i, i + R / 2).
// Backward, with g = dy turned by the opposite angles and x^ = x r:
//   dw = sum over rows of g x^,   dx = r (g w - x^ mean(g w x^)).
//
// Both are bound by memory: 2 (3 backward) passes over the elements against about 6 (14)
// operations per element. A row (one head of one token) lies in a group of GL lanes, 8
// elements per lane, so every access is 16 bytes per lane and the row sums are shuffles
// inside the group; the rotation's partner element is in the same lane (interleaved) or in the lane
// R / 16 further (halves). A warp takes a run of ROWS * 32 / GL heads of one token: the run's
// loads are all in flight before the first sum, and the token's angles are read once per run.
// All arithmetic is in 32 bits and rounded once, when y (dx) is stored.
#include "common.cuh"
#include "norm_rope.cuh"

#include <cuda_fp16.h>

namespace solb200 {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRowsFwd = 4, kRowsBwd = 2;   // rows per lane group in flight

template <typename T>
struct Vec8;   // 8 elements of a row as they lie in memory

template <>
struct Vec8<float> {
  float4 a, b;
  __device__ void load(const float* p) { a = __ldg(reinterpret_cast<const float4*>(p)); b = __ldg(reinterpret_cast<const float4*>(p) + 1); }
  __device__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  static __device__ void store(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

template <typename T>
struct Vec8 {   // 16-bit types
  uint4 w;
  __device__ void load(const T* p) { w = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ void zero() { w = make_uint4(0, 0, 0, 0); }
  static __device__ float2 widen(uint32_t u);
  static __device__ uint32_t narrow(float lo, float hi);
  __device__ void get(float (&f)[8]) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = widen(u[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ void store(T* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(narrow(f[0], f[1]), narrow(f[2], f[3]), narrow(f[4], f[5]),
                                              narrow(f[6], f[7]));
  }
};

template <>
__device__ __forceinline__ float2 Vec8<__nv_bfloat16>::widen(uint32_t u) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
}
template <>
__device__ __forceinline__ uint32_t Vec8<__nv_bfloat16>::narrow(float lo, float hi) {
  return pack_bf16x2(lo, hi);
}
template <>
__device__ __forceinline__ float2 Vec8<__half>::widen(uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <>
__device__ __forceinline__ uint32_t Vec8<__half>::narrow(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int GL>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The rotation of a lane's 8 elements. A lane past R turns by the angle 0.
template <bool INTER>
struct Turn {
  float c[INTER ? 4 : 8], s[INTER ? 4 : 8];   // halves: s carries the pair's sign
  int src;                                    // halves: the lane that holds the partner elements

  __device__ void load(const RopeParams& p, int64_t b, int64_t t, int lg, int lane) {
    const int64_t off = b * p.ts[0] + t * p.ts[1];
    const bool in = lg * 8 < p.R;
    src = lane;
    int col = lg * 4;
    if (!INTER) {
      const int half = p.R >> 1;
      const bool second = lg * 8 >= half;
      col = second ? lg * 8 - half : lg * 8;
      if (in) src = second ? lane - (p.R >> 4) : lane + (p.R >> 4);
    }
#pragma unroll
    for (int i = 0; i < (INTER ? 1 : 2); ++i) {
      float4 vc = make_float4(1.f, 1.f, 1.f, 1.f), vs = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in) {
        vc = __ldg(reinterpret_cast<const float4*>(p.cos + off + col) + i);
        vs = __ldg(reinterpret_cast<const float4*>(p.sin + off + col) + i);
      }
      const float sg = (!INTER && lg * 8 < (p.R >> 1)) ? -1.f : 1.f;
      c[4 * i] = vc.x; c[4 * i + 1] = vc.y; c[4 * i + 2] = vc.z; c[4 * i + 3] = vc.w;
      s[4 * i] = sg * vs.x; s[4 * i + 1] = sg * vs.y; s[4 * i + 2] = sg * vs.z; s[4 * i + 3] = sg * vs.w;
    }
  }

  // BACK: by the opposite angle. Warp-collective (halves exchange partners by shuffles).
  template <bool BACK>
  __device__ void apply(float (&f)[8]) const {
    if (INTER) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float a = f[2 * i], b = f[2 * i + 1], si = BACK ? -s[i] : s[i];
        f[2 * i] = a * c[i] - b * si;
        f[2 * i + 1] = fmaf(a, si, b * c[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float other = __shfl_sync(0xffffffffu, f[i], src);
        f[i] = fmaf(f[i], c[i], other * (BACK ? -s[i] : s[i]));
      }
    }
  }
};

// Item -> tensor (0 q, 1 k), first head of its run, batch and token.
struct RopeItem {
  int which, head0;
  int64_t b, t;
  __device__ RopeItem(const RopeParams& p, int64_t item, int heads_per_item) {
    const int per = p.chunks[0] + p.chunks[1];
    const int64_t bt = item / per;
    const int c = (int)(item - bt * per);
    which = c >= p.chunks[0];
    head0 = (which ? c - p.chunks[0] : c) * heads_per_item;
    b = bt / p.T;
    t = bt - b * p.T;
  }
};

template <typename T>
__device__ __forceinline__ float weight_at(const void* w, int wdtype, int d) {
  return wdtype == kDtypeF32 ? __ldg(static_cast<const float*>(w) + d) : (float)static_cast<const T*>(w)[d];
}

template <typename T, int GL, bool INTER>
__global__ void __launch_bounds__(kRopeThreads)
norm_rope_kernel(const __grid_constant__ RopeParams p, int wdtype) {
  pdl_begin();
  constexpr int GPW = 32 / GL, HPI = GPW * kRowsFwd;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lg = lane % GL, grp = lane / GL;
  const bool in = lg * 8 < p.D;
  const int64_t stride = (int64_t)gridDim.x * (kRopeThreads / 32);
  const float inv_d = 1.f / (float)p.D;
  for (int64_t item = (int64_t)blockIdx.x * (kRopeThreads / 32) + warp; item < p.items; item += stride) {
    const RopeItem it(p, item, HPI);
    const RopeTensor& x = p.t[it.which];
    const T* src = static_cast<const T*>(x.x) + it.b * x.xs[0] + it.t * x.xs[1] + lg * 8;
    Vec8<T> v[kRowsFwd];
#pragma unroll
    for (int r = 0; r < kRowsFwd; ++r) {
      const int h = it.head0 + r * GPW + grp;
      if (in && h < x.heads) v[r].load(src + h * x.xs[2]);
      else v[r].zero();
    }
    Turn<INTER> turn;
    turn.load(p, it.b, it.t, lg, lane);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = in ? weight_at<T>(x.weight, wdtype, lg * 8 + i) : 0.f;
    T* dst = static_cast<T*>(x.out) + ((it.b * p.T + it.t) * x.heads) * p.D + lg * 8;
#pragma unroll
    for (int r = 0; r < kRowsFwd; ++r) {
      float f[8];
      v[r].get(f);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
      const float rstd = rsqrtf(fmaf(group_sum<GL>(ss), inv_d, p.eps));
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * rstd * w[i];
      turn.template apply<false>(f);
      const int h = it.head0 + r * GPW + grp;
      if (in && h < x.heads) Vec8<T>::store(dst + (int64_t)h * p.D, f);
    }
  }
}

// Every CTA walks the items with a stride and keeps its lanes' sums of the weight gradients in
// registers; they are joined over the CTA in a fixed order and written as one row of
// p.partial, which weight_grad_kernel adds up, again in a fixed order: no atomics, the same
// result every time.
template <typename T, int GL, bool INTER>
__global__ void __launch_bounds__(kRopeThreads)
norm_rope_backward_kernel(const __grid_constant__ RopeParams p, int wdtype) {
  pdl_begin();
  constexpr int GPW = 32 / GL, HPI = GPW * kRowsBwd, WARPS = kRopeThreads / 32;
  __shared__ float sums[WARPS][2][GL * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lg = lane % GL, grp = lane / GL;
  const bool in = lg * 8 < p.D;
  const int64_t stride = (int64_t)gridDim.x * WARPS;
  const float inv_d = 1.f / (float)p.D;
  float acc[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[0][i] = acc[1][i] = 0.f;
  for (int64_t item = (int64_t)blockIdx.x * WARPS + warp; item < p.items; item += stride) {
    const RopeItem it(p, item, HPI);
    const RopeTensor& x = p.t[it.which];
    const T* xsrc = static_cast<const T*>(x.x) + it.b * x.xs[0] + it.t * x.xs[1] + lg * 8;
    const T* gsrc = static_cast<const T*>(x.dy) + it.b * x.dys[0] + it.t * x.dys[1] + lg * 8;
    Vec8<T> vx[kRowsBwd], vg[kRowsBwd];
#pragma unroll
    for (int r = 0; r < kRowsBwd; ++r) {
      const int h = it.head0 + r * GPW + grp;
      if (in && h < x.heads) {
        vx[r].load(xsrc + h * x.xs[2]);
        vg[r].load(gsrc + h * x.dys[2]);
      } else {
        vx[r].zero();
        vg[r].zero();
      }
    }
    Turn<INTER> turn;
    turn.load(p, it.b, it.t, lg, lane);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = in ? weight_at<T>(x.weight, wdtype, lg * 8 + i) : 0.f;
    T* dst = static_cast<T*>(x.out) + ((it.b * p.T + it.t) * x.heads) * p.D + lg * 8;
#pragma unroll
    for (int r = 0; r < kRowsBwd; ++r) {
      float f[8], g[8];
      vx[r].get(f);
      vg[r].get(g);
      turn.template apply<true>(g);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
      const float rstd = rsqrtf(fmaf(group_sum<GL>(ss), inv_d, p.eps));
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[i] *= rstd;
        const float gx = g[i] * f[i];
        if (it.which) acc[1][i] += gx;
        else acc[0][i] += gx;
        g[i] *= w[i];
        dot = fmaf(g[i], f[i], dot);
      }
      dot = group_sum<GL>(dot) * inv_d;
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] = rstd * fmaf(-f[i], dot, g[i]);
      const int h = it.head0 + r * GPW + grp;
      if (in && h < x.heads) Vec8<T>::store(dst + (int64_t)h * p.D, g);
    }
  }
  // join the warp's groups, then the warps
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = acc[k][i];
#pragma unroll
      for (int o = GL; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (grp == 0) sums[warp][k][lg * 8 + i] = v;
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * p.D; c += kRopeThreads) {
    const int k = c >= p.D, d = c - k * p.D;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) v += sums[i][k][d];
    p.partial[(int64_t)blockIdx.x * 2 * p.D + c] = v;
  }
}

// dweight[c] = sum of column c of partial [rows, 2 D]: one CTA per 32 columns, 32 warps of
// rows, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* partial, int rows, int D, void* dq, void* dk,
                                                           int wdtype) {
  pdl_begin();
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < 2 * D)
    for (int r = warp; r < rows; r += 32) v += partial[(int64_t)r * 2 * D + c];
  sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < 2 * D) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sums[i][lane];
    void* out = c < D ? dq : dk;
    const int d = c < D ? c : c - D;
    if (wdtype == kDtypeF32) static_cast<float*>(out)[d] = s;
    else static_cast<T*>(out)[d] = (T)s;
  }
}

int lanes_of(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }

void plan_items(RopeParams& p, int rows) {
  const int hpi = 32 / lanes_of(p.D) * rows;
  p.chunks[0] = (p.t[0].heads + hpi - 1) / hpi;
  p.chunks[1] = (p.t[1].heads + hpi - 1) / hpi;
  p.items = (int64_t)p.B * p.T * (p.chunks[0] + p.chunks[1]);
}

int rope_ctas(int64_t items, int most) {
  const int64_t want = (items + kRopeThreads / 32 - 1) / (kRopeThreads / 32);
  return (int)(want < most ? want : most);
}

constexpr int kBwdCtas = 148 * 4;    // resident at 256 threads and up to 64 registers
constexpr int kFwdCtas = 148 * 64;

template <typename T, int GL, bool INTER>
cudaError_t launch_t(const RopeParams& p, int wdtype, bool backward, int ctas, cudaStream_t st) {
  return backward ? launch_pdl(norm_rope_backward_kernel<T, GL, INTER>, dim3(ctas), dim3(kRopeThreads), 0, st, p, wdtype)
                  : launch_pdl(norm_rope_kernel<T, GL, INTER>, dim3(ctas), dim3(kRopeThreads), 0, st, p, wdtype);
}

template <typename T>
cudaError_t launch_dtype(const RopeParams& p, int wdtype, bool inter, bool backward, int ctas, cudaStream_t st) {
  switch (lanes_of(p.D)) {
    case 8: return inter ? launch_t<T, 8, true>(p, wdtype, backward, ctas, st) : launch_t<T, 8, false>(p, wdtype, backward, ctas, st);
    case 16: return inter ? launch_t<T, 16, true>(p, wdtype, backward, ctas, st) : launch_t<T, 16, false>(p, wdtype, backward, ctas, st);
    default: return inter ? launch_t<T, 32, true>(p, wdtype, backward, ctas, st) : launch_t<T, 32, false>(p, wdtype, backward, ctas, st);
  }
}

cudaError_t launch_any(const RopeParams& p, int dtype, int wdtype, bool inter, bool backward, int ctas,
                       cudaStream_t st) {
  switch (dtype) {
    case kDtypeBF16: return launch_dtype<__nv_bfloat16>(p, wdtype, inter, backward, ctas, st);
    case kDtypeF16: return launch_dtype<__half>(p, wdtype, inter, backward, ctas, st);
    default: return launch_dtype<float>(p, wdtype, inter, backward, ctas, st);
  }
}

}  // namespace

cudaError_t launch_norm_rope(RopeParams p, int dtype, int wdtype, bool interleaved, cudaStream_t st) {
  plan_items(p, kRowsFwd);
  return launch_any(p, dtype, wdtype, interleaved, false, rope_ctas(p.items, kFwdCtas), st);
}

int norm_rope_backward_ctas(int64_t B, int64_t T, int64_t H, int64_t Hk, int D) {
  RopeParams p{};
  p.B = (int)B; p.T = (int)T; p.D = D;
  p.t[0].heads = (int)H; p.t[1].heads = (int)Hk;
  plan_items(p, kRowsBwd);
  return rope_ctas(p.items, kBwdCtas);
}

cudaError_t launch_norm_rope_backward(RopeParams p, int dtype, int wdtype, bool interleaved, cudaStream_t st) {
  plan_items(p, kRowsBwd);
  const int ctas = rope_ctas(p.items, kBwdCtas);
  cudaError_t e = launch_any(p, dtype, wdtype, interleaved, true, ctas, st);
  if (e != cudaSuccess) return e;
  const dim3 grid((2 * p.D + 31) / 32), block(1024);
  void *dq = p.t[0].dweight, *dk = p.t[1].dweight;
  const float* partial = p.partial;
  switch (dtype) {
    case kDtypeBF16: return launch_pdl(weight_grad_kernel<__nv_bfloat16>, grid, block, 0, st, partial, ctas, p.D, dq, dk, wdtype);
    case kDtypeF16: return launch_pdl(weight_grad_kernel<__half>, grid, block, 0, st, partial, ctas, p.D, dq, dk, wdtype);
    default: return launch_pdl(weight_grad_kernel<float>, grid, block, 0, st, partial, ctas, p.D, dq, dk, wdtype);
  }
}

}  // namespace solb200
