// Root-mean-square norm of every head of q and k with the position rotation of the result, in
// one pass over both tensors, and its gradient.
//
//   r = (mean(x^2) + eps)^(-1/2),  n = x r w,  y = n with its first R elements turned by the
//   token's angles: (a, b) -> (a cos - b sin, a sin + b cos) on the pairs (2i, 2i + 1)
//   (interleaved) or (i, i + R / 2).
// Backward, with g = dy turned by the opposite angles and x^ = x r:
//   dw = sum over rows of g x^,   dx = r (g w - x^ mean(g w x^)).
//
// Both are bound by memory: 2 (3 backward) passes over the elements. A row (one head of one
// token) lies in a group of GL lanes, 8 elements per lane, so every access is 16 bytes per lane and
// the row sums are shuffles inside the group; the rotation's partner element is in the same lane
// (interleaved) or in the lane R / 16 further (halves). The rows of a tensor are numbered token by
// token, head by head; a warp takes runs of ROWS * 32 / GL of them, whatever the number
// of heads, copied ahead into a ring of its own in shared memory (cp.async: the loads in flight cost no
// registers), and forms the token's weight-times-angle
// coefficients once per run where the run lies in one token. A CTA stays with one tensor,
// so a lane's 8 weights are read once. Arithmetic is in 32 bits, two elements an instruction
// (f32x2), and rounded once, when y (dx) is stored.
//
// Measured on a B200 (the copy peak is 6.56 TB/s): see rows_in_flight.
#include "common.cuh"
#include "norm_rope.cuh"

#include <cuda_fp16.h>

namespace solb200 {

namespace {

constexpr int kRopeThreads = 256;
// Rows per lane group of a run, and runs a warp has in flight or at work. Measured (bf16, short
// bursts; back to back 221 - 229 and 107 - 113 us; forward 32760 x 80 rows of 128, backward 16384 x 48): forward 4 rows x 3 runs 212 us (6.3 TB/s), x 2
// 252 us, x 4 229 us, 2 rows with a register prefetch 255 us; backward 4 rows x 2 runs 108 us
// (weights' join included; 5.6 TB/s), 2 rows x 3 runs 120 us. Three CTAs an SM: 64 registers for four
// spill (260 and 152 us).
constexpr int rows_in_flight(bool wide) { return wide ? 2 : 4; }
constexpr int run_stages(bool backward) { return backward ? 2 : 3; }
constexpr int kResident = 3;   // CTAs per SM
// bytes of shared memory: 2 KB per run of one tensor in every type
constexpr int ring_bytes(bool backward) {
  return kRopeThreads / 32 * run_stages(backward) * (backward ? 4096 : 2048);
}

template <typename T>
struct Vec8;   // 8 elements of a row as they lie in memory

template <>
struct Vec8<float> {
  float4 a, b;
  static constexpr int PARTS = 2;   // 16-byte accesses
  __device__ void load_ring(const uint8_t* p) {
    a = *reinterpret_cast<const float4*>(p);
    b = *reinterpret_cast<const float4*>(p + 512);
  }
  __device__ Vec8 from_lane(int src) const {
    Vec8 o;
    const float in[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    float out[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = __shfl_sync(0xffffffffu, in[i], src);
    o.a = make_float4(out[0], out[1], out[2], out[3]);
    o.b = make_float4(out[4], out[5], out[6], out[7]);
    return o;
  }
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
  static constexpr int PARTS = 1;   // 16-byte accesses
  __device__ void load_ring(const uint8_t* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ Vec8 from_lane(int src) const {
    Vec8 o;
    o.w = make_uint4(__shfl_sync(0xffffffffu, w.x, src), __shfl_sync(0xffffffffu, w.y, src),
                     __shfl_sync(0xffffffffu, w.z, src), __shfl_sync(0xffffffffu, w.w, src));
    return o;
  }
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

// A lane's 8 elements as 4 pairs for f32x2 arithmetic. Interleaved rotations keep the pairs'
// first and second members apart, (a0, a1) (b0, b1) (a2, a3) (b2, b3); halves keep the order.
template <bool INTER>
__device__ __forceinline__ void to_pairs(const float (&f)[8], float2 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = INTER ? make_float2(f[(i >> 1) * 4 + (i & 1)], f[(i >> 1) * 4 + (i & 1) + 2]) : make_float2(f[2 * i], f[2 * i + 1]);
}
template <bool INTER>
__device__ __forceinline__ void from_pairs(const float2 (&v)[4], float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[INTER ? (i >> 1) * 4 + (i & 1) : 2 * i] = v[i].x;
    f[INTER ? (i >> 1) * 4 + (i & 1) + 2 : 2 * i + 1] = v[i].y;
  }
}

__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }

template <int GL>
__device__ __forceinline__ float group_sum2(const float2 (&v)[4], const float2 (&w)[4]) {
  float2 s = mul2(v[0], w[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) s = fma2(v[i], w[i], s);
  return group_sum<GL>(s.x + s.y);
}

// Cosines and sines of a lane's pairs: interleaved 2 of each (a and b turn alike), halves 4, the
// sine with the sign that the lane's side takes (first half -, second +). A lane past R does not turn.
template <bool INTER>
struct Angles {
  static constexpr int N = INTER ? 2 : 4;
  float2 c[N], s[N];

  __device__ __forceinline__ void load(const RopeParams& p, int64_t b, int64_t t, int lg) {
    const int half = p.R >> 1;
    const bool second = !INTER && lg * 8 >= half;
    const int col = INTER ? lg * 4 : (second ? lg * 8 - half : lg * 8);
    const float* at = p.cos + (b * p.ts[0] + t * p.ts[1]) + col;
    const float* at_s = p.sin + (b * p.ts[0] + t * p.ts[1]) + col;
    const float sign = !INTER && !second ? -1.f : 1.f;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      float4 vc = make_float4(1.f, 1.f, 1.f, 1.f), vs = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lg * 8 < p.R) {
        vc = __ldg(reinterpret_cast<const float4*>(at) + i);
        vs = __ldg(reinterpret_cast<const float4*>(at_s) + i);
      }
      c[2 * i] = make_float2(vc.x, vc.y);
      c[2 * i + 1] = make_float2(vc.z, vc.w);
      s[2 * i] = make_float2(sign * vs.x, sign * vs.y);
      s[2 * i + 1] = make_float2(sign * vs.z, sign * vs.w);
    }
  }
};

// The lane that holds the partner elements of a halves rotation (itself past R).
__device__ __forceinline__ int partner_lane(const RopeParams& p, int lg, int lane) {
  const int d = p.R >> 4;
  return lg * 8 >= p.R ? lane : (lg < d ? lane + d : lane - d);
}

// A warp's walk over the rows of its CTA's tensor: runs of RUN rows, `stride` runs apart. The
// place of a run's first row (head h of token t of sequence b) is carried along with additions.
template <int RUN>
struct RopeWalk {
  int which, rows, heads, T;
  int row, step;         // the run's first row, and rows to the next
  int h, t, b;           // its place
  int dh, dt, db;        // and the way to the next, as digits of heads and T

  __device__ __forceinline__ RopeWalk(const RopeParams& p, int warp, int warps) {
    which = blockIdx.x >= (unsigned)p.ctas[0];
    const int cta = which ? blockIdx.x - p.ctas[0] : blockIdx.x;
    rows = p.rows[which];
    heads = p.t[which].heads;
    T = p.T;
    // past the last row when there are more warps than runs; the product stays below 2^31
    // because a tensor has at most 2^30 rows and a grid at most one idle CTA
    row = (cta * warps + warp) * RUN;
    step = p.ctas[which] * warps * RUN;
    place(row, h, t, b);
    place(step, dh, dt, db);
  }
  __device__ __forceinline__ void place(int r, int& h_, int& t_, int& b_) const {
    const int bt = (int)((unsigned)r / (unsigned)heads);
    h_ = r - bt * heads;
    b_ = (int)((unsigned)bt / (unsigned)T);
    t_ = bt - b_ * T;
  }
  __device__ __forceinline__ bool more() const { return row < rows; }
  __device__ __forceinline__ void next() {
    row += step;
    h += dh;
    t += dt;
    b += db;
    if (h >= heads) {
      h -= heads;
      ++t;
    }
    if (t >= T) {
      t -= T;
      ++b;
    }
  }
  // the whole run lies in one token (so all of its rows exist)
  __device__ __forceinline__ bool one_token() const { return h + RUN <= heads; }
  // place of row `row + i`
  __device__ __forceinline__ void row_at(int i, int& h_, int& t_, int& b_) const {
    int x = h + i;
    const int more_t = (int)((unsigned)x / (unsigned)heads);
    h_ = x - more_t * heads;
    x = t + more_t;
    const int more_b = (int)((unsigned)x / (unsigned)T);
    t_ = x - more_b * T;
    b_ = b + more_b;
  }
};

__device__ __forceinline__ int64_t row_offset(const int64_t (&s)[3], int b, int t, int h) {
  return b * s[0] + t * s[1] + h * s[2];
}

// 16 bytes global -> shared, asynchronous; zeros where `there` is false (nothing is read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The run's rows of one tensor (strides s) into this lane's places of a ring stage, row r at
// dst + r * PARTS * 512: a lane reads back only what it copied itself, so no barrier is
// needed. A row that does not exist, and lanes past the head, read zeros.
template <typename T, int GPW, int ROWS, int RUN>
__device__ __forceinline__ void copy_run(const RopeWalk<RUN>& walk, const void* base, const int64_t (&s)[3], int lg,
                                         int grp, bool in, uint32_t dst) {
  constexpr int PARTS = Vec8<T>::PARTS;
  const T* src = static_cast<const T*>(base);
  if (walk.one_token()) {
    if (in) src += row_offset(s, walk.b, walk.t, walk.h + grp) + lg * 8;
    const int64_t step = in ? GPW * s[2] : 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
        copy16(dst + (r * PARTS + i) * 512, reinterpret_cast<const uint8_t*>(src + r * step) + i * 16, in);
  } else {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const bool there = in && walk.row + r * GPW + grp < walk.rows;
      int64_t at = 0;
      if (there) {
        int h, t, b;
        walk.row_at(r * GPW + grp, h, t, b);
        at = row_offset(s, b, t, h) + lg * 8;
      }
#pragma unroll
      for (int i = 0; i < PARTS; ++i)
        copy16(dst + (r * PARTS + i) * 512, reinterpret_cast<const uint8_t*>(src + at) + i * 16, there);
    }
  }
}

template <typename T, bool INTER>
__device__ __forceinline__ void load_weight(const void* w, int wdtype, int lg, bool in, float2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    f[i] = !in ? 0.f
               : (wdtype == kDtypeF32 ? __ldg(static_cast<const float*>(w) + lg * 8 + i)
                                      : (float)static_cast<const T*>(w)[lg * 8 + i]);
  to_pairs<INTER>(f, v);
}

template <typename T, int GL, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kResident)
norm_rope_kernel(const __grid_constant__ RopeParams p, int wdtype) {
  pdl_begin();
  constexpr int ROWS = rows_in_flight(sizeof(T) == 4);
  constexpr int GPW = 32 / GL, RUN = GPW * ROWS, WARPS = kRopeThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lg = lane % GL, grp = lane / GL;
  const bool in = lg * 8 < p.D;
  RopeWalk<RUN> walk(p, warp, WARPS);
  const RopeTensor& x = p.t[walk.which];
  const float inv_d = 1.f / (float)p.D;
  const int src = INTER ? lane : partner_lane(p, lg, lane);
  float2 w[4], wp[4];   // the weights, and (halves) the partners'
  load_weight<T, INTER>(x.weight, wdtype, lg, in, w);
  if (!INTER)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      wp[i] = make_float2(__shfl_sync(0xffffffffu, w[i].x, src), __shfl_sync(0xffffffffu, w[i].y, src));
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr int STAGE = ROWS * Vec8<T>::PARTS * 512, STAGES = run_stages(false);
  const uint8_t* mine = ring + warp * STAGES * STAGE + lane * 16;
  const uint32_t mine_s = smem_u32(mine);
  RopeWalk<RUN> ahead = walk;   // the run whose copies are issued next
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) {
    if (ahead.more()) copy_run<T, GPW, ROWS>(ahead, x.x, x.xs, lg, grp, in, mine_s + i * STAGE);
    copy_commit();
    ahead.next();
  }
  for (int stage = 0; walk.more(); walk.next(), stage = stage + 1 == STAGES ? 0 : stage + 1) {
    if (ahead.more())
      copy_run<T, GPW, ROWS>(ahead, x.x, x.xs, lg, grp, in, mine_s + (stage == 0 ? STAGES - 1 : stage - 1) * STAGE);
    copy_commit();
    ahead.next();
    // y = r (x P + x' Q), x' the partners: P = w cos, Q = w' (-+ sin)
    float2 P[4], Q[4];
    auto coefficients = [&](int64_t b, int64_t t) {
      Angles<INTER> a;
      a.load(p, b, t, lg);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (INTER) {
          P[i] = mul2(w[i], a.c[(i >> 1) % Angles<INTER>::N]);
          Q[i] = mul2(w[i ^ 1], i & 1 ? a.s[(i >> 1) % Angles<INTER>::N] : neg2(a.s[(i >> 1) % Angles<INTER>::N]));
        } else {
          P[i] = mul2(w[i], a.c[i % Angles<INTER>::N]);
          Q[i] = mul2(wp[i], a.s[i % Angles<INTER>::N]);
        }
      }
    };
    const bool one_token = walk.one_token();   // (warp-uniform)
    if (one_token) coefficients(walk.b, walk.t);
    T* dst = static_cast<T*>(x.out) + (int64_t)(walk.row + grp) * p.D + lg * 8;
    copy_wait<STAGES - 1>();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const bool live = in && (one_token || walk.row + r * GPW + grp < walk.rows);
      if (!one_token) {
        int h, t, b;
        walk.row_at(live ? r * GPW + grp : 0, h, t, b);
        coefficients(b, t);
      }
      Vec8<T> v;
      v.load_ring(mine + stage * STAGE + r * Vec8<T>::PARTS * 512);
      float f[8];
      float2 a[4], y[4];
      v.get(f);
      to_pairs<INTER>(f, a);
      const float2 rstd = splat(rsqrtf(fmaf(group_sum2<GL>(a, a), inv_d, p.eps)));
      if (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = mul2(rstd, fma2(a[i], P[i], mul2(a[i ^ 1], Q[i])));
      } else {
        float2 b[4];
        Vec8<T> other = v.from_lane(src);
        other.get(f);
        to_pairs<INTER>(f, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = mul2(rstd, fma2(a[i], P[i], mul2(b[i], Q[i])));
      }
      from_pairs<INTER>(y, f);
      if (live) Vec8<T>::store(dst + (int64_t)(r * GPW) * p.D, f);
    }
  }
}

// Every CTA walks the rows of its tensor with a stride and keeps its lanes' sums of the weight
// gradient in registers; they are joined over the CTA in a fixed order and written as one line
// of p.partial, which weight_grad_kernel adds up, again in a fixed order: no atomics, the same
// result every time.
template <typename T, int GL, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kResident)
norm_rope_backward_kernel(const __grid_constant__ RopeParams p, int wdtype) {
  pdl_begin();
  constexpr int ROWS = rows_in_flight(sizeof(T) == 4);
  constexpr int GPW = 32 / GL, RUN = GPW * ROWS, WARPS = kRopeThreads / 32;
  __shared__ float sums[WARPS][GL * 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int lg = lane % GL, grp = lane / GL;
  const bool in = lg * 8 < p.D;
  RopeWalk<RUN> walk(p, warp, WARPS);
  const RopeTensor& x = p.t[walk.which];
  const float inv_d = 1.f / (float)p.D;
  const int src = INTER ? lane : partner_lane(p, lg, lane);
  float2 w[4], acc[4];
  load_weight<T, INTER>(x.weight, wdtype, lg, in, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = splat(0.f);
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr int HALF = ROWS * Vec8<T>::PARTS * 512, STAGE = 2 * HALF, STAGES = run_stages(true);   // x, then dy
  const uint8_t* mine = ring + warp * STAGES * STAGE + lane * 16;
  const uint32_t mine_s = smem_u32(mine);
  RopeWalk<RUN> ahead = walk;   // the run whose copies are issued next
  auto copy = [&](int i) {
    if (ahead.more()) {
      copy_run<T, GPW, ROWS>(ahead, x.x, x.xs, lg, grp, in, mine_s + i * STAGE);
      copy_run<T, GPW, ROWS>(ahead, x.dy, x.dys, lg, grp, in, mine_s + i * STAGE + HALF);
    }
    copy_commit();
    ahead.next();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) copy(i);
  for (int stage = 0; walk.more(); walk.next(), stage = stage + 1 == STAGES ? 0 : stage + 1) {
    copy(stage == 0 ? STAGES - 1 : stage - 1);
    Angles<INTER> ang;
    const bool one_token = walk.one_token();   // (warp-uniform)
    if (one_token) ang.load(p, walk.b, walk.t, lg);
    T* dst = static_cast<T*>(x.out) + (int64_t)(walk.row + grp) * p.D + lg * 8;
    copy_wait<STAGES - 1>();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const bool live = in && (one_token || walk.row + r * GPW + grp < walk.rows);
      if (!one_token) {
        int h, t, b;
        walk.row_at(live ? r * GPW + grp : 0, h, t, b);
        ang.load(p, b, t, lg);
      }
      float f[8];
      float2 a[4], d[4], g[4];
      Vec8<T> v;
      v.load_ring(mine + stage * STAGE + r * Vec8<T>::PARTS * 512);
      v.get(f);
      to_pairs<INTER>(f, a);
      v.load_ring(mine + stage * STAGE + HALF + r * Vec8<T>::PARTS * 512);
      v.get(f);
      to_pairs<INTER>(f, d);
      // (a row that does not exist reads zeros: at eps = 0 its root is infinite, its x^ in the weights' sums NaN)
      const float root = rsqrtf(fmaf(group_sum2<GL>(a, a), inv_d, p.eps));
      const float rs = live ? root : 0.f;
      // g: the gradient turned back
      if (INTER) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 c = ang.c[(i >> 1) % Angles<INTER>::N], s = ang.s[(i >> 1) % Angles<INTER>::N];
          g[i] = fma2(d[i], c, mul2(d[i ^ 1], i & 1 ? neg2(s) : s));
        }
      } else {
        float2 b[4];
        Vec8<T> other = v.from_lane(src);
        other.get(f);
        to_pairs<INTER>(f, b);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          g[i] = fma2(d[i], ang.c[i % Angles<INTER>::N], mul2(b[i], neg2(ang.s[i % Angles<INTER>::N])));
      }
      float2 dot2 = splat(0.f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = mul2(a[i], splat(rs));                 // x^
        const float2 gx = mul2(g[i], a[i]);
        acc[i] = add2(acc[i], gx);
        dot2 = fma2(gx, w[i], dot2);
        g[i] = mul2(mul2(g[i], w[i]), splat(rs));
      }
      const float2 k = splat(-rs * inv_d * group_sum<GL>(dot2.x + dot2.y));
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = fma2(a[i], k, g[i]);
      from_pairs<INTER>(g, f);
      if (live) Vec8<T>::store(dst + (int64_t)(r * GPW) * p.D, f);
    }
  }
  // join the warp's groups, then the warps
  float f[8];
  from_pairs<INTER>(acc, f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v = f[i];
#pragma unroll
    for (int o = GL; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (grp == 0) sums[warp][lg * 8 + i] = v;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += kRopeThreads) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) v += sums[i][d];
    p.partial[(int64_t)blockIdx.x * p.D + d] = v;
  }
}

// dweight: the sums of the columns of q's lines of partial [lines, D] (blockIdx.y 0) and of k's (1).
// One CTA per 32 columns, 32 warps of lines, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) weight_grad_kernel(const __grid_constant__ RopeParams p, int wdtype) {
  pdl_begin();
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + lane, which = blockIdx.y;
  const float* partial = p.partial + (which ? (int64_t)p.ctas[0] * p.D : 0) + d;
  float v = 0.f;
  if (d < p.D)
#pragma unroll 4
    for (int r = warp; r < p.ctas[which]; r += 32) v += partial[(int64_t)r * p.D];
  sums[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && d < p.D) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += sums[i][lane];
    if (wdtype == kDtypeF32) static_cast<float*>(p.t[which].dweight)[d] = s;
    else static_cast<T*>(p.t[which].dweight)[d] = (T)s;
  }
}

int lanes_of(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }

// CTAs of each tensor: one run per warp while they last, else `most` in proportion to the rows.
void plan_ctas(RopeParams& p, int nrows, int most) {
  const int64_t per = (int64_t)(32 / lanes_of(p.D)) * nrows * (kRopeThreads / 32);
  int64_t want[2];
  for (int i = 0; i < 2; ++i) {
    p.rows[i] = p.B * p.T * p.t[i].heads;
    want[i] = (p.rows[i] + per - 1) / per;
  }
  if (want[0] + want[1] > most)
    for (int i = 0; i < 2; ++i) {
      const int64_t share = most * (int64_t)p.rows[i] / ((int64_t)p.rows[0] + p.rows[1]);
      want[i] = want[i] < share ? want[i] : (share < 1 ? 1 : share);
    }
  p.ctas[0] = (int)want[0];
  p.ctas[1] = (int)want[1];
}

constexpr int kMostCtas = 148 * kResident;

template <typename T, int GL, bool INTER>
cudaError_t launch_t(const RopeParams& p, int wdtype, bool backward, int ctas, cudaStream_t st) {
  auto kern = backward ? norm_rope_backward_kernel<T, GL, INTER> : norm_rope_kernel<T, GL, INTER>;
  static std::atomic<uint64_t> allowed[2];
  const cudaError_t e = allow_smem(kern, ring_bytes(backward), allowed[backward]);
  return e != cudaSuccess ? e : launch_pdl(kern, dim3(ctas), dim3(kRopeThreads), ring_bytes(backward), st, p, wdtype);
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
  plan_ctas(p, rows_in_flight(dtype == kDtypeF32), kMostCtas);
  return launch_any(p, dtype, wdtype, interleaved, false, p.ctas[0] + p.ctas[1], st);
}

int norm_rope_backward_ctas(int64_t B, int64_t T, int64_t H, int64_t Hk, int D) {
  RopeParams p{};
  p.B = (int)B; p.T = (int)T; p.D = D;
  p.t[0].heads = (int)H; p.t[1].heads = (int)Hk;
  // the more of the two run lengths' plans (the element type is not known here): shorter runs take more
  // CTAs, but past kMostCtas the tensors' shares are rounded down and may add up to one less
  int most = 0;
  for (const bool wide : {false, true}) {
    plan_ctas(p, rows_in_flight(wide), kMostCtas);
    const int ctas = p.ctas[0] + p.ctas[1];
    most = ctas > most ? ctas : most;
  }
  return most;
}

cudaError_t launch_norm_rope_backward(RopeParams p, int dtype, int wdtype, bool interleaved, cudaStream_t st) {
  plan_ctas(p, rows_in_flight(dtype == kDtypeF32), kMostCtas);
  cudaError_t e = launch_any(p, dtype, wdtype, interleaved, true, p.ctas[0] + p.ctas[1], st);
  if (e != cudaSuccess) return e;
  const dim3 grid((p.D + 31) / 32, 2), block(1024);
  switch (dtype) {
    case kDtypeBF16: return launch_pdl(weight_grad_kernel<__nv_bfloat16>, grid, block, 0, st, p, wdtype);
    case kDtypeF16: return launch_pdl(weight_grad_kernel<__half>, grid, block, 0, st, p, wdtype);
    default: return launch_pdl(weight_grad_kernel<float>, grid, block, 0, st, p, wdtype);
  }
}

}  // namespace solb200
