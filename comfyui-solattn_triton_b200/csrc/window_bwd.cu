// Gradient of windowed attention with sinks on sm_100a tensor cores (tcgen05 + TMEM + TMA).
//
// With P = exp(scale q.k - lse) and delta = sum(dO * O) per query row:
//   dP = dO V^T,  dS = P (dP - delta),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
// Two kernels, each of which owns what it writes, so nothing is added with atomics and the
// result is the same every time (the price: S and dP are formed twice, 7 products instead of 5):
//   window_dkv_kernel  a tile of 128 keys; walks the query tiles that see any of them (all
//                      query heads of the key head are stacked in a tile's rows, so shared
//                      heads need no sum afterwards): S^T and dP^T in TMEM, one key per
//                      lane; P^T and dS^T go back, both over dP^T, as bf16 A operands of
//                      dV += P^T dO, dK += dS^T Q;
//   window_dq_kernel   a tile of 128 query rows; walks the 128-key steps of WinSteps: S and
//                      dP, one query row per lane; dQ += dS K.
// All products are M = 128, N = 128 (N = head_dim for the sums); sums stay in 32 bits in TMEM,
// P and dS are rounded to bf16 for the tensor cores. 512 softmax threads (each 32 of a row's 128
// columns; 256 threads took 616 us where these took 566, in the first form of window_dkv_kernel), one
// TMA warp, one MMA warp, one CTA per SM.
//
// Measured on a B200, 4 x 4096 tokens x 24 heads x 128, about 1000 keys a row, in short bursts: window_dq_kernel
// 370 us, window_dkv_kernel 472 us, 0.90 and 0.94 PFLOP/s of products executed. An iteration takes 2400 and
// 3300 cycles against 1536 and 2048 of products: the softmax threads are busy for most of them, and
// only what the barriers allow runs at the same time.
//
// Where the tiles are too few to fill the GPU, a tile's walk is divided over split_q (split_k) CTAs,
// which write their sums in 32 bits; window_grad_join_kernel adds them up in order.
//
// window_dq_kernel comes first and leaves -delta and -lse * log2(e) of its rows, by query tile, for
// window_dkv_kernel: -inf for rows that see nothing and for the tile's rows past the last token, which
// makes their P zero. (As a kernel of their own they took 26 us of the 1103 that the forward and the
// gradient took at the sizes above.)
// delta = sum(dO * O) carries the rounding of O to bf16, which counts where a row sees few keys (one
// key: dS is zero). For tiles of up to kFewSteps steps the kernel therefore forms delta =
// sum(P dP) / sum(P) in 32 bits before dS (sum(P) is 1 up to the rounding of lse).
#include "fwd_common.cuh"
#include "window.cuh"

namespace solb200 {

namespace {

constexpr int kTile = 128;
constexpr uint32_t kBox = kTile * 128;   // a 128-row box of 64 bf16 columns
constexpr int kSoftmax = 512;            // softmax threads: 4 per TMEM lane, 32 columns each
constexpr int kThreads = kSoftmax + 64;
constexpr int kFewSteps = 3;             // query tiles with up to this many key steps refine delta

// D (128 x 128) = A B^T, both K-major in shared memory (HD columns).
template <int HD>
__device__ __forceinline__ void mma_scores(uint32_t mine, uint32_t d, uint64_t a, uint64_t b) {
  constexpr uint32_t IDESC = make_idesc(kFmtF32, kFmtBF16, kFmtBF16, 0, 0, 128, 128);
#pragma unroll
  for (int k = 0; k < HD / 16; ++k) {
    const uint32_t o = (k >> 2) * kBox + (k & 3) * 32;
    mma_bf16_ss_warp(mine, d, desc_at(a, o), desc_at(b, o), IDESC, k > 0);
  }
}

// D (128 x HD) += A B over a quarter of the 128 summed rows, those of one column group: A bf16 in
// TMEM (at a + 32 quarter, in columns that only the group's threads read and write), B MN-major in
// shared memory (128 rows of HD columns).
template <int HD>
__device__ __forceinline__ void mma_sum_quarter(uint32_t mine, uint32_t d, uint32_t a, uint64_t b, int quarter, bool first) {
  constexpr uint32_t IDESC = make_idesc(kFmtF32, kFmtBF16, kFmtBF16, 0, 1, 128, HD);
#pragma unroll
  for (int k = 0; k < 2; ++k)
    mma_bf16_ts_warp(mine, d, a + quarter * 32 + k * 8, desc_at(b, (quarter * 2 + k) * 2048), IDESC,
                     (first && quarter == 0 && k == 0) ? 0u : 1u);
}

// Descriptors of a tile of 128 rows x HD columns: as a K-major operand (rows are M or N), and as
// an MN-major one (rows are summed over).
__device__ __forceinline__ uint64_t rows_desc(const uint8_t* tile) { return make_sw128_desc(smem_u32(tile), 16, 1024); }
__device__ __forceinline__ uint64_t sum_desc(const uint8_t* tile) { return make_sw128_desc(smem_u32(tile), kBox, 1024); }

// Zero rows [first, 128) of a tile of HD/64 boxes, by `n` threads.
template <int HD>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int first, int i0, int n) {
  const int per = (kTile - first) * 8;
  for (int i = i0; i < (HD / 64) * per; i += n)
    *reinterpret_cast<uint4*>(tile + (i / per) * kBox + first * 128 + (i % per) * 16) = make_uint4(0, 0, 0, 0);
}

// Channels [c0, c0 + NC) of a lane's row of the scaled accumulator, as bf16 into a tile of 128-row
// boxes with the 128-byte swizzle of a TMA store. (Rows stored from the lanes straight to global
// memory cost about 7000 cycles a tile: 16 bytes from each of 32 rows per instruction.)
template <int NC>
__device__ __forceinline__ void stage_row(uint32_t taddr, float scale, uint8_t* tile, int row, int c0, bool zero) {
#pragma unroll 1
  for (int c = c0; c < c0 + NC; c += 32) {
    uint32_t r[32];
    if (!zero) {
      tmem_ld32(taddr + c, r);
      tmem_wait_ld();
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = zero ? 0u : pack_bf16x2(__uint_as_float(r[v * 8 + 2 * i]) * scale,
                                       __uint_as_float(r[v * 8 + 2 * i + 1]) * scale);
      const int chunk = ((c & 63) >> 3) + v;
      *reinterpret_cast<uint4*>(tile + (c >> 6) * kBox + row * 128 + ((chunk ^ (row & 7)) << 4)) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The same channels in 32 bits straight to a part's row in memory (few tiles: its cost counts little).
template <int NC>
__device__ __forceinline__ void store_part(uint32_t taddr, float scale, float* dst, int c0, bool live, bool zero) {
#pragma unroll 1
  for (int c = c0; c < c0 + NC; c += 32) {
    uint32_t r[32];
    if (!zero) {
      tmem_ld32(taddr + c, r);
      tmem_wait_ld();
    }
    if (live) {
#pragma unroll
      for (int v = 0; v < 8; ++v)
        *reinterpret_cast<float4*>(dst + c + v * 4) =
            zero ? make_float4(0.f, 0.f, 0.f, 0.f)
                 : make_float4(__uint_as_float(r[v * 4]) * scale, __uint_as_float(r[v * 4 + 1]) * scale,
                               __uint_as_float(r[v * 4 + 2]) * scale, __uint_as_float(r[v * 4 + 3]) * scale);
    }
  }
}

// dq, dk and dv from their parts: blockIdx.y 0 joins dq (split_q parts), 1 dv and 2 dk (split_k parts); 8
// elements per thread.
__global__ void __launch_bounds__(256) window_grad_join_kernel(const __grid_constant__ WinParams p, int64_t nq, int64_t nk) {
  pdl_begin();
  const int which = blockIdx.y;
  const int64_t n = which ? nk : nq, i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  const int parts = which ? p.split_k : p.split_q;
  if (i >= n || parts == 1) return;
  const float* src = (which ? p.part_dkv + (which - 1) * nk : p.part_dq) + i;
  const int64_t step = which ? 2 * nk : nq;
  float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(src + s * step), y = *reinterpret_cast<const float4*>(src + s * step + 4);
    a[0] += x.x; a[1] += x.y; a[2] += x.z; a[3] += x.w;
    a[4] += y.x; a[5] += y.y; a[6] += y.z; a[7] += y.w;
  }
  __nv_bfloat16* dst = which == 0 ? p.out : (which == 1 ? p.dv : p.dk);
  *reinterpret_cast<uint4*>(dst + i) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]),
                                                  pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
}

// A query tile's row numbers, from the forward's output and log-sum-exp and from dO: -lse * log2(e)
// (-inf for rows that see nothing and past the tile's tokens) and -delta, into shared memory. One row
// per HD / 8 of the softmax threads; the loads land while the first tiles and scores are on their way.
template <int HD>
struct RowNumbers {
  static constexpr int GL = HD / 8, AT_ONCE = kSoftmax / GL, PASSES = kTile / AT_ONCE;
  uint4 wo[PASSES], wd[PASSES];
  float lse[PASSES];

  __device__ __forceinline__ RowNumbers(const WinParams& p, int b, int hk, int t0, int rows) {
    const int lg = threadIdx.x % GL;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const int row = i * AT_ONCE + threadIdx.x / GL;
      const DivMod by_g(row, p.G);
      const int tok = t0 + by_g.quot, h = hk * p.G + by_g.rem;
      wo[i] = wd[i] = make_uint4(0, 0, 0, 0);
      lse[i] = -INFINITY;
      if (row < rows) {
        wo[i] = __ldg(reinterpret_cast<const uint4*>(p.o_in + b * p.os[0] + tok * p.os[1] + h * p.os[2]) + lg);
        wd[i] = __ldg(reinterpret_cast<const uint4*>(p.do_in + b * p.dos[0] + tok * p.dos[1] + h * p.dos[2]) + lg);
        lse[i] = __ldg(p.lse_in + ((int64_t)b * p.H + h) * p.Tq + tok);
      }
    }
  }
  __device__ __forceinline__ void store(float* neg_lse, float* neg_delta) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      const uint32_t o[4] = {wo[i].x, wo[i].y, wo[i].z, wo[i].w}, g[4] = {wd[i].x, wd[i].y, wd[i].z, wd[i].w};
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        d = fmaf(__uint_as_float(o[j] << 16), __uint_as_float(g[j] << 16), d);
        d = fmaf(__uint_as_float(o[j] & 0xffff0000u), __uint_as_float(g[j] & 0xffff0000u), d);
      }
#pragma unroll
      for (int x = GL / 2; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
      const int row = i * AT_ONCE + threadIdx.x / GL;
      if (threadIdx.x % GL == 0) {
        neg_lse[row] = lse[i] == -INFINITY ? -INFINITY : -lse[i] * 1.4426950408889634f;
        neg_delta[row] = lse[i] == -INFINITY ? 0.f : -d;
      }
    }
  }
};

// 32 columns of P for one TMEM lane: 2^(s * s2 - lse * log2(e)), s the raw scores in r. `nl(i)` gives
// -lse * log2(e) of columns 4 i .. 4 i + 3 (where a lane is a query row, the same for all).
template <bool MASKED, typename NL>
__device__ __forceinline__ void probs(const uint32_t (&r)[32], float s2, uint32_t mask, float2 (&pr)[16], NL&& nl) {
  const float2 s22 = make_float2(s2, s2);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 l = nl(i);
    const float2 x = fma2(make_float2(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1])), s22, make_float2(l.x, l.y));
    const float2 y = fma2(make_float2(__uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3])), s22, make_float2(l.z, l.w));
    pr[2 * i] = make_float2(fast_exp2(x.x), fast_exp2(x.y));
    pr[2 * i + 1] = make_float2(fast_exp2(y.x), fast_exp2(y.y));
  }
  if (MASKED) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (!((mask >> (2 * i)) & 1u)) pr[i].x = 0.f;
      if (!((mask >> (2 * i + 1)) & 1u)) pr[i].y = 0.f;
    }
  }
}

__device__ __forceinline__ void store_cols(uint32_t t_out, const float2 (&x)[16]) {
  uint32_t w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(x[i].x, x[i].y);
  tmem_st16(t_out, w);
}

// dP of the same columns. MASKED: a hidden key's dP may be anything, its P is 0.
template <bool MASKED>
__device__ __forceinline__ void load_dp(uint32_t t_dp, uint32_t mask, float2 (&dp)[16]) {
  uint32_t r[32];
  tmem_ld32(t_dp, r);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (MASKED && !((mask >> i) & 1u)) r[i] = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) dp[i] = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
window_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                  const __grid_constant__ CUtensorMap tm_dk, const __grid_constant__ CUtensorMap tm_dv,
                  const __grid_constant__ WinParams p) {
  constexpr int NBOX = HD / 64;
  constexpr uint32_t TILE = NBOX * kBox;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  // (227 KB leave 768 bytes for the alignment of a base that is aligned already; one that needs
  // more is refused)
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (smem - smem_raw > 768) {
    pdl_begin();
    if (threadIdx.x == 0) atomicOr(p.err, kErrWaitLoad);
    return;
  }
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE;
  uint8_t* sQ = sV + TILE;               // 3 stages: Q(i) is read until dK(i), S(i+2) is next but one
  uint8_t* sG = sQ + 3 * TILE;           // dO, 2 stages
  float* sRow = reinterpret_cast<float*>(sG + 2 * TILE);   // 2 stages of [-lse2 128, -delta 128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRow + 2 * 256);
  uint64_t* bar_kv = bars + 0;
  uint64_t* bar_q = bars + 1;            // [3]
  uint64_t* bar_g = bars + 4;            // [2] dO and its rows' numbers
  uint64_t* bar_done = bars + 6;         // [2] dV(i) and dK(i) complete
  uint64_t* bar_s = bars + 8;
  uint64_t* bar_taken = bars + 9;        // S(i) is in the softmax threads' registers
  uint64_t* bar_dp = bars + 10;
  uint64_t* bar_drain = bars + 11;
  uint64_t* bar_p = bars + 12;           // [4] P(i) stored, by column group
  uint64_t* bar_ds = bars + 16;          // [4] dS(i) stored
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // the set-up that touches no global memory runs while the grid before this one finishes
  if (warp == kSoftmax / 32 && lane == 0) {
    mbar_init(bar_kv, 1);
    for (int i = 0; i < 3; ++i) mbar_init(bar_q + i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_g + i, 1);
      mbar_init(bar_done + i, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(bar_p + i, kSoftmax / 4);
      mbar_init(bar_ds + i, kSoftmax / 4);
    }
    mbar_init(bar_s, 1);
    mbar_init(bar_taken, kSoftmax);
    mbar_init(bar_dp, 1);
    mbar_init(bar_drain, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_do);
  }
  if (warp == kSoftmax / 32 + 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_begin();
  // key tiles are the slow index: under a causal mask, and with sinks, the first ones
  // are seen by the most queries, and the longest CTAs start first
  const DivMod by_hk(blockIdx.x, p.Hk), by_b(by_hk.quot, p.B), by_split(by_b.quot, p.split_k);
  const int hk = by_hk.rem, b = by_b.rem, split = by_split.rem, j0 = by_split.quot * kTile;
  // the first loads wait neither for the rest of the arithmetic nor for the other warps
  if (warp == kSoftmax / 32 && lane == 0) {
    mbar_arrive_expect_tx(bar_kv, 2 * TILE);
    for (int i = 0; i < NBOX; ++i) {
      tma_load_4d(sK + i * kBox, &tm_k, bar_kv, i * 64, hk, j0, b);
      tma_load_4d(sV + i * kBox, &tm_v, bar_kv, i * 64, hk, j0, b);
    }
  }
  const WinSeq seq(p, b);
  const int j1 = min(j0 + kTile, seq.L);   // keys [j0, j1) of this tile count
  // tokens that see any of them
  const int ta = p.right < 0 ? 0 : clamp_to((int64_t)j0 - p.right - seq.off, 0, p.Tq);
  const int tb = (p.left < 0 || j0 < p.sinks) ? p.Tq : clamp_to((int64_t)j1 - 1 + p.left - seq.off + 1, 0, p.Tq);
  const int q_first = udiv(ta, p.TPT), n_all = (j1 > j0 && tb > ta) ? udiv(tb + p.TPT - 1, p.TPT) - q_first : 0;
  const int q_begin = q_first + part_begin(n_all, split, p.split_k);
  const int n = __shfl_sync(0xffffffffu, q_first + part_begin(n_all, split + 1, p.split_k) - q_begin, 0);

  auto load_q = [&](int i) {
    mbar_arrive_expect_tx(bar_q + i % 3, NBOX * p.RT * 128);
    for (int x = 0; x < NBOX; ++x)
      tma_load_4d(sQ + (i % 3) * TILE + x * kBox, &tm_q, bar_q + i % 3, x * 64, hk * p.G, (q_begin + i) * p.TPT, b);
  };
  auto load_g = [&](int i) {
    const int st = i & 1, qt = q_begin + i;
    mbar_arrive_expect_tx(bar_g + st, NBOX * p.RT * 128 + 1024);
    const int64_t r = (((int64_t)b * p.Hk + hk) * p.nqt + qt) * kTile;
    bulk_load(sRow + st * 256, p.rows_lse + r, 512, bar_g + st);
    bulk_load(sRow + st * 256 + 128, p.rows_delta + r, 512, bar_g + st);
    for (int x = 0; x < NBOX; ++x)
      tma_load_4d(sG + st * TILE + x * kBox, &tm_do, bar_g + st, x * 64, hk * p.G, qt * p.TPT, b);
  };
  if (warp == kSoftmax / 32 && lane == 0 && n > 0) {
    load_q(0);
    load_g(0);
    if (n > 1) {
      load_q(1);
      load_g(1);
    }
    if (n > 2) load_q(2);
  }
  // rows that no box fills are summed over (with P = dS = 0): they have to be finite
  if (p.RT < kTile && n > 0)
    for (int i = 0; i < 5; ++i) zero_rows<HD>(sQ + i * TILE, p.RT, threadIdx.x, kThreads);
  if (p.RT < kTile) fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 128, tDV = tmem + 256, tDK = tmem + 384;

  if (warp == kSoftmax / 32) {
    // ------------------------------------------- TMA producer (after the first loads above)
    if (lane == 0 && n == 0) mbar_wait(bar_kv, 0, p.err, kErrWaitDrain);
    if (lane == 0 && n > 0) {
      int last_q = min(3, n) - 1, last_g = min(2, n) - 1;
      bool ok = true;
      for (int i = 0; i + 2 < n; ++i) {
        if (!(ok = mbar_wait(bar_done + (i & 1), (i >> 1) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
        load_g(last_g = i + 2);
        if (i + 3 < n) load_q(last_q = i + 3);
      }
      if (!ok) {
        // exit path: every issued copy lands before the CTA's shared memory goes away
        mbar_wait(bar_kv, 0, p.err, kErrWaitDrain);
        for (int i = max(0, last_q - 2); i <= last_q; ++i) mbar_wait(bar_q + i % 3, (i / 3) & 1, p.err, kErrWaitDrain);
        for (int i = max(0, last_g - 1); i <= last_g; ++i) mbar_wait(bar_g + (i & 1), (i >> 1) & 1, p.err, kErrWaitDrain);
      }
    }
  } else if (warp == kSoftmax / 32 + 1) {
    // -------------------------------------------------------------- MMA issuer
    //   S(0) dP(0) S(1) | dV(i) dK(i) dP(i+1) S(i+2) | ...  The softmax forms P(i+1) while dV(i),
    //   dK(i) and dP(i+1) run, and dS(i+1) while S(i+2) and dV(i+1) run.
    if (n > 0) {
      const uint32_t mine = elect_one();
      const uint64_t k_rows = rows_desc(sK), v_rows = rows_desc(sV), q_rows = rows_desc(sQ), g_rows = rows_desc(sG);
      const uint64_t q_sum = sum_desc(sQ), g_sum = sum_desc(sG);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool done = mbar_wait_warp(bar, parity, p.err, kErrWaitMma, p.wait_ns);
        tc_fence_after();
        return done;
      };
      auto issue_s = [&](int i) {
        if (!wait(bar_q + i % 3, (i / 3) & 1)) return false;
        mma_scores<HD>(mine, tS, k_rows, desc_at(q_rows, (i % 3) * TILE));
        tc_commit_warp(mine, bar_s);
        return true;
      };
      auto issue_dp = [&](int i) {
        if (!wait(bar_g + (i & 1), (i >> 1) & 1)) return false;
        mma_scores<HD>(mine, tDP, v_rows, desc_at(g_rows, (i & 1) * TILE));
        tc_commit_warp(mine, bar_dp);
        return true;
      };
      bool ok = wait(bar_kv, 0) && issue_s(0) && issue_dp(0) && (n == 1 || (wait(bar_taken, 0) && issue_s(1)));
      for (int i = 0; ok && i < n; ++i) {
        const int st = i & 1;
        for (int c = 0; ok && c < 4; ++c)
          if ((ok = wait(bar_p + c, i & 1))) mma_sum_quarter<HD>(mine, tDV, tDP, desc_at(g_sum, st * TILE), c, i == 0);
        for (int c = 0; ok && c < 4; ++c)
          if ((ok = wait(bar_ds + c, i & 1)))
            mma_sum_quarter<HD>(mine, tDK, tDP + 16, desc_at(q_sum, (i % 3) * TILE), c, i == 0);
        if (!ok) break;
        tc_commit_warp(mine, bar_done + st);
        // dP(i+1) overwrites P(i) and dS(i), S(i+2) S(i+1)
        if (i + 1 < n) ok = wait(bar_done + st, (i >> 1) & 1) && issue_dp(i + 1);
        if (ok && i + 2 < n) ok = wait(bar_taken, (i + 1) & 1) && issue_s(i + 2);
      }
      // every product issued has completed once bar_drain fires
      tc_commit_warp(mine, bar_drain);
      mbar_wait_warp(bar_drain, 0, p.err, kErrWaitDrain);
    }
  } else {
    // -------------------------------------------- softmax + epilogue (one key per lane)
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane, c0 = wg * 32;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tS + lane_base + c0, tdp = tDP + lane_base + c0;
    const int j = j0 + row;
    // tokens [first, last) see this lane's key; tokens [full_first, full_last) see every key of the tile
    const int first = p.right < 0 ? 0 : clamp_to((int64_t)j - p.right - seq.off, 0, p.Tq);
    const int last = j >= seq.L ? 0 : (p.left < 0 || j < p.sinks ? p.Tq : clamp_to((int64_t)j + p.left - seq.off + 1, 0, p.Tq));
    const int full_first = p.right < 0 ? 0 : clamp_to((int64_t)j0 + kTile - 1 - p.right - seq.off, 0, p.Tq);
    const int full_last = j0 + kTile > seq.L ? 0
                          : (p.left < 0 || j0 + kTile <= p.sinks ? p.Tq : clamp_to((int64_t)j0 + p.left - seq.off + 1, 0, p.Tq));
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int st = i & 1, t0 = (q_begin + i) * p.TPT;
      const float4* neg = reinterpret_cast<const float4*>(sRow + st * 256 + c0);
      const float4* ndelta = neg + 32;
      // (rows of tokens past the last have P = 0 without a mask)
      const bool full = t0 >= full_first && min(t0 + p.TPT, p.Tq) <= full_last;
      uint32_t mask = 0;
      if (!full) {
        const int lo = min(max(first - t0, 0), p.TPT) * p.G, hi = min(max(last - t0, 0), p.TPT) * p.G;
        mask = win_low_bits(hi - c0) & ~win_low_bits(lo - c0);
      }
      if (!(ok = mbar_wait_warp(bar_g + st, (i >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      if (!(ok = mbar_wait_warp(bar_s, i & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      uint32_t r[32];
      tmem_ld32(ts, r);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(bar_taken);
      float2 pr[16], dp[16];
      if (full) probs<false>(r, p.s2, mask, pr, [&](int c) { return neg[c]; });
      else probs<true>(r, p.s2, mask, pr, [&](int c) { return neg[c]; });
      if (!(ok = mbar_wait_warp(bar_dp, i & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      if (full) load_dp<false>(tdp, mask, dp);
      else load_dp<true>(tdp, mask, dp);
      store_cols(tdp, pr);
      // queries and dO of tokens that see nothing may hold anything: their rows are zeroed before the
      // sums, each column group its own quarter (S(i) and dP(i), which read them too, are complete)
      const WinBlind blind(p, seq, t0);
      if (!full && blind.any(p)) {
        if (!(ok = mbar_wait_warp(bar_q + i % 3, (i / 3) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
        for (int c = threadIdx.x & 127; c < 32 * NBOX * 8; c += 128) {
          const int r = c0 + c / (NBOX * 8), x = c % (NBOX * 8);
          if (r < blind.t0 * p.G || r >= blind.t1 * p.G) {
            const uint32_t at = (x >> 3) * kBox + r * 128 + (x & 7) * 16;
            *reinterpret_cast<uint4*>(sG + st * TILE + at) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(sQ + (i % 3) * TILE + at) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar_p + wg);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float4 d = ndelta[c];
        dp[2 * c] = mul2(pr[2 * c], add2(dp[2 * c], make_float2(d.x, d.y)));
        dp[2 * c + 1] = mul2(pr[2 * c + 1], add2(dp[2 * c + 1], make_float2(d.z, d.w)));
      }
      store_cols(tdp + 16, dp);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar_ds + wg);
    }
    // (without iterations: the loads of K and V, whose tiles take the zeros, have landed)
    if (ok) ok = mbar_wait_warp(n > 0 ? bar_drain : bar_kv, 0, p.err, kErrWaitEpilogue, p.wait_ns);
    tc_fence_after();
    if (ok && p.split_k > 1) {
      constexpr int NC = HD / 2;
      const int64_t row0 = ((int64_t)split * 2 + (wg < 2 ? 0 : 1)) * p.B * p.Tk;
      store_part<NC>((wg < 2 ? tDV : tDK) + lane_base, wg < 2 ? 1.f : p.scale,
                     p.part_dkv + ((row0 + (int64_t)b * p.Tk + j) * p.Hk + hk) * HD, (wg & 1) * NC, j < p.Tk, n == 0);
    } else if (ok) {
      // two of the four column groups take dV, two dK, half of the channels each; the tiles of V and
      // K are free (every product is complete)
      constexpr int NC = HD / 2;
      stage_row<NC>((wg < 2 ? tDV : tDK) + lane_base, wg < 2 ? 1.f : p.scale, wg < 2 ? sV : sK, row, (wg & 1) * NC,
                    n == 0);
      fence_proxy_async_smem();
    }
    if (named_bar_all(1, kSoftmax, ok) && p.split_k == 1 && threadIdx.x == 0) {
      for (int i = 0; i < NBOX; ++i) {
        tma_store_4d(&tm_dv, sV + i * kBox, i * 64, hk, j0, b);
        tma_store_4d(&tm_dk, sK + i * kBox, i * 64, hk, j0, b);
      }
      bulk_commit_group();
      bulk_wait_group_read0();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftmax / 32 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
window_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ CUtensorMap tm_dq, const __grid_constant__ WinParams p) {
  constexpr int NBOX = HD / 64;
  constexpr uint32_t TILE = NBOX * kBox;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sG = sQ + TILE;
  uint8_t* sK = sG + TILE;               // 3 stages: K(i) is read until dQ(i), S(i+2) needs the next
  uint8_t* sV = sK + 3 * TILE;           // 2 stages
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * TILE);
  uint64_t* bar_q = bars + 0;
  uint64_t* bar_k = bars + 1;            // [3]
  uint64_t* bar_v = bars + 4;            // [2]
  uint64_t* bar_dq = bars + 6;           // [3] dQ(i) complete
  uint64_t* bar_dp = bars + 9;           // [2]
  uint64_t* bar_s = bars + 11;           // [2]
  uint64_t* bar_ds = bars + 13;          // [2][4] by step parity (dS(i+1) may be stored before dS(i) is waited
                                         // for) and column group
  uint64_t* bar_drain = bars + 21;
  uint64_t* bar_taken = bars + 22;       // dP(i) is in the softmax threads' registers
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 23);
  float* sRow = reinterpret_cast<float*>(bars + 24);   // -lse * log2(e) [128], -delta [128]

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // the set-up that touches no global memory runs while the grid before this one finishes
  if (warp == kSoftmax / 32 && lane == 0) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < 3; ++i) {
      mbar_init(bar_k + i, 1);
      mbar_init(bar_dq + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_v + i, 1);
      mbar_init(bar_dp + i, 1);
      mbar_init(bar_s + i, 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(bar_ds + i, kSoftmax / 4);
    mbar_init(bar_taken, kSoftmax);
    mbar_init(bar_drain, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_do);
  }
  if (warp == kSoftmax / 32 + 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  pdl_begin();
  const DivMod by_split(blockIdx.x, p.split_q), by_tile(by_split.quot, p.nqt), by_hk(by_tile.quot, p.Hk);
  const int split = by_split.rem, qt = p.nqt - 1 - by_tile.rem, hk = by_hk.rem, b = by_hk.quot;
  const int t0 = qt * p.TPT, ntok = min(p.TPT, p.Tq - t0);
  // the first loads wait neither for the rest of the arithmetic nor for the other warps
  if (warp == kSoftmax / 32 && lane == 0) {
    mbar_arrive_expect_tx(bar_q, 2 * NBOX * p.RT * 128);
    for (int x = 0; x < NBOX; ++x) {
      tma_load_4d(sQ + x * kBox, &tm_q, bar_q, x * 64, hk * p.G, t0, b);
      tma_load_4d(sG + x * kBox, &tm_do, bar_q, x * 64, hk * p.G, t0, b);
    }
  }
  const int rows = ntok * p.G;
  RowNumbers<HD> numbers(p, b, hk, t0, warp < kSoftmax / 32 ? rows : 0);
  const WinSeq seq(p, b);
  const int64_t pa = seq.off + t0, pb = pa + ntok - 1;
  const WinSteps<kTile> steps(p, seq.L, pa, pb);
  // passes over steps: with 2 .. kFewSteps steps, one pass for delta before the one for dS (a
  // single step has all of a row's P and dP at hand)
  const bool few = steps.n <= kFewSteps;   // (not divided: the first part takes all)
  const int s_begin = few ? 0 : part_begin(steps.n, split, p.split_q);
  const int mine_n = few ? (split == 0 ? steps.n : 0) : part_begin(steps.n, split + 1, p.split_q) - s_begin;
  const int npre = __shfl_sync(0xffffffffu, few && mine_n > 1 ? mine_n : 0, 0);
  const int n = __shfl_sync(0xffffffffu, npre + mine_n, 0);
  auto key0 = [&](int i) { return steps.key0(s_begin + (i < npre ? i : i - npre)); };

  auto load_k = [&](int i) {
    uint64_t* bar = bar_k + i % 3;
    mbar_arrive_expect_tx(bar, TILE);
    for (int x = 0; x < NBOX; ++x)
      tma_load_4d(sK + (i % 3) * TILE + x * kBox, &tm_k, bar, x * 64, hk, key0(i), b);
  };
  auto load_v = [&](int i) {
    uint64_t* bar = bar_v + (i & 1);
    mbar_arrive_expect_tx(bar, TILE);
    for (int x = 0; x < NBOX; ++x)
      tma_load_4d(sV + (i & 1) * TILE + x * kBox, &tm_v, bar, x * 64, hk, key0(i), b);
  };
  if (warp == kSoftmax / 32 && lane == 0 && n > 0) {
    load_k(0);
    load_v(0);
    if (n > 1) {
      load_k(1);
      load_v(1);
    }
    if (n > 2) load_k(2);
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0;   // the call's error word
  if (p.RT < kTile && n > 0) {
    zero_rows<HD>(sQ, p.RT, threadIdx.x, kThreads);
    zero_rows<HD>(sG, p.RT, threadIdx.x, kThreads);
  }
  if (p.RT < kTile) fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 256, tDQ = tmem + 384;   // two slots of S (dS written over them)

  if (warp == kSoftmax / 32) {
    // ------------------------------------------- TMA producer (after the first loads above)
    if (lane == 0 && n == 0) mbar_wait(bar_q, 0, p.err, kErrWaitDrain);
    if (lane == 0 && n > 0) {
      int last_k = min(3, n) - 1, last_v = min(2, n) - 1;
      bool ok = true;
      for (int i = 0; i + 2 < n; ++i) {
        if (!(ok = mbar_wait(bar_dp + (i & 1), (i >> 1) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
        load_v(last_v = i + 2);
        if (i + 3 < n) {
          if (!(ok = mbar_wait(bar_dq + i % 3, (i / 3) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
          load_k(last_k = i + 3);
        }
      }
      if (!ok) {
        mbar_wait(bar_q, 0, p.err, kErrWaitDrain);
        for (int i = max(0, last_k - 2); i <= last_k; ++i) mbar_wait(bar_k + i % 3, (i / 3) & 1, p.err, kErrWaitDrain);
        for (int i = max(0, last_v - 1); i <= last_v; ++i) mbar_wait(bar_v + (i & 1), (i >> 1) & 1, p.err, kErrWaitDrain);
      }
    }
  } else if (warp == kSoftmax / 32 + 1) {
    // -------------------------------------------------------------- MMA issuer
    //   S(0) dP(0) S(1) | dP(i+1) dQ(i) S(i+2) | ...
    if (n > 0) {
      const uint32_t mine = elect_one();
      const uint64_t q_rows = rows_desc(sQ), g_rows = rows_desc(sG), k_rows = rows_desc(sK), v_rows = rows_desc(sV);
      const uint64_t k_sum = sum_desc(sK);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool done = mbar_wait_warp(bar, parity, p.err, kErrWaitMma, p.wait_ns);
        tc_fence_after();
        return done;
      };
      auto issue_s = [&](int i) {
        if (!wait(bar_k + i % 3, (i / 3) & 1)) return false;
        mma_scores<HD>(mine, tS + (i & 1) * 128, q_rows, desc_at(k_rows, (i % 3) * TILE));
        tc_commit_warp(mine, bar_s + (i & 1));
        return true;
      };
      auto issue_dp = [&](int i) {
        if (!wait(bar_v + (i & 1), (i >> 1) & 1)) return false;
        mma_scores<HD>(mine, tDP, g_rows, desc_at(v_rows, (i & 1) * TILE));
        tc_commit_warp(mine, bar_dp + (i & 1));
        return true;
      };
      bool ok = wait(bar_q, 0) && issue_s(0) && issue_dp(0) && (n == 1 || issue_s(1));
      for (int i = 0; ok && i < n; ++i) {
        if (i + 1 < n && !(ok = wait(bar_taken, i & 1) && issue_dp(i + 1))) break;
        // the first product overwrites the columns through which all four groups exchanged their sums for
        // delta (refine): each has read them once its dS is stored
        if (few && i == npre)
          for (int c = 0; ok && c < 4; ++c) ok = wait(bar_ds + (i & 1) * 4 + c, (i >> 1) & 1);
        for (int c = 0; ok && c < 4; ++c)
          if ((ok = wait(bar_ds + (i & 1) * 4 + c, (i >> 1) & 1)) && i >= npre)
            mma_sum_quarter<HD>(mine, tDQ, tS + (i & 1) * 128, desc_at(k_sum, (i % 3) * TILE), c, i == npre);
        if (!ok) break;
        tc_commit_warp(mine, bar_dq + i % 3);
        // S(i+2) overwrites dS(i): dQ(i) has to have read it
        if (i + 2 < n) ok = wait(bar_dq + i % 3, (i / 3) & 1) && issue_s(i + 2);
      }
      tc_commit_warp(mine, bar_drain);
      mbar_wait_warp(bar_drain, 0, p.err, kErrWaitDrain);
    }
  } else {
    // ---------------------------------------- softmax + epilogue (one query row per lane)
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane, c0 = wg * 32;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int tok = row / p.G, head = row - tok * p.G;
    const bool live = row < rows;
    const int64_t pos = pa + tok;
    const int hi = live ? win_hi(p, seq.L, pos) : 0, lo = live ? win_lo(p, pos) : 0;
    // every row of the tile sees the keys [full_lo, full_hi), and the sinks before full_hi
    const int full_hi = win_hi(p, seq.L, pa), full_lo = win_lo(p, pb);
    const int64_t slot = (((int64_t)b * p.Hk + hk) * p.nqt + qt) * kTile + row;
    numbers.store(sRow, sRow + kTile);
    named_bar_sync(1, kSoftmax);
    const float neg = sRow[row];
    float ndelta = sRow[kTile + row];
    if (split == 0 && wg == 0) {
      p.rows_lse[slot] = neg;
      p.rows_delta[slot] = ndelta;
    }
    float sum = 0.f, psum = 0.f;   // of P dP and P over this thread's columns, for delta
    bool owes = few && n > 0;
    // delta of the row from its four threads' parts, for this kernel and for window_dkv_kernel; the
    // parts meet in dQ's columns: the first dQ product waits until every group's dS is stored, after this
    auto refine = [&]() {
      owes = false;
      tmem_st1(tDQ + lane_base + wg, __float_as_uint(sum));
      tmem_st1(tDQ + lane_base + 4 + wg, __float_as_uint(psum));
      tmem_wait_st();
      tc_fence_before();
      named_bar_sync(1, kSoftmax);
      tc_fence_after();
      uint32_t r[4], q[4];
      tmem_ld4(tDQ + lane_base, r);
      tmem_ld4(tDQ + lane_base + 4, q);
      tmem_wait_ld();
      auto total = [](const uint32_t (&x)[4]) {
        return (__uint_as_float(x[0]) + __uint_as_float(x[1])) + (__uint_as_float(x[2]) + __uint_as_float(x[3]));
      };
      const float weights = total(q);
      ndelta = weights == 0.f ? 0.f : -total(r) / weights;   // (0: the row sees nothing)
      if (wg == 0) p.rows_delta[slot] = ndelta;
    };
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int k0 = key0(i);
      const uint32_t ts = tS + (i & 1) * 128 + lane_base + c0, tdp = tDP + lane_base + c0;
      const bool full = k0 + kTile <= full_hi && (k0 >= full_lo || k0 + kTile <= p.sinks);
      const uint32_t mask = !full && live ? win_bits(k0 + c0, lo, hi, p.sinks) : 0u;
      if (!(ok = mbar_wait_warp(bar_s + (i & 1), (i >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      float2 pr[16], dp[16];
      {
        uint32_t r[32];
        tmem_ld32(ts, r);
        tmem_wait_ld();
        if (full) probs<false>(r, p.s2, mask, pr, [&](int) { return make_float4(neg, neg, neg, neg); });
        else probs<true>(r, p.s2, mask, pr, [&](int) { return make_float4(neg, neg, neg, neg); });
      }
      if (!(ok = mbar_wait_warp(bar_dp + (i & 1), (i >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      if (full) load_dp<false>(tdp, mask, dp);
      else load_dp<true>(tdp, mask, dp);
      tc_fence_before();
      mbar_arrive(bar_taken);
      if (few && (i < npre || n == 1)) {
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          sum = fmaf(pr[c].x, dp[c].x, fmaf(pr[c].y, dp[c].y, sum));
          psum += pr[c].x + pr[c].y;
        }
        if (n == 1 || i + 1 == npre) refine();
      }
      if (i >= npre) {
        const float2 nd = make_float2(ndelta, ndelta);
#pragma unroll
        for (int c = 0; c < 16; ++c) dp[c] = mul2(pr[c], add2(dp[c], nd));
        store_cols(ts, dp);
        if (!full) {
          const WinUnseen unseen(p, seq.L, pa, pb, k0, kTile);
          if (unseen.any(kTile)) {
            // (S(i) is complete, and bar_k was waited for before it was issued)
            if (!(ok = mbar_wait_warp(bar_k + i % 3, (i / 3) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
            // each column group zeroes the rows of its own quarter of the sum: bar_ds is per group
            uint8_t* tile = sK + (i % 3) * TILE;
            for (int c = threadIdx.x & 127; c < 32 * NBOX * 8; c += 128) {
              const int r = c0 + c / (NBOX * 8), x = c % (NBOX * 8);
              if ((r >= unseen.a0 && r < unseen.a1) || r >= unseen.b0)
                *reinterpret_cast<uint4*>(tile + (x >> 3) * kBox + r * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        tmem_wait_st();
      }
      tc_fence_before();
      mbar_arrive(bar_ds + (i & 1) * 4 + wg);
    }
    if (owes) named_bar_sync(1, kSoftmax);   // (a wait failed before the refinement: take part in its barrier)
    // (without iterations: the load of Q, whose tile takes the zeros, has landed)
    if (ok) ok = mbar_wait_warp(n > 0 ? bar_drain : bar_q, 0, p.err, kErrWaitEpilogue, p.wait_ns);
    tc_fence_after();
    if (ok && wg < HD / 32 && p.split_q > 1) {
      const int64_t orow = ((int64_t)split * p.B * p.Tq + (int64_t)b * p.Tq + t0 + tok) * p.H + hk * p.G + head;
      store_part<32>(tDQ + lane_base, p.scale, p.part_dq + orow * HD, wg * 32, live, n == 0);
    } else if (ok && wg < HD / 32) {
      // (the tile of Q is free: every product is complete)
      stage_row<32>(tDQ + lane_base, p.scale, sQ, row, wg * 32, n == 0);
      fence_proxy_async_smem();
    }
    if (named_bar_all(1, kSoftmax, ok) && p.split_q == 1 && threadIdx.x == 0) {
      for (int i = 0; i < NBOX; ++i) tma_store_4d(&tm_dq, sQ + i * kBox, i * 64, hk * p.G, t0, b);
      bulk_commit_group();
      bulk_wait_group_read0();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kSoftmax / 32 + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
cudaError_t launch_t(const WinMaps& m, const WinParams& p, cudaStream_t st) {
  constexpr size_t TILE = (HD / 64) * kBox;
  constexpr size_t smem_kv = 7 * TILE + 2048 + 256 + 768, smem_q = 7 * TILE + 256 + 1024 + 1024;
  static std::atomic<uint64_t> allowed_kv{0}, allowed_q{0};
  cudaError_t e = allow_smem(window_dkv_kernel<HD>, smem_kv, allowed_kv);
  if (e == cudaSuccess) e = allow_smem(window_dq_kernel<HD>, smem_q, allowed_q);
  if (e != cudaSuccess) return e;
  // window_dq_kernel leaves the rows' numbers for window_dkv_kernel
  const int64_t heads = (int64_t)p.B * p.Hk;
  e = launch_pdl(window_dq_kernel<HD>, dim3((unsigned)(heads * p.nqt * p.split_q)), dim3(kThreads), smem_q, st, m.q, m.k,
                 m.v, m.dout, m.o, p);
  if (e != cudaSuccess) return e;
  e = launch_pdl(window_dkv_kernel<HD>, dim3((unsigned)(heads * p.nkt * p.split_k)), dim3(kThreads), smem_kv, st, m.q,
                 m.k, m.v, m.dout, m.dk, m.dv, p);
  if (e != cudaSuccess || (p.split_q == 1 && p.split_k == 1)) return e;
  const int64_t nq = p.split_q > 1 ? (int64_t)p.B * p.Tq * p.H * HD : 0;
  const int64_t nk = p.split_k > 1 ? (int64_t)p.B * p.Tk * p.Hk * HD : 0;
  const int64_t most = nq > nk ? nq : nk;
  return launch_pdl(window_grad_join_kernel, dim3((unsigned)((most + 2047) / 2048), 3), dim3(256), 0, st, p, nq, nk);
}

}  // namespace

cudaError_t launch_window_bwd(int hd, const WinMaps& m, const WinParams& p, cudaStream_t st) {
  return hd == 128 ? launch_t<128>(m, p, st) : launch_t<64>(m, p, st);
}

}  // namespace solb200
