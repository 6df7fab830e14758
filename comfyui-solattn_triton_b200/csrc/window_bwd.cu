// Gradient of windowed attention with sinks on sm_100a tensor cores (tcgen05 + TMEM + TMA).
//
// With P = exp(scale q.k - lse) and delta = sum(dO * O) per query row:
//   dP = dO V^T,  dS = P (dP - delta),  dV = P^T dO,  dK = scale dS^T Q,  dQ = scale dS K.
// Two kernels, each of which owns what it writes, so nothing is added with atomics and the
// result is the same every time (the price: S and dP are formed twice, 7 products instead of 5):
//   window_dkv_kernel  a tile of 128 keys; walks the query tiles that see any of them (all
//                      query heads of the key head are stacked in a tile's rows, so shared
//                      heads need no sum afterwards): S^T and dP^T in TMEM, one key per
//                      lane; P^T and dS^T go back as bf16 A operands of dV += P^T dO, dK += dS^T Q;
//   window_dq_kernel   a tile of 128 query rows; walks the 128-key steps of WinSteps: S and
//                      dP, one query row per lane; dQ += dS K.
// All products are M = 128, N = 128 (N = head_dim for the sums); sums stay in 32 bits in TMEM,
// P and dS are rounded to bf16 for the tensor cores. 256 softmax threads (each 64 of a row's 128 columns),
// one TMA warp, one MMA warp, one CTA per SM.
//
// window_rows_kernel comes first: delta and -lse * log2(e) laid out by query tile, -inf for rows
// that see nothing and for the tile's rows past the last token, which makes their P zero.
#include "fwd_common.cuh"
#include "window.cuh"

namespace solb200 {

namespace {

constexpr int kTile = 128;
constexpr uint32_t kBox = kTile * 128;   // a 128-row box of 64 bf16 columns

// D (128 x 128) = A B^T, both K-major in shared memory (HD columns).
template <int HD>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_smem, uint32_t b_smem) {
  constexpr uint32_t IDESC = make_idesc(kFmtF32, kFmtBF16, kFmtBF16, 0, 0, 128, 128);
#pragma unroll
  for (int k = 0; k < HD / 16; ++k) {
    const uint32_t o = (k >> 2) * kBox + (k & 3) * 32;
    mma_bf16_ss(d, make_sw128_desc(a_smem + o, 16, 1024), make_sw128_desc(b_smem + o, 16, 1024), IDESC, k > 0);
  }
}

// D (128 x HD) += A B, A bf16 in TMEM (rows 0-63 of the sum at a, rows 64-127 at a + 64), B
// MN-major in shared memory (128 rows of HD columns).
template <int HD>
__device__ __forceinline__ void mma_sum(uint32_t d, uint32_t a, uint32_t b_smem, bool first) {
  constexpr uint32_t IDESC = make_idesc(kFmtF32, kFmtBF16, kFmtBF16, 0, 1, 128, HD);
#pragma unroll
  for (int k = 0; k < kTile / 16; ++k)
    mma_bf16_ts(d, a + (k >> 2) * 64 + (k & 3) * 8, make_sw128_desc(b_smem + k * 2048, kBox, 1024), IDESC,
                (first && k == 0) ? 0u : 1u);
}

// Zero rows [first, 128) of a tile of HD/64 boxes, by `n` threads.
template <int HD>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int first, int i0, int n) {
  const int per = (kTile - first) * 8;
  for (int i = i0; i < (HD / 64) * per; i += n)
    *reinterpret_cast<uint4*>(tile + (i / per) * kBox + first * 128 + (i % per) * 16) = make_uint4(0, 0, 0, 0);
}

// A row of the scaled accumulator, columns [c0, c0 + NC), as bf16 to global memory.
template <int NC>
__device__ __forceinline__ void store_row(uint32_t taddr, float scale, __nv_bfloat16* dst, bool live, bool zero) {
#pragma unroll 1
  for (int c = 0; c < NC / 32; ++c) {
    uint32_t r[32];
    if (!zero) {
      tmem_ld32(taddr + c * 32, r);
      tmem_wait_ld();
    }
    if (live) {
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = zero ? 0u : pack_bf16x2(__uint_as_float(r[v * 8 + 2 * i]) * scale,
                                         __uint_as_float(r[v * 8 + 2 * i + 1]) * scale);
        *reinterpret_cast<uint4*>(dst + c * 32 + v * 8) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// One row per HD / 8 lanes.
template <int HD>
__global__ void __launch_bounds__(256) window_rows_kernel(const __grid_constant__ WinParams p) {
  pdl_begin();
  constexpr int GL = HD / 8;
  const int lg = threadIdx.x % GL;
  const int64_t slot = ((int64_t)blockIdx.x * 256 + threadIdx.x) / GL;   // [B, Hk, nqt, 128]
  const int row = (int)(slot & 127);
  const int64_t tile = slot >> 7;
  const int qt = (int)(tile % p.nqt);
  const int64_t bh = tile / p.nqt;
  const int hk = (int)(bh % p.Hk), b = (int)(bh / p.Hk);
  const int tok = qt * p.TPT + row / p.G, h = hk * p.G + row % p.G;
  const bool live = b < p.B && row < p.RT && tok < p.Tq;
  float d = 0.f, neg = -INFINITY;
  if (live) {
    const uint4 wo = __ldg(reinterpret_cast<const uint4*>(p.o_in + b * p.os[0] + tok * p.os[1] + h * p.os[2]) + lg);
    const uint4 wd = __ldg(reinterpret_cast<const uint4*>(p.do_in + b * p.dos[0] + tok * p.dos[1] + h * p.dos[2]) + lg);
    const uint32_t o[4] = {wo.x, wo.y, wo.z, wo.w}, g[4] = {wd.x, wd.y, wd.z, wd.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      d = fmaf(__uint_as_float(o[i] << 16), __uint_as_float(g[i] << 16), d);
      d = fmaf(__uint_as_float(o[i] & 0xffff0000u), __uint_as_float(g[i] & 0xffff0000u), d);
    }
    const float lse = __ldg(p.lse_in + ((int64_t)b * p.H + h) * p.Tq + tok);
    if (lse != -INFINITY) neg = -lse * 1.4426950408889634f;
  }
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
  if (lg == 0 && b < p.B) {
    p.rows_lse[slot] = neg;
    p.rows_delta[slot] = neg == -INFINITY ? 0.f : d;
  }
}

// 64 columns of P and dS for one TMEM lane. `nl(c)` and `dl(c)` give -lse * log2(e) and delta of
// column c (0..63) - the same value for every column where a lane is a query row.
template <bool MASKED, typename NL>
__device__ __forceinline__ void probs(uint32_t t_s, float s2, uint32_t m0, uint32_t m1, float (&pr)[64], NL&& nl) {
  uint32_t ra[32], rb[32];
  tmem_ld32(t_s, ra);
  tmem_ld32(t_s + 32, rb);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    pr[i] = fast_exp2(fmaf(__uint_as_float(ra[i]), s2, nl(i)));
    pr[i + 32] = fast_exp2(fmaf(__uint_as_float(rb[i]), s2, nl(i + 32)));
    if (MASKED) {
      if (!((m0 >> i) & 1u)) pr[i] = 0.f;
      if (!((m1 >> i) & 1u)) pr[i + 32] = 0.f;
    }
  }
}

template <bool MASKED, typename DL>
__device__ __forceinline__ void score_grads(uint32_t t_dp, uint32_t t_out, uint32_t m0, uint32_t m1,
                                            const float (&pr)[64], DL&& dl) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t r[32], w[16];
    tmem_ld32(t_dp + c * 32, r);
    tmem_wait_ld();
    const uint32_t m = c ? m1 : m0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float g = pr[c * 32 + i] * (__uint_as_float(r[i]) - dl(c * 32 + i));
      if (MASKED && !((m >> i) & 1u)) g = 0.f;   // a hidden key's dP may be anything
      r[i] = __float_as_uint(g);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
    tmem_st16(t_out + c * 16, w);
  }
}

__device__ __forceinline__ void store_probs(uint32_t t_out, const float (&pr)[64]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(pr[c * 32 + 2 * i], pr[c * 32 + 2 * i + 1]);
    tmem_st16(t_out + c * 16, w);
  }
}

template <int HD>
__global__ void __launch_bounds__(320, 1)
window_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                  const __grid_constant__ WinParams p) {
  pdl_begin();
  constexpr int NBOX = HD / 64;
  constexpr uint32_t TILE = NBOX * kBox;

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + TILE;
  uint8_t* sQ = sV + TILE;               // 2 stages
  uint8_t* sG = sQ + 2 * TILE;           // dO, 2 stages
  float* sRow = reinterpret_cast<float*>(sG + 2 * TILE);   // 2 stages of [-lse2 128, delta 128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRow + 2 * 256);
  uint64_t* bar_kv = bars + 0;
  uint64_t* bar_q = bars + 1;            // [2] Q and its rows' numbers
  uint64_t* bar_g = bars + 3;            // [2] dO
  uint64_t* bar_dv = bars + 5;           // [2] dV(i) complete
  uint64_t* bar_dk = bars + 7;           // [2] dK(i) complete
  uint64_t* bar_s = bars + 9;
  uint64_t* bar_p = bars + 10;
  uint64_t* bar_dp = bars + 11;
  uint64_t* bar_ds = bars + 12;
  uint64_t* bar_drain = bars + 13;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // key tiles are the slow index: under a causal mask, and with sinks, the first ones
  // are seen by the most queries, and the longest CTAs start first
  int id = blockIdx.x;
  const int hk = id % p.Hk;
  id /= p.Hk;
  const int b = id % p.B, kt = id / p.B;
  const WinSeq seq(p, b);
  const int j0 = kt * kTile, j1 = min(j0 + kTile, seq.L);   // keys [j0, j1) of this tile count
  // tokens that see any of them
  const int ta = p.right < 0 ? 0 : clamp_to((int64_t)j0 - p.right - seq.off, 0, p.Tq);
  const int tb = (p.left < 0 || j0 < p.sinks) ? p.Tq : clamp_to((int64_t)j1 - 1 + p.left - seq.off + 1, 0, p.Tq);
  const int q_begin = ta / p.TPT;
  const int n = (j1 > j0 && tb > ta) ? (tb + p.TPT - 1) / p.TPT - q_begin : 0;

  if (threadIdx.x == 0) {
    mbar_init(bar_kv, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_q + i, 1);
      mbar_init(bar_g + i, 1);
      mbar_init(bar_dv + i, 1);
      mbar_init(bar_dk + i, 1);
    }
    mbar_init(bar_s, 1);
    mbar_init(bar_p, 256);
    mbar_init(bar_dp, 1);
    mbar_init(bar_ds, 256);
    mbar_init(bar_drain, 1);
    fence_barrier_init();
  }
  // rows that no box fills are summed over (with P = dS = 0): they have to be finite
  if (p.RT < kTile && n > 0)
    for (int i = 0; i < 2; ++i) {
      zero_rows<HD>(sQ + i * TILE, p.RT, threadIdx.x, 320);
      zero_rows<HD>(sG + i * TILE, p.RT, threadIdx.x, 320);
    }
  fence_proxy_async_smem();
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 128, tDV = tmem + 256, tDK = tmem + 384;

  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(bar_kv, 2 * TILE);
      for (int i = 0; i < NBOX; ++i) tma_load_4d(sK + i * kBox, &tm_k, bar_kv, i * 64, hk, j0, b);
      auto load_q = [&](int i) {
        const int st = i & 1, qt = q_begin + i;
        mbar_arrive_expect_tx(bar_q + st, NBOX * p.RT * 128 + 1024);
        for (int x = 0; x < NBOX; ++x)
          tma_load_4d(sQ + st * TILE + x * kBox, &tm_q, bar_q + st, x * 64, hk * p.G, qt * p.TPT, b);
        const int64_t r = (((int64_t)b * p.Hk + hk) * p.nqt + qt) * kTile;
        bulk_load(sRow + st * 256, p.rows_lse + r, 512, bar_q + st);
        bulk_load(sRow + st * 256 + 128, p.rows_delta + r, 512, bar_q + st);
      };
      auto load_g = [&](int i) {
        const int st = i & 1;
        mbar_arrive_expect_tx(bar_g + st, NBOX * p.RT * 128);
        for (int x = 0; x < NBOX; ++x)
          tma_load_4d(sG + st * TILE + x * kBox, &tm_do, bar_g + st, x * 64, hk * p.G, (q_begin + i) * p.TPT, b);
      };
      load_q(0);
      for (int i = 0; i < NBOX; ++i) tma_load_4d(sV + i * kBox, &tm_v, bar_kv, i * 64, hk, j0, b);
      load_g(0);
      int last_q = 0, last_g = 0;
      if (n > 1) {
        load_q(last_q = 1);
        load_g(last_g = 1);
      }
      bool ok = true;
      for (int i = 2; i < n; ++i) {
        if (!(ok = mbar_wait(bar_dv + (i & 1), ((i - 2) >> 1) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
        load_g(last_g = i);
        if (!(ok = mbar_wait(bar_dk + (i & 1), ((i - 2) >> 1) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
        load_q(last_q = i);
      }
      if (!ok) {
        // exit path: every issued copy lands before the CTA's shared memory goes away
        mbar_wait(bar_kv, 0, p.err, kErrWaitDrain);
        for (int i = max(0, last_q - 1); i <= last_q; ++i) mbar_wait(bar_q + (i & 1), (i >> 1) & 1, p.err, kErrWaitDrain);
        for (int i = max(0, last_g - 1); i <= last_g; ++i) mbar_wait(bar_g + (i & 1), (i >> 1) & 1, p.err, kErrWaitDrain);
      }
    }
  } else if (warp == 9) {
    // -------------------------------------------------------------- MMA issuer
    //   S(0) dP(0) | dV(i) S(i+1) dK(i) dP(i+1) | ...  The softmax works on dS(i) while
    //   dV(i) and S(i+1) run, and on P(i+1) while dK(i) and dP(i+1) run.
    if (lane == 0 && n > 0) {
      const uint32_t k_s = smem_u32(sK), v_s = smem_u32(sV), q_s = smem_u32(sQ), g_s = smem_u32(sG);
      bool ok = mbar_wait(bar_kv, 0, p.err, kErrWaitMma, p.wait_ns) &&
                mbar_wait(bar_q, 0, p.err, kErrWaitMma, p.wait_ns);
      if (ok) {
        tc_fence_after();
        mma_scores<HD>(tS, k_s, q_s);
        tc_commit(bar_s);
        ok = mbar_wait(bar_g, 0, p.err, kErrWaitMma, p.wait_ns);
      }
      if (ok) {
        tc_fence_after();
        mma_scores<HD>(tDP, v_s, g_s);
        tc_commit(bar_dp);
      }
      for (int i = 0; ok && i < n; ++i) {
        const int st = i & 1, nx = st ^ 1;
        const uint32_t par = (i >> 1) & 1, npar = ((i + 1) >> 1) & 1;
        if (!(ok = mbar_wait(bar_p, i & 1, p.err, kErrWaitMma, p.wait_ns))) break;
        tc_fence_after();
        mma_sum<HD>(tDV, tS, g_s + st * TILE, i == 0);
        tc_commit(bar_dv + st);
        if (i + 1 < n) {
          // S(i+1) overwrites P(i): dV(i) has to have read it
          if (!(ok = mbar_wait(bar_q + nx, npar, p.err, kErrWaitMma, p.wait_ns))) break;
          if (!(ok = mbar_wait(bar_dv + st, par, p.err, kErrWaitMma, p.wait_ns))) break;
          tc_fence_after();
          mma_scores<HD>(tS, k_s, q_s + nx * TILE);
          tc_commit(bar_s);
        }
        if (!(ok = mbar_wait(bar_ds, i & 1, p.err, kErrWaitMma, p.wait_ns))) break;
        tc_fence_after();
        mma_sum<HD>(tDK, tDP, q_s + st * TILE, i == 0);
        tc_commit(bar_dk + st);
        if (i + 1 < n) {
          if (!(ok = mbar_wait(bar_g + nx, npar, p.err, kErrWaitMma, p.wait_ns))) break;
          if (!(ok = mbar_wait(bar_dk + st, par, p.err, kErrWaitMma, p.wait_ns))) break;
          tc_fence_after();
          mma_scores<HD>(tDP, v_s, g_s + nx * TILE);
          tc_commit(bar_dp);
        }
      }
      // every MMA this thread issued has completed once bar_drain fires
      tc_commit(bar_drain);
      mbar_wait(bar_drain, 0, p.err, kErrWaitDrain);
    }
  } else {
    // -------------------------------------------- softmax + epilogue (one key per lane)
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane, c0 = wg * 64;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tS + lane_base + c0, tdp = tDP + lane_base + c0;
    const int j = j0 + row;
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int st = i & 1, t0 = (q_begin + i) * p.TPT;
      const int64_t pa = seq.off + t0, pb = pa + p.TPT - 1;
      const float* neg = sRow + st * 256 + c0;
      const float* delta = neg + 128;
      // every query of the tile sees every key of the tile?
      const bool full = j0 + kTile <= seq.L && (p.right < 0 || pa + p.right >= j0 + kTile - 1) &&
                        (p.left < 0 || pb - p.left <= j0 || j0 + kTile <= p.sinks);
      uint32_t m0 = 0, m1 = 0;
      if (!full && j < seq.L) {
        const int lo = p.right < 0 ? 0 : clamp_to((int64_t)j - p.right - pa, 0, p.TPT) * p.G;
        const int hi = (p.left < 0 || j < p.sinks) ? kTile : clamp_to((int64_t)j + p.left - pa + 1, 0, p.TPT) * p.G;
        m0 = win_low_bits(hi - c0) & ~win_low_bits(lo - c0);
        m1 = win_low_bits(hi - c0 - 32) & ~win_low_bits(lo - c0 - 32);
      }
      if (!(ok = mbar_wait_warp(bar_q + st, (i >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      if (!(ok = mbar_wait_warp(bar_s, i & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      float pr[64];
      if (full) probs<false>(ts, p.s2, m0, m1, pr, [&](int c) { return neg[c]; });
      else probs<true>(ts, p.s2, m0, m1, pr, [&](int c) { return neg[c]; });
      store_probs(ts, pr);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar_p);
      if (!(ok = mbar_wait_warp(bar_dp, i & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      if (full) score_grads<false>(tdp, tdp, m0, m1, pr, [&](int c) { return delta[c]; });
      else score_grads<true>(tdp, tdp, m0, m1, pr, [&](int c) { return delta[c]; });
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar_ds);
    }
    if (ok && n > 0) ok = mbar_wait_warp(bar_drain, 0, p.err, kErrWaitEpilogue, p.wait_ns);
    tc_fence_after();
    if (ok) {
      __nv_bfloat16* dst = (wg ? p.dk : p.dv) + (((int64_t)b * p.Tk + j) * p.Hk + hk) * HD;
      store_row<HD>((wg ? tDK : tDV) + lane_base, wg ? p.scale : 1.f, dst, j < p.Tk, n == 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
__global__ void __launch_bounds__(320, 1)
window_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                 const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_do,
                 const __grid_constant__ WinParams p) {
  pdl_begin();
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
  uint64_t* bar_ds = bars + 13;
  uint64_t* bar_drain = bars + 14;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 15);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int id = blockIdx.x;
  const int qt = p.nqt - 1 - id % p.nqt;
  id /= p.nqt;
  const int hk = id % p.Hk, b = id / p.Hk;
  const WinSeq seq(p, b);
  const int t0 = qt * p.TPT, ntok = min(p.TPT, p.Tq - t0);
  const int64_t pa = seq.off + t0, pb = pa + ntok - 1;
  const WinSteps<kTile> steps(p, seq.L, pa, pb);
  const int n = steps.n, rows = ntok * p.G;

  if (threadIdx.x == 0) {
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
    mbar_init(bar_ds, 256);
    mbar_init(bar_drain, 1);
    fence_barrier_init();
  }
  if (p.RT < kTile && n > 0) {
    zero_rows<HD>(sQ, p.RT, threadIdx.x, 320);
    zero_rows<HD>(sG, p.RT, threadIdx.x, 320);
  }
  fence_proxy_async_smem();
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem, tDP = tmem + 256, tDQ = tmem + 384;   // two slots of S (dS written over them)

  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      auto load_k = [&](int i) {
        uint64_t* bar = bar_k + i % 3;
        mbar_arrive_expect_tx(bar, TILE);
        for (int x = 0; x < NBOX; ++x)
          tma_load_4d(sK + (i % 3) * TILE + x * kBox, &tm_k, bar, x * 64, hk, steps.key0(i), b);
      };
      auto load_v = [&](int i) {
        uint64_t* bar = bar_v + (i & 1);
        mbar_arrive_expect_tx(bar, TILE);
        for (int x = 0; x < NBOX; ++x)
          tma_load_4d(sV + (i & 1) * TILE + x * kBox, &tm_v, bar, x * 64, hk, steps.key0(i), b);
      };
      mbar_arrive_expect_tx(bar_q, 2 * NBOX * p.RT * 128);
      for (int x = 0; x < NBOX; ++x) tma_load_4d(sQ + x * kBox, &tm_q, bar_q, x * 64, hk * p.G, t0, b);
      load_k(0);
      for (int x = 0; x < NBOX; ++x) tma_load_4d(sG + x * kBox, &tm_do, bar_q, x * 64, hk * p.G, t0, b);
      load_v(0);
      int last_k = 0, last_v = 0;
      if (n > 1) {
        load_k(last_k = 1);
        load_v(last_v = 1);
      }
      if (n > 2) load_k(last_k = 2);
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
  } else if (warp == 9) {
    // -------------------------------------------------------------- MMA issuer
    //   S(0) dP(0) S(1) | dP(i+1) dQ(i) S(i+2) | ...
    if (lane == 0 && n > 0) {
      const uint32_t q_s = smem_u32(sQ), g_s = smem_u32(sG), k_s = smem_u32(sK), v_s = smem_u32(sV);
      bool ok = mbar_wait(bar_q, 0, p.err, kErrWaitMma, p.wait_ns);
      auto issue_s = [&](int i) {
        ok = mbar_wait(bar_k + i % 3, (i / 3) & 1, p.err, kErrWaitMma, p.wait_ns);
        if (!ok) return;
        tc_fence_after();
        mma_scores<HD>(tS + (i & 1) * 128, q_s, k_s + (i % 3) * TILE);
        tc_commit(bar_s + (i & 1));
      };
      auto issue_dp = [&](int i) {
        ok = mbar_wait(bar_v + (i & 1), (i >> 1) & 1, p.err, kErrWaitMma, p.wait_ns);
        if (!ok) return;
        tc_fence_after();
        mma_scores<HD>(tDP, g_s, v_s + (i & 1) * TILE);
        tc_commit(bar_dp + (i & 1));
      };
      if (ok) issue_s(0);
      if (ok) issue_dp(0);
      if (ok && n > 1) issue_s(1);
      for (int i = 0; ok && i < n; ++i) {
        if (!(ok = mbar_wait(bar_ds, i & 1, p.err, kErrWaitMma, p.wait_ns))) break;
        tc_fence_after();
        if (i + 1 < n) issue_dp(i + 1);   // the softmax has taken dP(i) out
        if (!ok) break;
        mma_sum<HD>(tDQ, tS + (i & 1) * 128, k_s + (i % 3) * TILE, i == 0);
        tc_commit(bar_dq + i % 3);
        if (i + 2 < n) {
          // S(i+2) overwrites dS(i): dQ(i) has to have read it
          if (!(ok = mbar_wait(bar_dq + i % 3, (i / 3) & 1, p.err, kErrWaitMma, p.wait_ns))) break;
          issue_s(i + 2);
        }
      }
      tc_commit(bar_drain);
      mbar_wait(bar_drain, 0, p.err, kErrWaitDrain);
    }
  } else {
    // ---------------------------------------- softmax + epilogue (one query row per lane)
    const int wg = warp >> 2, row = (warp & 3) * 32 + lane, c0 = wg * 64;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int tok = row / p.G, head = row - tok * p.G;
    const bool live = row < rows;
    const int64_t pos = pa + tok;
    const int hi = live ? win_hi(p, seq.L, pos) : 0, lo = live ? win_lo(p, pos) : 0;
    const int64_t slot = (((int64_t)b * p.Hk + hk) * p.nqt + qt) * kTile + row;
    const float neg = p.rows_lse[slot], delta = p.rows_delta[slot];
    bool ok = true;
    for (int i = 0; i < n; ++i) {
      const int k0 = steps.key0(i);
      const uint32_t ts = tS + (i & 1) * 128 + lane_base + c0, tdp = tDP + lane_base + c0;
      const bool full = win_full(p, seq.L, pa, pb, k0, kTile);
      uint32_t m0 = 0, m1 = 0;
      if (!full && live) {
        m0 = win_bits(k0 + c0, lo, hi, p.sinks);
        m1 = win_bits(k0 + c0 + 32, lo, hi, p.sinks);
      }
      if (!(ok = mbar_wait_warp(bar_s + (i & 1), (i >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      float pr[64];
      if (full) probs<false>(ts, p.s2, m0, m1, pr, [&](int) { return neg; });
      else probs<true>(ts, p.s2, m0, m1, pr, [&](int) { return neg; });
      if (!(ok = mbar_wait_warp(bar_dp + (i & 1), (i >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
      tc_fence_after();
      if (full) score_grads<false>(tdp, ts, m0, m1, pr, [&](int) { return delta; });
      else score_grads<true>(tdp, ts, m0, m1, pr, [&](int) { return delta; });
      if (k0 + kTile > seq.L && seq.L < p.Tk) {
        // keys past the sequence's length may hold anything: zero their rows for dS K
        // (S(i) is complete, and bar_k was waited for before it was issued)
        if (!(ok = mbar_wait_warp(bar_k + i % 3, (i / 3) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
        zero_rows<HD>(sK + (i % 3) * TILE, seq.L - k0, threadIdx.x, 256);
        fence_proxy_async_smem();
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(bar_ds);
    }
    if (ok && n > 0) ok = mbar_wait_warp(bar_drain, 0, p.err, kErrWaitEpilogue, p.wait_ns);
    tc_fence_after();
    if (ok) {
      constexpr int NC = HD / 2;
      const int64_t orow = ((int64_t)b * p.Tq + t0 + tok) * p.H + hk * p.G + head;
      store_row<NC>(tDQ + lane_base + wg * NC, p.scale, p.out + orow * HD + wg * NC, live, n == 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int HD>
cudaError_t launch_t(const WinMaps& m, const WinParams& p, cudaStream_t st) {
  constexpr size_t TILE = (HD / 64) * kBox;
  constexpr size_t smem_kv = 6 * TILE + 2048 + 128 + 1024, smem_q = 7 * TILE + 128 + 1024;
  cudaError_t e = cudaFuncSetAttribute(window_dkv_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_kv);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(window_dq_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_q);
  if (e != cudaSuccess) return e;
  const int64_t slots = (int64_t)p.B * p.Hk * p.nqt * kTile;
  e = launch_pdl(window_rows_kernel<HD>, dim3((unsigned)(slots * (HD / 8) / 256)), dim3(256), 0, st, p);
  if (e != cudaSuccess) return e;
  e = launch_pdl(window_dkv_kernel<HD>, dim3((unsigned)((int64_t)p.B * p.Hk * p.nkt)), dim3(320), smem_kv, st, m.q, m.k,
                 m.v, m.dout, p);
  if (e != cudaSuccess) return e;
  return launch_pdl(window_dq_kernel<HD>, dim3((unsigned)((int64_t)p.B * p.Hk * p.nqt)), dim3(320), smem_q, st, m.q, m.k,
                    m.v, m.dout, p);
}

}  // namespace

cudaError_t launch_window_bwd(int hd, const WinMaps& m, const WinParams& p, cudaStream_t st) {
  return hd == 128 ? launch_t<128>(m, p, st) : launch_t<64>(m, p, st);
}

}  // namespace solb200
