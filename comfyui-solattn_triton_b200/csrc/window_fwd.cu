// Windowed attention with sinks, forward, on sm_100a tensor cores (tcgen05 + TMEM + TMA).
//
// One CTA per (batch, key head, query tile, part of the key axis). The query heads of one
// key head are stacked into a tile's 128 rows, row = token * G + head, so their keys and
// values are read once and a tile spans fewer positions (a narrower band). The CTA walks the
// 64-key steps that any of its rows sees (WinSteps): the sinks', then the window's. Steps
// that every row sees whole skip the mask.
//
// The online softmax keeps a per-row reference maximum that is raised only when a step
// exceeds it by more than 2^8 (sums stay in 32 bits; P is rounded to bf16 for the tensor
// cores, at most a relative 2^-8 per weight). Two slots for K, V and scores:
//   MMA issuer:  QK(0) QK(1) | PV(0) QK(2) | PV(1) QK(3) | ...
// Warps 0-3 softmax and epilogue (thread = row = TMEM lane; a warp without rows takes no
// part), warp 4 TMA, warp 5 TMEM and MMA. 96 KB of shared memory and 256 TMEM columns: two CTAs per SM.
//
// When the tiles are too few to fill the GPU (single tokens, short chunks against a long
// cache), the steps are divided over nsplit CTAs, which write their unnormalised sums, maxima
// and row sums; window_join_kernel joins them in order.
//
// Keys that no row of the tile sees may hold anything (WinUnseen).
//
// Measured on a B200, 40 heads x 128: 32760 queries seeing about 5940 keys each 3.5 ms in a short
// burst (1.14 PFLOP/s), 4.0 back to back (0.99, at the power cap), bound by one CTA's softmax and the
// other's products taking turns (tensor pipe 59 % busy, exponentials 60 %); one token over 262001 keys
// 744 us in a burst (7.2 TB/s, reads alone), 796 - 858 back to back (6.7 - 6.3; a copy, which writes
// too, runs at 6.56).
#include "fwd_common.cuh"
#include "window.cuh"

namespace solb200 {

namespace {

constexpr int kStep = 64;

template <int HD>
__global__ void __launch_bounds__(192, 2)
window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_o,
                  const __grid_constant__ WinParams p) {
  constexpr int NBOX = HD / 64;            // 64-column (128-byte) boxes per row
  constexpr uint32_t QBOX = 128 * 128;     // a 128-row box
  constexpr uint32_t HBOX = kStep * 128;   // a 64-row box
  constexpr uint32_t SLOT = NBOX * HBOX;   // one step of K (or V)
  constexpr uint32_t IDESC_QK = make_idesc(kFmtF32, kFmtBF16, kFmtBF16, 0, 0, 128, 64);
  constexpr uint32_t IDESC_PV = make_idesc(kFmtF32, kFmtBF16, kFmtBF16, 0, 1, 128, HD);

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + NBOX * QBOX;
  uint8_t* sV = sK + 2 * SLOT;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * SLOT);
  uint64_t* bar_q = bars + 0;
  uint64_t* bar_kfull = bars + 1;          // [2] each
  uint64_t* bar_vfull = bars + 3;
  uint64_t* bar_sfull = bars + 5;
  uint64_t* bar_pfull = bars + 7;
  uint64_t* bar_pvdone = bars + 9;
  uint64_t* bar_drain = bars + 11;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // the set-up that touches no global memory runs while the grid before this one finishes
  // (bar_pfull counts the threads of the warps with rows: after the tile is known)
  if (warp == 4 && lane == 0) {
    mbar_init(bar_q, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_kfull + i, 1);
      mbar_init(bar_vfull + i, 1);
      mbar_init(bar_sfull + i, 1);
      mbar_init(bar_pvdone + i, 1);
    }
    mbar_init(bar_drain, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  pdl_begin();
  // CTA -> (batch, key head, tile, part): a head's tiles together (they share K and V in
  // L2), the last tiles first (under a causal mask they see the most keys)
  const DivMod by_split(blockIdx.x, p.nsplit), by_tile(by_split.quot, p.nqt), by_hk(by_tile.quot, p.Hk);
  const int split = by_split.rem, qt = p.nqt - 1 - by_tile.rem, hk = by_hk.rem, b = by_hk.quot;
  const int t0 = qt * p.TPT, ntok = min(p.TPT, p.Tq - t0);
  // the first loads wait neither for the rest of the arithmetic nor for the other warps
  if (warp == 4 && lane == 0) {
    mbar_arrive_expect_tx(bar_q, NBOX * p.RT * 128);
    for (int i = 0; i < NBOX; ++i) tma_load_4d(sQ + i * QBOX, &tm_q, bar_q, i * 64, hk * p.G, t0, b);
  }
  const WinSeq seq(p, b);
  const int64_t pa = seq.off + t0, pb = pa + ntok - 1;
  const WinSteps<kStep> steps(p, seq.L, pa, pb);
  const int s_begin = part_begin(steps.n, split, p.nsplit);
  const int nsteps = __shfl_sync(0xffffffffu, part_begin(steps.n, split + 1, p.nsplit) - s_begin, 0);
  const int rows = ntok * p.G;                     // rows of this tile that exist
  const int active = (rows + 31) / 32;             // softmax warps that hold any

  // the call's error word: nothing else writes it until a wait of some CTA runs out
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.err = 0;
  // loads in the order of their use: K0 V0 K1 V1 | K(s+2) after QK(s), V(s+2) after PV(s)
  auto load = [&](int s, bool is_v) {
    uint64_t* bar = (is_v ? bar_vfull : bar_kfull) + (s & 1);
    uint8_t* dst = (is_v ? sV : sK) + (s & 1) * SLOT;
    mbar_arrive_expect_tx(bar, SLOT);
    for (int i = 0; i < NBOX; ++i)
      tma_load_4d(dst + i * HBOX, is_v ? &tm_v : &tm_k, bar, i * 64, hk, steps.key0(s_begin + s), b);
  };
  if (warp == 4 && lane == 0) {
    for (int i = 0; i < 2; ++i) mbar_init(bar_pfull + i, 32 * active);
    fence_barrier_init();
    for (int s = 0; s < min(2, nsteps); ++s) {
      load(s, false);
      load(s, true);
    }
  }
  // rows of the tile that no box fills (G does not divide 128): finite scores for them
  for (int i = threadIdx.x; i < NBOX * (128 - p.RT) * 8; i += blockDim.x) {
    const int box = i / ((128 - p.RT) * 8), rest = i % ((128 - p.RT) * 8);
    *reinterpret_cast<uint4*>(sQ + box * QBOX + p.RT * 128 + rest * 16) = make_uint4(0, 0, 0, 0);
  }
  if (p.RT < 128) fence_proxy_async_smem();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tS = tmem;          // scores: slot 0 columns [0, 64), slot 1 [64, 128)
  const uint32_t tO = tmem + 128;    // output accumulator (HD columns)

  if (warp == 4) {
    // ------------------------------------------- TMA producer (after the first loads above)
    if (lane == 0 && nsteps == 0) mbar_wait(bar_q, 0, p.err, kErrWaitDrain);
    if (lane == 0 && nsteps > 0) {
      bool ok = true;
      int last_k = min(2, nsteps) - 1, last_v = last_k;
      for (int s = 0; s + 2 < nsteps; ++s) {
        if (!(ok = mbar_wait(bar_sfull + (s & 1), (s >> 1) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
        load(last_k = s + 2, false);
        if (!(ok = mbar_wait(bar_pvdone + (s & 1), (s >> 1) & 1, p.err, kErrWaitLoad, p.wait_ns))) break;
        load(last_v = s + 2, true);
      }
      if (!ok) {
        // exit path: every issued copy lands before the CTA's shared memory goes away
        mbar_wait(bar_q, 0, p.err, kErrWaitDrain);
        for (int s = max(0, last_k - 1); s <= last_k; ++s) mbar_wait(bar_kfull + (s & 1), (s >> 1) & 1, p.err, kErrWaitDrain);
        for (int s = max(0, last_v - 1); s <= last_v; ++s) mbar_wait(bar_vfull + (s & 1), (s >> 1) & 1, p.err, kErrWaitDrain);
      }
    }
  } else if (warp == 5) {
    // -------------------------------------------------------------- MMA issuer
    if (nsteps > 0) {
      const uint32_t mine = elect_one();
      const uint64_t q_desc = make_sw128_desc(smem_u32(sQ), 16, 1024);
      const uint64_t k_desc = make_sw128_desc(smem_u32(sK), 16, 1024);
      const uint64_t v_desc = make_sw128_desc(smem_u32(sV), HBOX, 1024);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool done = mbar_wait_warp(bar, parity, p.err, kErrWaitMma, p.wait_ns);
        tc_fence_after();
        return done;
      };
      auto issue_qk = [&](int s) {
        const int slot = s & 1;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          mma_bf16_ss_warp(mine, tS + slot * 64, desc_at(q_desc, (k >> 2) * QBOX + (k & 3) * 32),
                           desc_at(k_desc, slot * SLOT + (k >> 2) * HBOX + (k & 3) * 32), IDESC_QK, k > 0);
        tc_commit_warp(mine, bar_sfull + slot);
      };
      bool ok = wait(bar_q, 0);
      for (int s = 0; ok && s < min(2, nsteps); ++s) {
        if (!(ok = wait(bar_kfull + s, 0))) break;
        issue_qk(s);
      }
      for (int s = 0; ok && s < nsteps; ++s) {
        const int slot = s & 1;
        const uint32_t par = (s >> 1) & 1;
        if (!(ok = wait(bar_pfull + slot, par) && wait(bar_vfull + slot, par))) break;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          mma_bf16_ts_warp(mine, tO, tS + slot * 64 + kk * 8, desc_at(v_desc, slot * SLOT + kk * 2048), IDESC_PV,
                           (s > 0 || kk > 0) ? 1u : 0u);
        tc_commit_warp(mine, bar_pvdone + slot);
        if (s + 2 < nsteps) {
          // QK(s+2) overwrites slot s's P: PV(s) has to have read it
          if (!(ok = wait(bar_pvdone + slot, par) && wait(bar_kfull + slot, ((s + 2) >> 1) & 1))) break;
          issue_qk(s + 2);
        }
      }
      // every product issued has completed once bar_drain fires
      tc_commit_warp(mine, bar_drain);
      mbar_wait_warp(bar_drain, 0, p.err, kErrWaitDrain);
    }
  } else {
    // ------------------------------------------------- softmax + epilogue (rows)
    const int row = threadIdx.x;
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const int tok = row / p.G, head = row - tok * p.G;
    const bool live = row < rows;
    const int64_t pos = pa + tok;
    const int hi = live ? win_hi(p, seq.L, pos) : 0, lo = live ? win_lo(p, pos) : 0;
    // every row of the tile sees the keys [full_lo, full_hi), and the sinks before full_hi
    const int full_hi = win_hi(p, seq.L, pa), full_lo = win_lo(p, pb);
    float m_ref = -INFINITY, l_sum = 0.f;
    bool ok = true;
    if (warp < active) {
      for (int s = 0; s < nsteps; ++s) {
        const int slot = s & 1, k0 = steps.key0(s_begin + s);
        if (!(ok = mbar_wait_warp(bar_sfull + slot, (s >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) break;
        tc_fence_after();
        const uint32_t ts = tS + lane_base + slot * 64;
        // before O is rescaled, every P*V issued so far has to be complete
        auto drain = [&]() {
          ok = mbar_wait_warp(bar_pvdone + ((s - 1) & 1), ((s - 1) >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns);
          tc_fence_after();
        };
        uint32_t bits[2];
        if (k0 + kStep <= full_hi && (k0 >= full_lo || k0 + kStep <= p.sinks)) {
          softmax_half<false, false, HD>(ts, tO + lane_base, bits, p.s2, m_ref, l_sum, s > 0, -1, 0.f, 1.f, drain);
        } else {
          bits[0] = live ? win_bits(k0, lo, hi, p.sinks) : 0u;
          bits[1] = live ? win_bits(k0 + 32, lo, hi, p.sinks) : 0u;
          softmax_half<true, false, HD>(ts, tO + lane_base, bits, p.s2, m_ref, l_sum, s > 0, -1, 0.f, 1.f, drain);
          const WinUnseen unseen(p, seq.L, pa, pb, k0, kStep);
          if (ok && unseen.any(kStep)) {
            if ((ok = mbar_wait_warp(bar_vfull + slot, (s >> 1) & 1, p.err, kErrWaitSoftmax, p.wait_ns))) {
              for (int i = row; i < kStep * NBOX * 8; i += 32 * active) {
                const int r = i / (NBOX * 8), x = i % (NBOX * 8);
                if ((r >= unseen.a0 && r < unseen.a1) || r >= unseen.b0)
                  *reinterpret_cast<uint4*>(sV + slot * SLOT + (x >> 3) * HBOX + r * 128 + (x & 7) * 16) =
                      make_uint4(0, 0, 0, 0);
              }
              fence_proxy_async_smem();
            }
          }
        }
        if (!ok) break;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar_pfull + slot);
      }
      if (ok) {
        // (without steps: the load of Q, whose tile takes the zeros, has landed)
        ok = nsteps > 0 ? mbar_wait_warp(bar_pvdone + ((nsteps - 1) & 1), ((nsteps - 1) >> 1) & 1, p.err,
                                         kErrWaitEpilogue, p.wait_ns)
                        : mbar_wait_warp(bar_q, 0, p.err, kErrWaitEpilogue, p.wait_ns);
        tc_fence_after();
      }
      const bool none = l_sum == 0.f;              // nothing seen (a NaN row is not that)
      const int64_t orow = ((int64_t)b * p.Tq + t0 + tok) * p.H + hk * p.G + head;
      if (ok && p.nsplit > 1) {
        const int64_t part = (int64_t)split * p.B * p.Tq * p.H + orow;
        if (live) p.part_ml[part] = make_float2(none ? -INFINITY : m_ref, l_sum);
        for (int c = 0; nsteps > 0 && c < HD / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(tO + lane_base + c * 32, r);
          tmem_wait_ld();
          if (live && !none) {
            float4* dst = reinterpret_cast<float4*>(p.part_o + part * HD + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i] = make_float4(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]),
                                   __uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
          }
        }
      } else if (ok) {
        // O / l -> bf16 -> swizzled staging (the free Q buffer) -> TMA store
        const float inv = none ? 0.f : 1.f / l_sum;
        if (live && p.lse)
          p.lse[((int64_t)b * p.H + hk * p.G + head) * p.Tq + t0 + tok] =
              none ? -INFINITY : (m_ref + log2f(l_sum)) * 0.69314718055994531f;
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t r[32];
          if (nsteps > 0) {
            tmem_ld32(tO + lane_base + c * 32, r);
            tmem_wait_ld();
          }
          const int box = (c * 32) / 64, chunk0 = ((c * 32) % 64) >> 3;
          if (row < p.RT) {
#pragma unroll
            for (int v4 = 0; v4 < 4; ++v4) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = none ? 0u : pack_bf16x2(__uint_as_float(r[v4 * 8 + 2 * i]) * inv,
                                               __uint_as_float(r[v4 * 8 + 2 * i + 1]) * inv);
              *reinterpret_cast<uint4*>(sQ + box * QBOX + row * 128 + (((chunk0 + v4) ^ (row & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        fence_proxy_async_smem();
      }
    }
    // every warp's rows are staged (or its wait failed, and nothing is stored)
    if (named_bar_all(1, 128, ok) && p.nsplit == 1 && threadIdx.x == 0) {
      for (int i = 0; i < NBOX; ++i) tma_store_4d(&tm_o, sQ + i * QBOX, i * 64, hk * p.G, t0, b);
      bulk_commit_group();
      bulk_wait_group_read0();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// The parts of the key axis joined: with M the largest of the parts' maxima m_i,
//   O = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.
// One warp per row; lane i weighs parts i and i + 32, so that the parts' sums are loaded without
// waiting for one another (one part after the other took 7 us for 7 parts, all of it latency). A part
// that saw nothing has l = 0 and no sums in memory.
template <int HD>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ WinParams p) {
  pdl_begin();
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.B * p.Tq * p.H;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  float2 ml[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    ml[i] = lane + 32 * i < p.nsplit ? p.part_ml[(lane + 32 * i) * rows + row] : make_float2(-INFINITY, 0.f);
  float top = fmaxf(ml[0].x, ml[1].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  float w[2], l = 0.f, acc[E];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = ml[i].y == 0.f ? 0.f : fast_exp2(ml[i].x - top);
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  const float* src = p.part_o + row * HD + lane * E;
#pragma unroll 8
  for (int i = 0; i < p.nsplit; ++i) {
    const float wi = __shfl_sync(0xffffffffu, i < 32 ? w[0] : w[1], i & 31);
    const float li = __shfl_sync(0xffffffffu, i < 32 ? ml[0].y : ml[1].y, i & 31);
    l = fmaf(wi, li, l);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    if (li != 0.f) {
      if (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src + i * rows * HD);
        v[0] = x.x;
        v[1] = x.y;
        v[E - 2] = x.z;
        v[E - 1] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(src + i * rows * HD);
        v[0] = x.x;
        v[1] = x.y;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(wi, v[e], acc[e]);
  }
  const bool none = l == 0.f;
  const float inv = none ? 0.f : 1.f / l;
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + row * HD + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = pack_bf16x2(acc[e] * inv, acc[e + 1] * inv);
  if (p.lse && lane == 0) {
    const int64_t bt = row / p.H, b = bt / p.Tq;
    p.lse[(b * p.H + (row - bt * p.H)) * p.Tq + (bt - b * p.Tq)] =
        none ? -INFINITY : (top + log2f(l)) * 0.69314718055994531f;
  }
}

template <int HD>
cudaError_t launch_t(const WinMaps& m, const WinParams& p, cudaStream_t st) {
  auto kern = window_fwd_kernel<HD>;
  // at least ~100 KB, so that at most two CTAs (512 TMEM columns) share an SM
  constexpr size_t need = (HD / 64) * (128 * 128 + 4 * kStep * 128) + 256 + 1024;
  const size_t smem = need < 100 * 1024 ? 100 * 1024 : need;
  static std::atomic<uint64_t> allowed{0};
  cudaError_t e = allow_smem(kern, smem, allowed);
  if (e != cudaSuccess) return e;
  const int64_t grid = (int64_t)p.B * p.Hk * p.nqt * p.nsplit;
  e = launch_pdl(kern, dim3((unsigned)grid), dim3(192), smem, st, m.q, m.k, m.v, m.o, p);
  if (e != cudaSuccess || p.nsplit == 1) return e;
  const int64_t rows = (int64_t)p.B * p.Tq * p.H;
  return launch_pdl(window_join_kernel<HD>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p);
}

}  // namespace

cudaError_t launch_window_fwd(int hd, const WinMaps& m, const WinParams& p, cudaStream_t st) {
  return hd == 128 ? launch_t<128>(m, p, st) : launch_t<64>(m, p, st);
}

}  // namespace solb200
