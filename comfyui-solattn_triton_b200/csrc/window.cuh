// Windowed attention with sinks (solb200_window_attn and its gradient): what query sees
// which key, and the tiles that follow from it, shared by the kernels (window_fwd.cu,
// window_bwd.cu) and the entry points (layer_api.cu).
//
// Query i of sequence b sits at position p = off_b + i. It sees key j when
//   0 <= j < L_b,   j <= p + right,   and (j >= p - left or j < sinks).
// The right bound holds for the sinks too, so a causal call (right = 0) stays causal.
#pragma once

#include "common.cuh"

namespace solb200 {

struct WinParams {
  int B, Tq, Tk, H, Hk;
  int G;                    // query heads per key head (H / Hk), 1..128
  int TPT, RT, nqt;         // tokens and rows (TPT * G) of a query tile, tiles per (b, key head)
  int nsplit;               // forward: parts of the key axis, joined by a second kernel
  int64_t left, right;      // < 0: no bound
  int sinks;
  const int* lengths;       // [B] or null (Tk)
  const int* offsets;       // [B] or null (L - Tq)
  float scale, s2;          // softmax scale, and times log2(e)
  int* err;
  uint64_t wait_ns;
  __nv_bfloat16* out;       // split forward, split dq: dense [B, Tq, H, D]
  float* lse;               // forward: [B, H, Tq] or null
  float* part_o;            // split forward: [nsplit, B, Tq, H, D] unnormalised sums
  float2* part_ml;          // split forward: [nsplit, B, Tq, H] (row maximum in log2 units, row sum)
  // backward
  const float* lse_in;      // [B, H, Tq]
  const __nv_bfloat16 *o_in, *do_in;
  int64_t os[3], dos[3];    // strides {batch, token, head}
  float* rows_lse;          // [B, Hk, nqt, 128] -lse * log2(e) by tile row (-inf: nothing seen, or no row)
  float* rows_delta;        // [B, Hk, nqt, 128] -sum(dO * O) by tile row
  int nkt;                  // key tiles of 128
  int split_q, split_k;     // parts of a query tile's key steps (dq) and of a key tile's query tiles (dk, dv)
  float* part_dq;           // [split_q, B, Tq, H, D] if split_q > 1
  float* part_dkv;          // [split_k, 2 (dv, dk), B, Tk, Hk, D] if split_k > 1
  __nv_bfloat16 *dk, *dv;   // what the parts are joined into (dq: out)
};

// A sequence's place: valid keys and the position of query 0.
struct WinSeq {
  int L;
  int64_t off;
  __device__ WinSeq(const WinParams& p, int b) {
    L = p.lengths ? min(max(__ldg(p.lengths + b), 0), p.Tk) : p.Tk;
    off = p.offsets ? (int64_t)__ldg(p.offsets + b) : (int64_t)L - p.Tq;
  }
};

// Quotient and remainder of non-negative numbers (unsigned division is the cheaper one); by 1 without any.
__device__ __forceinline__ int udiv(int a, int b) { return b == 1 ? a : (int)((unsigned)a / (unsigned)b); }
struct DivMod {
  int quot, rem;
  __device__ __forceinline__ DivMod(int a, int b) : quot(udiv(a, b)), rem(a - quot * b) {}
};
// First of n steps that part `i` of `parts` takes (n and i * n below 2^31).
__device__ __forceinline__ int part_begin(int n, int i, int parts) { return parts == 1 ? (i ? n : 0) : udiv(n * i, parts); }

__device__ __forceinline__ int clamp_to(int64_t x, int lo, int hi) {
  return (int)(x < lo ? lo : (x > hi ? hi : x));
}

// First key past the right bound, and first key inside the left bound, of a query at `pos`.
__device__ __forceinline__ int win_hi(const WinParams& p, int L, int64_t pos) {
  return p.right < 0 ? L : clamp_to(pos + p.right + 1, 0, L);
}
__device__ __forceinline__ int win_lo(const WinParams& p, int64_t pos) {
  return p.left < 0 ? 0 : clamp_to(pos - p.left, 0, p.Tk);
}

// The runs of STEP keys that the queries at positions [pa, pb] see any key of: steps
// [0, n1) hold the sinks, steps [start, start + n - n1) the window.
template <int STEP>
struct WinSteps {
  int n1, start, n;
  __device__ WinSteps(const WinParams& p, int L, int64_t pa, int64_t pb) {
    const int hi = win_hi(p, L, pb), lo = win_lo(p, pa);
    const int end = (hi + STEP - 1) / STEP;
    n1 = (min(p.sinks, hi) + STEP - 1) / STEP;
    start = lo / STEP;
    if (start <= n1) {
      n1 = 0;
      start = 0;
      n = end;
    } else {
      n = n1 + max(0, end - start);
    }
  }
  __device__ int key0(int s) const { return (s < n1 ? s : start + s - n1) * STEP; }
};

__device__ __forceinline__ uint32_t win_low_bits(int n) {
  return n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : ((1u << n) - 1u));
}

// Bits of the 32 keys from k0 on that a query with bounds [lo, hi) sees.
__device__ __forceinline__ uint32_t win_bits(int k0, int lo, int hi, int sinks) {
  return win_low_bits(hi - k0) & (~win_low_bits(lo - k0) | win_low_bits(sinks - k0));
}

// Of the n keys from k0 on, those that no query at positions [pa, pb] sees: [a0, a1) between the
// sinks and the window, [b0, n) past it. Their keys and values may hold anything, NaN included,
// and 0 * NaN would reach the tile's sums: their rows are zeroed in shared memory.
struct WinUnseen {
  int a0, a1, b0;
  __device__ WinUnseen(const WinParams& p, int L, int64_t pa, int64_t pb, int k0, int n) {
    const int hi = win_hi(p, L, pb);
    a0 = max(0, min(n, min(p.sinks, hi) - k0));   // (sinks past the visible end are not seen either)
    a1 = max(a0, min(n, win_lo(p, pa) - k0));
    b0 = hi < p.Tk ? max(a1, min(n, hi - k0)) : n;   // (past Tk the loads fill in zeros)
  }
  __device__ bool any(int n) const { return a1 > a0 || b0 < n; }
};

// Of the TPT tokens from t0 on, those outside [t0, t1) (counted from t0) see nothing: they come
// before the first key by more than the right bound, or past the last one by more than the left.
struct WinBlind {
  int t0, t1;
  __device__ WinBlind(const WinParams& p, const WinSeq& seq, int first) {
    t0 = p.right < 0 ? 0 : clamp_to(-p.right - seq.off - first, 0, p.TPT);
    t1 = p.left < 0 || p.sinks > 0 ? p.TPT : clamp_to(seq.L + p.left - seq.off - first, 0, p.TPT);
  }
  __device__ bool any(const WinParams& p) const { return t0 > 0 || t1 < p.TPT; }
};

struct WinMaps {
  CUtensorMap q, k, v, o;        // o: the forward's output, the gradient's dq
  CUtensorMap dout, dk, dv;      // gradient
};

cudaError_t launch_window_fwd(int hd, const WinMaps& m, const WinParams& p, cudaStream_t st);
cudaError_t launch_window_bwd(int hd, const WinMaps& m, const WinParams& p, cudaStream_t st);

}  // namespace solb200
