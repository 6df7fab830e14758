// Host side of the C ABI's layer operators (include/solb200.h): head norms with the position
// rotation, and windowed attention with sinks. Argument checks, the workspace plan, tensor
// maps and launches; nothing here allocates device memory or synchronises.
#include <string>

#include <nvtx3/nvToolsExt.h>

#include "internal.h"
#include "norm_rope.cuh"
#include "solb200.h"
#include "window.cuh"

using namespace solb200;

namespace {

struct NvtxRange {
  explicit NvtxRange(const char* name) { nvtxRangePushA(name); }
  ~NvtxRange() { nvtxRangePop(); }
  NvtxRange(const NvtxRange&) = delete;
  NvtxRange& operator=(const NvtxRange&) = delete;
};

int32_t invalid(const char* msg) { return set_last_error(SOLB200_ERR_INVALID, msg); }

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

constexpr int64_t kMost = (int64_t)1 << 30;

// A [B, T, heads, D] tensor read with 16-byte accesses: base and the strides of dimensions
// longer than one are multiples of 16 bytes (0 repeats the dimension).
int32_t check_rows16(const char* name, const void* ptr, const int64_t* s, int64_t B, int64_t T, int64_t H, int esize,
                     bool positive) {
  if (!ptr || !s) return set_last_error(SOLB200_ERR_INVALID, std::string(name) + ": null pointer");
  if (!aligned16(ptr))
    return set_last_error(SOLB200_ERR_ALIGNMENT, std::string(name) + ": base not 16-byte aligned");
  const int64_t n[3] = {B, T, H};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] < (positive ? 1 : 0) || s[i] > ((int64_t)1 << 40) || (s[i] * esize) % 16))
      return set_last_error(SOLB200_ERR_ALIGNMENT,
                            std::string(name) + ": batch/token/head strides must be multiples of 16 bytes" +
                                (positive ? " above 0" : ", 0 or above"));
  return SOLB200_OK;
}

// ------------------------------------------------------- head norms and rotation

// batch x tokens x heads rows are numbered with 32-bit integers
bool rope_rows_fit(int64_t B, int64_t T, int64_t H) {
  return B <= kMost && T <= kMost && H <= 65536 && B * T <= kMost && B * T * H <= kMost;
}

int32_t rope_params(RopeParams& p, const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* wq,
                    const void* wk, int32_t weight_dtype, const float* cos, const float* sin, const int64_t* ts,
                    int64_t B, int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t R, int32_t dtype, float eps,
                    int32_t interleaved) {
  int32_t rc = check_sm100();
  if (rc) return rc;
  if (B < 1 || T < 1 || H < 1 || Hk < 1) return invalid("batch, tokens and heads must be >= 1");
  if (!rope_rows_fit(B, T, H) || !rope_rows_fit(B, T, Hk)) return invalid("more than 2^30 rows in q or k");
  if (D < 8 || D > 256 || D % 8) return invalid("head_dim must be a multiple of 8 in [8, 256]");
  if (dtype < 0 || dtype > 2) return invalid("dtype must be SOLB200_BF16, SOLB200_F16 or SOLB200_F32");
  if (weight_dtype != dtype && weight_dtype != kDtypeF32)
    return invalid("weights must have the tensors' dtype or be float32");
  const int step = interleaved ? 8 : 16;
  if (R < step || R > D || R % step)
    return invalid("rotated elements must be a multiple of 8 (interleaved) or 16 (halves) in head_dim");
  if (!(eps >= 0.f)) return invalid("eps must be >= 0");
  const int es = dtype == kDtypeF32 ? 4 : 2;
  if ((rc = check_rows16("q", q, qs, B, T, H, es, false))) return rc;
  if ((rc = check_rows16("k", k, ks, B, T, Hk, es, false))) return rc;
  if (!wq || !wk || !cos || !sin || !ts) return invalid("weights or tables: null pointer");
  if (!aligned16(cos) || !aligned16(sin) || (B > 1 && (ts[0] % 4 || ts[0] < 0)) || (T > 1 && (ts[1] % 4 || ts[1] < 0)))
    return set_last_error(SOLB200_ERR_ALIGNMENT, "cos / sin: base or row strides not multiples of 16 bytes");
  p = RopeParams{};
  p.t[0].x = q; p.t[0].weight = wq; p.t[0].heads = (int)H;
  p.t[1].x = k; p.t[1].weight = wk; p.t[1].heads = (int)Hk;
  for (int i = 0; i < 3; ++i) {
    p.t[0].xs[i] = qs[i];
    p.t[1].xs[i] = ks[i];
  }
  p.cos = cos; p.sin = sin; p.ts[0] = ts[0]; p.ts[1] = ts[1];
  p.B = (int)B; p.T = (int)T; p.D = (int)D; p.R = (int)R; p.eps = eps;
  return SOLB200_OK;
}

// ------------------------------------------------------------- windowed attention

constexpr int kSlots = 148 * 2;   // forward CTAs resident on the GPU
constexpr int kStepKeys = 64, kTileRows = 128;

// Parts of the key axis: the count with the least estimated time, in steps of 64 keys of one CTA
// (about a microsecond, whether the tensor cores or memory set the pace). The CTAs run in waves
// of kSlots, each wave as long as a part of `steps` steps (the most that the shapes and bounds allow;
// lengths live on the device) but together no shorter than the GPU needs at nine tenths of its slots,
// and kOpen steps to open and close each; the joining kernel takes kJoin and reads what the parts
// wrote (`row_bytes` each, there and back at 5 MB a step), a third of a step per part.
// Measured (us, short bursts): 8 tiles x 64 steps 53 whole, 17.6 in 9 parts, 26.9 in 60; 40 tiles x 4096
// steps 2841 whole, 755 in 7, 946 in 9 (two waves), 784 in 22; 520 tiles x 195 steps 451 whole, 479 in 2.
int window_splits(int64_t tiles, int64_t steps, int64_t row_bytes) {
  constexpr double kOpen = 3, kJoin = 2;
  constexpr int kMostSplits = 64;
  const double whole = (double)tiles * steps / (0.9 * kSlots);
  int best = 1;
  double best_cost = 0;
  for (int n = 1; n <= kMostSplits && (n == 1 || n * 2 <= steps); ++n) {
    const int64_t waves = (tiles * n + kSlots - 1) / kSlots;
    const double run = (double)waves * ((steps + n - 1) / n);
    const double cost = (run > whole ? run : whole) + waves * kOpen +
                        (n > 1 ? kJoin + n * (0.33 + 2.0 * row_bytes / 5e6) : 0);
    if (n == 1 || cost < best_cost) {
      best_cost = cost;
      best = n;
    }
  }
  return best;
}

// The gradient's parts, in steps of one CTA (about 2 us each, one CTA per SM): `most` steps of the longest
// tile, `mean` of all of them, kOpen to open and close a CTA; the joining kernel takes kJoin and moves
// part_bytes per part there and back (8 MB a step). Measured in short bursts, forward and gradient (us): 2 heads x 2000
// causal tokens 84 whole, 65 in parts; 2 x 4000 in a window of 200 with 64 sinks 102 and 69; 8 x 800 53 and 59.
int gradient_splits(int64_t tiles, int64_t most, double mean, int64_t part_bytes) {
  constexpr double kOpen = 3, kJoin = 3.5, kSms = 148;
  int best = 1;
  double best_cost = 0;
  for (int n = 1; n <= 16 && (n == 1 || n * 2 <= most); ++n) {
    const double longest = (double)((most + n - 1) / n) + kOpen, all = (double)tiles * (mean + n * kOpen) / kSms;
    const double cost = (longest > all ? longest : all) + (n > 1 ? kJoin + n * 2.0 * part_bytes / 8e6 : 0);
    if (n == 1 || cost < best_cost) {
      best_cost = cost;
      best = n;
    }
  }
  return best;
}

struct WinPlan {
  WinParams p;
  int64_t off_ml, off_o, off_lse, off_delta, off_dq, off_dkv, fwd_bytes, bwd_bytes;
};

int32_t window_plan(WinPlan& w, int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hk, int64_t D, int64_t left,
                    int64_t right, int64_t sinks) {
  if (B < 1 || Tq < 1 || Tk < 1 || H < 1 || Hk < 1) return invalid("batch, tokens and heads must be >= 1");
  if (D != 64 && D != 128) return invalid("head_dim must be 64 or 128");
  if (B > 65536 || Tq > kMost || Tk > kMost || H > 65536) return invalid("batch, tokens or heads too large");
  if (H % Hk || H / Hk > kTileRows) return invalid("heads must be a multiple of key heads, at most 128 times as many");
  if (left < -1 || right < -1 || sinks < 0) return invalid("left and right must be >= -1 (-1: no bound), sinks >= 0");
  WinParams& p = w.p;
  p = WinParams{};
  p.B = (int)B; p.Tq = (int)Tq; p.Tk = (int)Tk; p.H = (int)H; p.Hk = (int)Hk;
  p.G = (int)(H / Hk);
  p.TPT = kTileRows / p.G;
  p.RT = p.TPT * p.G;
  p.nqt = (int)((Tq + p.TPT - 1) / p.TPT);
  p.nkt = (int)((Tk + kTileRows - 1) / kTileRows);
  const int64_t far = (int64_t)1 << 40;   // past every position
  p.left = left > far ? far : left;
  p.right = right > far ? far : right;
  p.sinks = (int)(sinks < Tk ? sinks : Tk);
  const int64_t tiles = B * Hk * p.nqt;
  if (tiles >= ((int64_t)1 << 24) || B * Hk * p.nkt >= ((int64_t)1 << 31)) return invalid("too many tiles");
  int64_t keys = Tk;
  if (left >= 0 && right >= 0 && left < Tk && right < Tk) {
    const int64_t span = p.sinks + left + right + (Tq < p.TPT ? Tq : p.TPT);
    if (span < keys) keys = span;
  }
  p.nsplit = window_splits(tiles, (keys + kStepKeys - 1) / kStepKeys + 1, B * Tq * H * (D * 4 + 8));
  auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
  int64_t cur = 256;   // the error word
  w.off_ml = cur;
  if (p.nsplit > 1) cur = up(cur + p.nsplit * B * Tq * H * (int64_t)sizeof(float2));
  w.off_o = cur;
  if (p.nsplit > 1) cur = up(cur + p.nsplit * B * Tq * H * D * (int64_t)sizeof(float));
  w.fwd_bytes = cur;
  const int64_t slots = tiles * kTileRows * (int64_t)sizeof(float);
  w.off_lse = 256;
  w.off_delta = w.off_lse + slots;   // (tiles of 128 rows: 512-byte multiples)
  // gradient: key steps of a query tile, query tiles of a key tile; a causal call without a left bound has
  // half of them on average, and sinks are seen by every tile
  const int64_t steps_q = (keys + kTileRows - 1) / kTileRows + 1;
  const bool bounded = left >= 0 && right >= 0 && left < Tq && right < Tq;
  const int64_t near = bounded ? (kTileRows + left + right) / p.TPT + 2 : p.nqt;
  const int64_t tiles_k = near < p.nqt ? near : p.nqt;
  const double half = left < 0 && right >= 0 ? 0.5 : 1.0;
  p.split_q = gradient_splits(tiles, steps_q < p.nkt ? steps_q : p.nkt, half * (steps_q < p.nkt ? steps_q : p.nkt),
                              B * Tq * H * D * 4);
  p.split_k = gradient_splits(B * Hk * p.nkt, p.sinks > 0 ? p.nqt : tiles_k, half * tiles_k, 2 * B * Tk * Hk * D * 4);
  cur = up(w.off_delta + slots);
  w.off_dq = cur;
  if (p.split_q > 1) cur = up(cur + p.split_q * B * Tq * H * D * (int64_t)sizeof(float));
  w.off_dkv = cur;
  if (p.split_k > 1) cur = up(cur + 2 * p.split_k * B * Tk * Hk * D * (int64_t)sizeof(float));
  w.bwd_bytes = cur;
  return SOLB200_OK;
}

int32_t window_common(WinPlan& w, WinMaps& m, const void* q, const int64_t* qs, const void* k, const int64_t* ks,
                      const void* v, const int64_t* vs, const int32_t* lengths, const int32_t* offsets, int64_t B,
                      int64_t Tq, int64_t Tk, int64_t H, int64_t Hk, int64_t D, float scale, int key_box,
                      void* workspace, int64_t workspace_bytes, int64_t need) {
  int32_t rc;
  if ((rc = check_rows16("q", q, qs, B, Tq, H, 2, true))) return rc;
  if ((rc = check_rows16("k", k, ks, B, Tk, Hk, 2, true))) return rc;
  if ((rc = check_rows16("v", v, vs, B, Tk, Hk, 2, true))) return rc;
  if (!(scale > 0.f)) return invalid("scale must be > 0");
  if (reinterpret_cast<uintptr_t>(lengths) % 4 || reinterpret_cast<uintptr_t>(offsets) % 4)
    return set_last_error(SOLB200_ERR_ALIGNMENT, "lengths / offsets: not aligned to 4 bytes");
  if (!workspace || workspace_bytes < need)
    return set_last_error(SOLB200_ERR_WORKSPACE, "workspace missing or too small (" + std::to_string(workspace_bytes) +
                                                     " of " + std::to_string(need) + " bytes)");
  if (!aligned16(workspace)) return set_last_error(SOLB200_ERR_ALIGNMENT, "workspace not 16-byte aligned");
  WinParams& p = w.p;
  p.lengths = lengths;
  p.offsets = offsets;
  p.scale = scale;
  p.s2 = scale * 1.4426950408889634f;
  p.err = static_cast<int*>(workspace);
  p.wait_ns = current_wait_ns();
  if ((rc = bthd_map(&m.q, q, D, H, Tq, B, qs, p.G, p.TPT, "q"))) return rc;
  if ((rc = bthd_map(&m.k, k, D, Hk, Tk, B, ks, 1, key_box, "k"))) return rc;
  return bthd_map(&m.v, v, D, Hk, Tk, B, vs, 1, key_box, "v");
}

}  // namespace

extern "C" {

int32_t solb200_qk_norm_rope(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                             const void* q_weight, const void* k_weight, int32_t weight_dtype, const float* cos,
                             const float* sin, const int64_t* table_strides, void* q_out, void* k_out, int64_t batch,
                             int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotated,
                             int32_t dtype, float eps, int32_t interleaved, void* stream) {
  RopeParams p;
  const int32_t rc = rope_params(p, q, q_strides, k, k_strides, q_weight, k_weight, weight_dtype, cos, sin,
                                 table_strides, batch, tokens, heads, kv_heads, head_dim, rotated, dtype, eps,
                                 interleaved);
  if (rc) return rc;
  if (!q_out || !k_out || !aligned16(q_out) || !aligned16(k_out))
    return set_last_error(SOLB200_ERR_ALIGNMENT, "outputs: null or not 16-byte aligned");
  p.t[0].out = q_out;
  p.t[1].out = k_out;
  NvtxRange r("solb200.qk_norm_rope");
  const cudaError_t e = launch_norm_rope(p, dtype, weight_dtype, interleaved != 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SOLB200_OK : set_cuda_error(e, "qk_norm_rope launch");
}

int32_t solb200_qk_norm_rope_backward_workspace(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                int64_t head_dim, int64_t* bytes) {
  if (!bytes) return invalid("null pointer");
  if (batch < 1 || tokens < 1 || heads < 1 || kv_heads < 1) return invalid("batch, tokens and heads must be >= 1");
  if (!rope_rows_fit(batch, tokens, heads) || !rope_rows_fit(batch, tokens, kv_heads))
    return invalid("more than 2^30 rows in q or k");
  if (head_dim < 8 || head_dim > 256 || head_dim % 8) return invalid("head_dim must be a multiple of 8 in [8, 256]");
  *bytes = (int64_t)norm_rope_backward_ctas(batch, tokens, heads, kv_heads, (int)head_dim) * head_dim *
           (int64_t)sizeof(float);
  return SOLB200_OK;
}

int32_t solb200_qk_norm_rope_backward(const void* dq_out, const int64_t* dq_out_strides, const void* dk_out,
                                      const int64_t* dk_out_strides, const void* q, const int64_t* q_strides,
                                      const void* k, const int64_t* k_strides, const void* q_weight,
                                      const void* k_weight, int32_t weight_dtype, const float* cos, const float* sin,
                                      const int64_t* table_strides, void* dq, void* dk, void* dq_weight,
                                      void* dk_weight, int64_t batch, int64_t tokens, int64_t heads,
                                      int64_t kv_heads, int64_t head_dim, int64_t rotated, int32_t dtype, float eps,
                                      int32_t interleaved, void* workspace, int64_t workspace_bytes, void* stream) {
  RopeParams p;
  int32_t rc = rope_params(p, q, q_strides, k, k_strides, q_weight, k_weight, weight_dtype, cos, sin, table_strides,
                           batch, tokens, heads, kv_heads, head_dim, rotated, dtype, eps, interleaved);
  if (rc) return rc;
  const int es = dtype == kDtypeF32 ? 4 : 2;
  if ((rc = check_rows16("dq_out", dq_out, dq_out_strides, batch, tokens, heads, es, false))) return rc;
  if ((rc = check_rows16("dk_out", dk_out, dk_out_strides, batch, tokens, kv_heads, es, false))) return rc;
  if (!dq || !dk || !aligned16(dq) || !aligned16(dk) || !dq_weight || !dk_weight)
    return set_last_error(SOLB200_ERR_ALIGNMENT, "gradients: null or not 16-byte aligned");
  int64_t need = 0;
  if ((rc = solb200_qk_norm_rope_backward_workspace(batch, tokens, heads, kv_heads, head_dim, &need))) return rc;
  if (!workspace || workspace_bytes < need)
    return set_last_error(SOLB200_ERR_WORKSPACE, "workspace missing or too small");
  if (!aligned16(workspace)) return set_last_error(SOLB200_ERR_ALIGNMENT, "workspace not 16-byte aligned");
  p.t[0].dy = dq_out; p.t[0].out = dq; p.t[0].dweight = dq_weight;
  p.t[1].dy = dk_out; p.t[1].out = dk; p.t[1].dweight = dk_weight;
  for (int i = 0; i < 3; ++i) {
    p.t[0].dys[i] = dq_out_strides[i];
    p.t[1].dys[i] = dk_out_strides[i];
  }
  p.partial = static_cast<float*>(workspace);
  NvtxRange r("solb200.qk_norm_rope_backward");
  const cudaError_t e =
      launch_norm_rope_backward(p, dtype, weight_dtype, interleaved != 0, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SOLB200_OK : set_cuda_error(e, "qk_norm_rope backward launch");
}

int32_t solb200_window_attn_workspace(int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads,
                                      int64_t kv_heads, int64_t head_dim, int64_t left, int64_t right, int64_t sinks,
                                      int32_t backward, int64_t* bytes) {
  if (!bytes) return invalid("null pointer");
  WinPlan w;
  const int32_t rc = window_plan(w, batch, q_tokens, kv_tokens, heads, kv_heads, head_dim, left, right, sinks);
  if (rc) return rc;
  *bytes = backward ? w.bwd_bytes : w.fwd_bytes;
  return SOLB200_OK;
}

int32_t solb200_window_attn(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, void* out, float* lse, const int32_t* lengths,
                            const int32_t* offsets, int64_t batch, int64_t q_tokens, int64_t kv_tokens, int64_t heads,
                            int64_t kv_heads, int64_t head_dim, int64_t left, int64_t right, int64_t sinks,
                            float scale, void* workspace, int64_t workspace_bytes, void* stream) {
  int32_t rc = check_sm100();
  if (rc) return rc;
  WinPlan w;
  WinMaps m;
  if ((rc = window_plan(w, batch, q_tokens, kv_tokens, heads, kv_heads, head_dim, left, right, sinks))) return rc;
  if (!out || !aligned16(out)) return set_last_error(SOLB200_ERR_ALIGNMENT, "out: null or not 16-byte aligned");
  if ((rc = window_common(w, m, q, q_strides, k, k_strides, v, v_strides, lengths, offsets, batch, q_tokens,
                          kv_tokens, heads, kv_heads, head_dim, scale, kStepKeys, workspace, workspace_bytes,
                          w.fwd_bytes)))
    return rc;
  WinParams& p = w.p;
  const int64_t os[3] = {q_tokens * heads * head_dim, heads * head_dim, head_dim};
  if ((rc = bthd_map(&m.o, out, head_dim, heads, q_tokens, batch, os, p.G, p.TPT, "out"))) return rc;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(workspace) + w.off_ml);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.off_o);
  NvtxRange r("solb200.window_attn");
  const cudaError_t e = launch_window_fwd((int)head_dim, m, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SOLB200_OK : set_cuda_error(e, "window_attn launch");
}

int32_t solb200_window_attn_backward(const void* dout, const int64_t* dout_strides, const void* q,
                                     const int64_t* q_strides, const void* k, const int64_t* k_strides, const void* v,
                                     const int64_t* v_strides, const void* out, const int64_t* out_strides,
                                     const float* lse, void* dq, void* dk, void* dv, const int32_t* lengths,
                                     const int32_t* offsets, int64_t batch, int64_t q_tokens, int64_t kv_tokens,
                                     int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t left, int64_t right,
                                     int64_t sinks, float scale, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  int32_t rc = check_sm100();
  if (rc) return rc;
  WinPlan w;
  WinMaps m;
  if ((rc = window_plan(w, batch, q_tokens, kv_tokens, heads, kv_heads, head_dim, left, right, sinks))) return rc;
  if ((rc = check_rows16("dout", dout, dout_strides, batch, q_tokens, heads, 2, true))) return rc;
  if ((rc = check_rows16("out", out, out_strides, batch, q_tokens, heads, 2, true))) return rc;
  if (!lse || !dq || !dk || !dv || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return set_last_error(SOLB200_ERR_ALIGNMENT, "lse or gradients: null or not 16-byte aligned");
  if ((rc = window_common(w, m, q, q_strides, k, k_strides, v, v_strides, lengths, offsets, batch, q_tokens,
                          kv_tokens, heads, kv_heads, head_dim, scale, kTileRows, workspace, workspace_bytes,
                          w.bwd_bytes)))
    return rc;
  WinParams& p = w.p;
  if ((rc = bthd_map(&m.dout, dout, head_dim, heads, q_tokens, batch, dout_strides, p.G, p.TPT, "dout"))) return rc;
  const int64_t D = head_dim, dqs[3] = {q_tokens * heads * D, heads * D, D};
  const int64_t dks[3] = {kv_tokens * kv_heads * D, kv_heads * D, D};
  if ((rc = bthd_map(&m.o, dq, D, heads, q_tokens, batch, dqs, p.G, p.TPT, "dq"))) return rc;
  if ((rc = bthd_map(&m.dk, dk, D, kv_heads, kv_tokens, batch, dks, 1, kTileRows, "dk"))) return rc;
  if ((rc = bthd_map(&m.dv, dv, D, kv_heads, kv_tokens, batch, dks, 1, kTileRows, "dv"))) return rc;
  p.out = static_cast<__nv_bfloat16*>(dq);
  p.dk = static_cast<__nv_bfloat16*>(dk);
  p.dv = static_cast<__nv_bfloat16*>(dv);
  p.part_dq = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.off_dq);
  p.part_dkv = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.off_dkv);
  p.lse_in = lse;
  p.o_in = static_cast<const __nv_bfloat16*>(out);
  p.do_in = static_cast<const __nv_bfloat16*>(dout);
  for (int i = 0; i < 3; ++i) {
    p.os[i] = out_strides[i];
    p.dos[i] = dout_strides[i];
  }
  p.rows_lse = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.off_lse);
  p.rows_delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + w.off_delta);
  NvtxRange r("solb200.window_attn_backward");
  const cudaError_t e = launch_window_bwd((int)head_dim, m, p, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? SOLB200_OK : set_cuda_error(e, "window_attn backward launch");
}

}  // extern "C"
