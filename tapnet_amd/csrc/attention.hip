// libtapir_hip: layer normalisation, rotary positions and cross attention -- argument checks, kernel choice and the C ABI
// (include/tapir_hip.h).  A translation unit of its own: nothing here touches a context's weights or workspaces.
#include "attention.hpp"

#include <math.h>
#include <stdio.h>

#include <algorithm>

#include "context.hpp"
#include "layer_norm.hpp"
#include "rotary.hpp"

using namespace tapir;

namespace {

#define OP_TRY(c, expr)                                                                   \
  do {                                                                                    \
    const hipError_t e_ = (expr);                                                         \
    if (e_ != hipSuccess) return ctx_fail((c), TAPIR_ERR_HIP, hipGetErrorString(e_));     \
  } while (0)
#define OP_REQUIRE(c, cond, code, msg)              \
  do {                                              \
    if (!(cond)) return ctx_fail((c), (code), msg); \
  } while (0)

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// workgroups of a grid-stride launch: all that are resident at once (8 of 256 threads a CU), no more than there is work for
unsigned stride_grid(long work, int per_cu = 8) { return (unsigned)std::max<long>(1, std::min<long>(work, 256L * per_cu)); }

// ---------------------------------------------------------------------------------------------------- layer norm
template <typename T, int EPT, int LPR, int NCH>
void ln_launch(const LnArgs& a, hipStream_t s) {
  const int rpb = LN_THREADS / LPR;
  hipLaunchKernelGGL((layer_norm_kernel<T, EPT, LPR, NCH>), dim3(stride_grid((a.rows + rpb - 1) / rpb)), dim3(LN_THREADS), 0, s, a);
}

template <typename T, int EPT>
void ln_dispatch(const LnArgs& a, hipStream_t s) {
  const int chunks = (a.C + EPT - 1) / EPT;
  if (chunks <= 8) ln_launch<T, EPT, 8, 1>(a, s);
  else if (chunks <= 16) ln_launch<T, EPT, 16, 1>(a, s);
  else if (chunks <= 32) ln_launch<T, EPT, 32, 1>(a, s);
  else if (chunks <= 64) ln_launch<T, EPT, 64, 1>(a, s);
  else if (chunks <= 128) ln_launch<T, EPT, 64, 2>(a, s);
  else if (chunks <= 256) ln_launch<T, EPT, 64, 4>(a, s);
  else if (EPT == 1 && chunks <= 1024) ln_launch<T, EPT, 64, EPT == 1 ? 16 : 4>(a, s);
  else hipLaunchKernelGGL((layer_norm_long_kernel<T>), dim3(stride_grid(a.rows)), dim3(LN_THREADS), 0, s, a);
}

// rows a backward workgroup covers a step, and the workgroups (= shares of the parameters' gradients) of a launch
int ln_bwd_rows(long chunks) { return chunks <= 8 ? 32 : chunks <= 16 ? 16 : chunks <= 32 ? 8 : 4; }

int ln_ept(int dtype, int C, long ldx, const void* x, long ldy, const void* y, const void* z) {
  const int v = dtype == TAPIR_BF16 ? 8 : 4;
  return C % v == 0 && ldx % v == 0 && ldy % v == 0 && aligned16(x) && aligned16(y) && aligned16(z) ? v : 1;
}

// (C % 8 == 0 says nothing about alignment: the count below holds for both element widths of a launch)
unsigned ln_bwd_grid(long rows, int C, int ept) {
  const long chunks = (C + ept - 1) / ept;
  const bool lng = chunks > (ept == 1 ? 1024 : 256);
  const int rpb = lng ? 1 : ln_bwd_rows(chunks);
  return stride_grid((rows + rpb - 1) / rpb, 2);
}

template <typename T, int EPT, int LPR, int NCH>
void ln_bwd_launch(const LnBwdArgs& a, unsigned grid, hipStream_t s) {
  hipLaunchKernelGGL((layer_norm_bwd_kernel<T, EPT, LPR, NCH>), dim3(grid), dim3(LN_THREADS), 0, s, a);
}

template <typename T, int EPT>
void ln_bwd_dispatch(const LnBwdArgs& a, unsigned grid, hipStream_t s) {
  const int chunks = (a.C + EPT - 1) / EPT;
  if (chunks <= 8) ln_bwd_launch<T, EPT, 8, 1>(a, grid, s);
  else if (chunks <= 16) ln_bwd_launch<T, EPT, 16, 1>(a, grid, s);
  else if (chunks <= 32) ln_bwd_launch<T, EPT, 32, 1>(a, grid, s);
  else if (chunks <= 64) ln_bwd_launch<T, EPT, 64, 1>(a, grid, s);
  else if (chunks <= 128) ln_bwd_launch<T, EPT, 64, 2>(a, grid, s);
  else if (chunks <= 256) ln_bwd_launch<T, EPT, 64, 4>(a, grid, s);
  else if (EPT == 1 && chunks <= 1024) ln_bwd_launch<T, EPT, 64, EPT == 1 ? 16 : 4>(a, grid, s);
  else hipLaunchKernelGGL((layer_norm_bwd_long_kernel<T>), dim3(grid), dim3(LN_THREADS), 0, s, a);
}

// ---------------------------------------------------------------------------------------------------- attention
int attn_pad(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
int attn_part(int dp) { return dp == 96 ? 128 : dp; }   // AtPart
int attn_row_step(int dtype, int dp) { return dtype != TAPIR_BF16 && dp > 32 ? 32 : 64; }   // AtRowTile

struct AttnPlan {
  int dp, row_tiles, splits, tiles_per_split, row_splits, row_steps_per_split;
  size_t part_o, part_ml, delta, part_dq, part_dkv;   // floats
};

size_t round4(size_t n) { return (n + 3) & ~(size_t)3; }   // (shares of a workspace start at multiples of 16 bytes)

// Splits of a long axis: `base` workgroups (or `other`, as likely) of `steps` steps each become base * s of steps / s, joined at `join` us
// a split.  The s of the least estimated time is taken.  Estimate: n workgroups that share a compute unit (of 256) take
// t1 max(1 + (n - 1) / 2, 0.7 n) a step (24576 keys x 64, forward: 1.11, 1.74, 2.49 us for 1 to 3), `occupancy` of them at once, and three
// steps' time to begin.  Measured, 256 x 49152 x 4 x 64, one part of p: forward 699 us unsplit, 34 / 30 / 32 / 34 / 39 us for 256 / 512 /
// 768 / 1024 / 1536 workgroups; keys of the forward pass and of dq, 3 x 1000 x 8200, 4 / 2 heads x 128, half full: training step 428 / 329 /
// 279 / 272 us with the forward pass in 1 / 2 / 4 / 8 splits, 476 / 346 / 282 / 274 with dq in as many (and the rows of dk / dv in two).
struct AttnSplit { long steps, base, other; int occupancy; double t1, join, join_first; };
void attn_split(const AttnSplit& x, int* splits, int* per_split) {
  double best = 0;
  *splits = 0;
  auto shared = [&](long n) { return n == 0 ? 0.0 : x.t1 * std::max(1 + 0.5 * (n - 1), 0.7 * n); };
  for (long s = 1, per = x.steps;; ) {
    const long n = (x.base * s + 255) / 256;
    auto rounds = [&](long n) { return n / x.occupancy * shared(x.occupancy) + shared(n % x.occupancy); };
    const double t = (per + 3) * 0.5 * (rounds(n) + rounds((x.other * s + 255) / 256)) + (s > 1 ? x.join_first + x.join * s : 0);
    if (*splits == 0 || t < best) { best = t; *splits = (int)s; *per_split = (int)per; }
    if (per == 1 || n > 2 * x.occupancy) break;
    --per;                                        // the next number of splits that shortens them
    s = (x.steps + per - 1) / per;
    per = (x.steps + s - 1) / s;
    if (s > 1024) break;
  }
}

AttnPlan attn_plan(const tapir_attn_args* a, int dtype, bool backward) {
  AttnPlan p{};
  const bool bf16 = dtype == TAPIR_BF16;
  p.dp = attn_pad(a->dim);
  const int w = p.dp / 32 - 1;
  const long rows = (long)(a->heads / a->kv_heads) * a->queries, heads = std::max<long>(1, (long)a->batch * a->kv_heads);
  p.row_tiles = (int)((rows + AT_QROWS - 1) / AT_QROWS);
  const int kt = bf16 ? 64 : 32;
  const long tiles = std::max<long>(1, (a->keys + kt - 1) / kt);
  const double us_per_byte = 1 / 9e6;   // partial results, mostly out of the last-level cache
  // us a step of a workgroup that has its compute unit to itself, and workgroups a compute unit holds (AtWaves)
  static const double fwd_us[2][4] = {{1.3, 2.6, 3.8, 5.0}, {0.9, 1.1, 1.7, 1.6}}, dq_us[2][4] = {{1.9, 3.6, 5.3, 7.0}, {0.8, 1.2, 1.8, 2.4}};
  static const double dkv_us[2][4] = {{5.0, 5.0, 7.5, 10.0}, {0.9, 1.4, 1.9, 2.4}};
  static const int fwd_occ[2][4] = {{4, 3, 2, 1}, {4, 3, 2, 2}}, dq_occ[2][4] = {{4, 2, 1, 1}, {4, 3, 2, 2}};
  static const int dkv_occ[2][4] = {{2, 2, 1, 1}, {3, 2, 1, 1}};
  const double row_bytes = 8.0 * heads * rows * p.dp, key_bytes = 16.0 * heads * a->keys * p.dp;   // written and read
  // (a padded batch is taken to hold two thirds of its tokens: the lengths themselves are on the device)
  auto filled = [&](long units) { return std::max<long>(1, a->key_lengths ? units * 2 / 3 : units); };
  const AttnSplit keys{tiles, filled(heads * p.row_tiles), filled(heads * p.row_tiles), backward ? dq_occ[bf16][w] : fwd_occ[bf16][w],
                       backward ? dq_us[bf16][w] : fwd_us[bf16][w], row_bytes * us_per_byte, backward ? 3.0 : 4.0};
  attn_split(keys, &p.splits, &p.tiles_per_split);
  if (!backward) {
    if (p.splits > 1) {
      const size_t r = (size_t)p.splits * a->batch * a->kv_heads * rows;
      p.part_o = r * attn_part(p.dp);
      p.part_ml = round4(r * 2);
    }
    return p;
  }
  const int rt = attn_row_step(dtype, p.dp);
  // Split rows mean f32 shares of dk and dv for every key, which pays only where compute units would be idle: a padded batch is
  // estimated at half and at two thirds of its tokens, so that one guess just past a whole number of rounds does not buy a split.  3 x
  // 1000 x 8200, 4 / 2 heads x 128, half full (195 units; 260 at two thirds): training step 249 us unsplit, 273 / 289 with 2 / 3 splits.  Where
  // units are few, splits stay: 3 x 3000 x 1000 x 2 x 128: 223 / 156 / 121 / 110 / 104 us with 1 / 2 / 4 / 6 / 8; 2 x 700 x 5000 x 2 x 96: 107 / 97 /
  // 108 with 1 / 2 / 3.
  const long key_units = heads * ((a->keys + AT_KEYS - 1) / AT_KEYS);
  const AttnSplit by_row{std::max<long>(1, (rows + rt - 1) / rt), filled(key_units), a->key_lengths ? std::max<long>(1, key_units / 2) : filled(key_units),
                         dkv_occ[bf16][w], dkv_us[bf16][w], key_bytes * us_per_byte, p.splits > 1 ? 1.0 : 3.0};
  attn_split(by_row, &p.row_splits, &p.row_steps_per_split);
  p.delta = round4((size_t)heads * rows);
  if (p.splits > 1 && a->dq) p.part_dq = (size_t)p.splits * a->batch * a->queries * a->heads * a->dim;
  if (p.row_splits > 1 && a->dk) p.part_dkv = (size_t)p.row_splits * a->batch * a->keys * a->kv_heads * a->dim;
  return p;
}

size_t attn_workspace_floats(const AttnPlan& p) { return p.part_o + p.part_ml + p.delta + p.part_dq + 2 * p.part_dkv; }

int attn_check(tapir_ctx* c, const tapir_attn_args* a, bool backward) {
  OP_REQUIRE(c, a != nullptr, TAPIR_ERR_INVALID, "cross_attention: null arguments");
  OP_REQUIRE(c, a->batch >= 0 && a->queries >= 0 && a->keys >= 0 && a->heads >= 1 && a->kv_heads >= 1, TAPIR_ERR_INVALID,
             "cross_attention: negative size or no heads");
  OP_REQUIRE(c, a->heads % a->kv_heads == 0, TAPIR_ERR_INVALID, "cross_attention: heads is not a multiple of kv_heads");
  OP_REQUIRE(c, a->dim >= 8 && a->dim <= 128 && a->dim % 8 == 0, TAPIR_ERR_UNSUPPORTED,
             "cross_attention: head dimension has to be a multiple of 8, at most 128");
  // (dk / dv in bf16 begin their products at numbers of the size of a score over the scale: far from the ends of f32's range)
  OP_REQUIRE(c, a->scale >= 0x1p-60f && a->scale <= 0x1p60f, TAPIR_ERR_INVALID, "cross_attention: scale has to be within 2^-60 .. 2^60");
  const long most = 1L << 30;   // rows, keys, and the workgroups of a launch stay below 2^31
  OP_REQUIRE(c, a->queries <= most && a->keys <= most && (long)a->heads * a->queries <= most && (long)a->batch * a->heads <= (1 << 20),
             TAPIR_ERR_UNSUPPORTED, "cross_attention: too many tokens or heads");
  OP_REQUIRE(c, (long)a->batch * a->kv_heads * (((long)(a->heads / a->kv_heads) * a->queries + AT_QROWS - 1) / AT_QROWS) <= most &&
                    (long)a->batch * a->kv_heads * ((a->keys + AT_KEYS - 1) / AT_KEYS) <= most,
             TAPIR_ERR_UNSUPPORTED, "cross_attention: too many workgroups");
  const int epc = ctx_info(c).dtype == TAPIR_BF16 ? 8 : 4;
  // (an axis of one element has no stride: nothing steps over it)
  auto tensor_ok = [&](const void* p, const int64_t* st, int64_t tokens, int heads) {
    if (a->batch == 0 || tokens == 0) return true;
    return p && aligned16(p) && (a->batch == 1 || st[0] % epc == 0) && (tokens == 1 || st[1] % epc == 0) && (heads == 1 || st[2] % epc == 0);
  };
  auto near = [](const int64_t* st) { return st[1] >= 0 && st[1] < AT_MAX_STRIDE; };
  OP_REQUIRE(c, a->queries <= 1 || (near(a->q_stride) && (!backward || near(a->dout_stride))), TAPIR_ERR_UNSUPPORTED,
             "cross_attention: tokens of q or dout are 2^22 elements apart or more, or in descending order");
  OP_REQUIRE(c, a->keys <= 1 || (near(a->k_stride) && near(a->v_stride)), TAPIR_ERR_UNSUPPORTED,
             "cross_attention: tokens of k or v are 2^22 elements apart or more, or in descending order");
  const bool no_q = a->batch == 0 || a->queries == 0;
  OP_REQUIRE(c, tensor_ok(a->q, a->q_stride, a->queries, a->heads) && tensor_ok(a->k, a->k_stride, a->keys, a->kv_heads) &&
                    tensor_ok(a->v, a->v_stride, a->keys, a->kv_heads) &&
                    (!backward || tensor_ok(a->dout, a->dout_stride, a->queries, a->heads)),
             TAPIR_ERR_INVALID, "cross_attention: null tensor, or one whose rows do not start at multiples of 16 bytes");
  OP_REQUIRE(c, no_q || (a->out && aligned16(a->out)) || backward, TAPIR_ERR_INVALID, "cross_attention: null or misaligned output");
  if (backward) {
    OP_REQUIRE(c, no_q || (a->out_f32 && aligned16(a->out_f32) && a->stats && aligned16(a->stats)), TAPIR_ERR_INVALID,
               "cross_attention: the backward pass needs out_f32 and stats of the forward pass");
    OP_REQUIRE(c, aligned16(a->dq) && aligned16(a->dk) && aligned16(a->dv) && (a->dk == nullptr) == (a->dv == nullptr), TAPIR_ERR_INVALID,
               "cross_attention: misaligned gradients, or one of dk and dv without the other");
  } else {
    OP_REQUIRE(c, (a->out_f32 == nullptr) == (a->stats == nullptr) && aligned16(a->out_f32) && aligned16(a->stats), TAPIR_ERR_INVALID,
               "cross_attention: out_f32 and stats go together");
  }
  return TAPIR_OK;
}

AttnArgs attn_args(const tapir_attn_args* a, const AttnPlan& p) {
  AttnArgs k{};
  k.q = a->q; k.k = a->k; k.v = a->v; k.dout = a->dout;
  for (int i = 0; i < 3; ++i) { k.qs[i] = a->q_stride[i]; k.ks[i] = a->k_stride[i]; k.vs[i] = a->v_stride[i]; k.ds[i] = a->dout_stride[i]; }
  k.key_lengths = a->key_lengths; k.key_mask = a->key_mask;
  k.out = a->out; k.out32 = a->out_f32; k.stats = a->stats; k.dq = a->dq; k.dk = a->dk; k.dv = a->dv;
  k.B = a->batch; k.Hkv = a->kv_heads; k.G = a->heads / a->kv_heads; k.D = a->dim;
  k.Nq = a->queries; k.Nk = a->keys; k.rows = (long)k.G * a->queries;
  k.scale = a->scale; k.scale2 = a->scale * kLog2e;
  k.splits = p.splits; k.tiles_per_split = p.tiles_per_split; k.row_tiles = p.row_tiles;
  k.row_splits = p.row_splits; k.row_steps_per_split = p.row_steps_per_split;
  k.n_dq = (long)a->batch * a->queries * a->heads * a->dim;
  k.n_dkv = (long)a->batch * a->keys * a->kv_heads * a->dim;
  float* w = (float*)a->workspace;
  if (p.part_o) { k.part_o = w; k.part_ml = w + p.part_o; w += p.part_o + p.part_ml; }
  k.delta = w; w += p.delta;
  if (p.part_dq) { k.part_dq = w; w += p.part_dq; }
  if (p.part_dkv) { k.part_dk = w; k.part_dv = w + p.part_dkv; }
  return k;
}

template <typename T, int DP>
void attn_fwd_launch(const AttnArgs& k, hipStream_t s) {
  const unsigned grid = (unsigned)((long)k.B * k.Hkv * k.row_tiles * k.splits);
  hipLaunchKernelGGL((attn_fwd_kernel<T, DP>), dim3(grid), dim3(AT_THREADS), 0, s, k);
  if (k.splits > 1) {
    const long rows = (long)k.B * k.Hkv * k.rows;
    if (k.splits >= 32) hipLaunchKernelGGL((attn_join_kernel<T, AtPart<DP>::V, AT_WAVES>), dim3((unsigned)rows), dim3(AT_THREADS), 0, s, k);
    else hipLaunchKernelGGL((attn_join_kernel<T, AtPart<DP>::V, 1>), dim3((unsigned)((rows + AT_WAVES - 1) / AT_WAVES)), dim3(AT_THREADS), 0, s, k);
  }
}

template <typename T, int DP>
void attn_bwd_launch(const AttnArgs& k, hipStream_t s) {
  if (k.rows > 0 && k.dq) {
    const unsigned grid = (unsigned)((long)k.B * k.Hkv * k.row_tiles * k.splits);
    hipLaunchKernelGGL((attn_dq_kernel<T, DP>), dim3(grid), dim3(AT_THREADS), 0, s, k);
  } else if (k.rows > 0) {
    const long rows = (long)k.B * k.Hkv * k.rows;
    hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((rows + 32 * AT_WAVES - 1) / (32 * AT_WAVES))), dim3(AT_THREADS), 0, s, k);
  }
  if (k.Nk > 0 && k.dk) {
    const unsigned grid = (unsigned)((long)k.B * k.Hkv * ((k.Nk + AT_KEYS - 1) / AT_KEYS) * k.row_splits);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DP>), dim3(grid), dim3(AT_THREADS), 0, s, k);
  }
  const long join = (k.part_dq ? k.n_dq : 0) + (k.part_dk ? 2 * k.n_dkv : 0);
  if (join > 0) hipLaunchKernelGGL((attn_join_grads_kernel<T>), dim3(stride_grid((join / 4 + AT_THREADS - 1) / AT_THREADS)), dim3(AT_THREADS), 0, s, k);
}

#define ATTN_DISPATCH_T(fn, T, dp, ...)           \
  do {                                            \
    if ((dp) == 32) fn<T, 32>(__VA_ARGS__);       \
    else if ((dp) == 64) fn<T, 64>(__VA_ARGS__);  \
    else if ((dp) == 96) fn<T, 96>(__VA_ARGS__);  \
    else fn<T, 128>(__VA_ARGS__);                 \
  } while (0)
#define ATTN_DISPATCH(fn, dtype, dp, ...)                                    \
  do {                                                                       \
    if ((dtype) == TAPIR_BF16) ATTN_DISPATCH_T(fn, bf16_t, dp, __VA_ARGS__); \
    else ATTN_DISPATCH_T(fn, float, dp, __VA_ARGS__);                        \
  } while (0)

}  // namespace

extern "C" {

int tapir_layer_norm(tapir_ctx* c, const void* x, int64_t x_stride, const float* gamma, const float* beta, void* y,
                     float* mean, float* rstd, int64_t rows, int channels, float eps, void* stream) {
  if (!c) return TAPIR_ERR_INVALID;
  const CtxInfo ci = ctx_info(c);
  OP_REQUIRE(c, rows >= 0 && channels >= 1 && eps >= 0.f && isfinite(eps), TAPIR_ERR_INVALID, "layer_norm: bad size or eps");
  OP_REQUIRE(c, channels <= LN_MAX_CHANNELS, TAPIR_ERR_UNSUPPORTED, "layer_norm: more than 2^30 channels");
  OP_REQUIRE(c, (mean == nullptr) == (rstd == nullptr), TAPIR_ERR_INVALID, "layer_norm: mean and rstd go together");
  if (rows == 0) return TAPIR_OK;
  OP_REQUIRE(c, x && y, TAPIR_ERR_INVALID, "layer_norm: null tensor");
  OP_TRY(c, hipSetDevice(ci.device));
  const LnArgs a{x, (long)x_stride, gamma, beta, y, mean, rstd, (long)rows, channels, eps};
  const int ept = ln_ept(ci.dtype, channels, x_stride, x, channels, y, y);
  hipStream_t s = (hipStream_t)stream;
  if (ci.dtype == TAPIR_BF16) { if (ept == 8) ln_dispatch<bf16_t, 8>(a, s); else ln_dispatch<bf16_t, 1>(a, s); }
  else { if (ept == 4) ln_dispatch<float, 4>(a, s); else ln_dispatch<float, 1>(a, s); }
  OP_TRY(c, hipGetLastError());
  return TAPIR_OK;
}

int tapir_layer_norm_workspace(tapir_ctx* c, int64_t rows, int channels, uint64_t* bytes) {
  if (!c) return TAPIR_ERR_INVALID;
  OP_REQUIRE(c, bytes && rows >= 0 && channels >= 1, TAPIR_ERR_INVALID, "layer_norm: bad size");
  OP_REQUIRE(c, channels <= LN_MAX_CHANNELS, TAPIR_ERR_UNSUPPORTED, "layer_norm: more than 2^30 channels");
  const int v = ctx_info(c).dtype == TAPIR_BF16 ? 8 : 4;
  const unsigned shares = std::max(ln_bwd_grid(rows, channels, 1), ln_bwd_grid(rows, channels, v));
  *bytes = (uint64_t)shares * 2 * ln_part_stride(channels) * sizeof(float);
  return TAPIR_OK;
}

int tapir_layer_norm_backward(tapir_ctx* c, const void* x, int64_t x_stride, const void* dy, int64_t dy_stride,
                              const float* gamma, const float* mean, const float* rstd, void* dx, float* dgamma, float* dbeta,
                              int64_t rows, int channels, void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!c) return TAPIR_ERR_INVALID;
  const CtxInfo ci = ctx_info(c);
  OP_REQUIRE(c, rows >= 0 && channels >= 1, TAPIR_ERR_INVALID, "layer_norm: bad size");
  OP_REQUIRE(c, channels <= LN_MAX_CHANNELS, TAPIR_ERR_UNSUPPORTED, "layer_norm: more than 2^30 channels");
  OP_REQUIRE(c, rows == 0 || (x && dy && mean && rstd), TAPIR_ERR_INVALID, "layer_norm: null tensor");
  const int ept = ln_ept(ci.dtype, channels, x_stride, x, dy_stride, dy, dx);
  const unsigned grid = ln_bwd_grid(rows, channels, ept);
  const bool params = dgamma || dbeta;
  OP_REQUIRE(c, !params || (workspace && aligned16(workspace) && workspace_bytes >= (uint64_t)grid * 2 * ln_part_stride(channels) * sizeof(float)),
             TAPIR_ERR_INVALID, "layer_norm: workspace missing or too small (tapir_layer_norm_workspace)");
  OP_TRY(c, hipSetDevice(ci.device));
  const LnBwdArgs a{x, (long)x_stride, dy, (long)dy_stride, gamma, mean, rstd, dx, params ? (float*)workspace : nullptr, (long)rows, channels};
  hipStream_t s = (hipStream_t)stream;
  if (rows > 0) {
    if (ci.dtype == TAPIR_BF16) { if (ept == 8) ln_bwd_dispatch<bf16_t, 8>(a, grid, s); else ln_bwd_dispatch<bf16_t, 1>(a, grid, s); }
    else { if (ept == 4) ln_bwd_dispatch<float, 4>(a, grid, s); else ln_bwd_dispatch<float, 1>(a, grid, s); }
    OP_TRY(c, hipGetLastError());
  }
  if (params) {
    hipLaunchKernelGGL(layer_norm_reduce_kernel, dim3((unsigned)((channels + LN_REDUCE_COLS - 1) / LN_REDUCE_COLS), 2), dim3(LN_THREADS), 0,
                       s, (const float*)workspace, rows > 0 ? (int)grid : 0, channels, dgamma, dbeta);
    OP_TRY(c, hipGetLastError());
  }
  return TAPIR_OK;
}

int tapir_rotary_positions(tapir_ctx* c, const tapir_rotary_args* r, void* stream) {
  if (!c) return TAPIR_ERR_INVALID;
  const CtxInfo ci = ctx_info(c);
  OP_REQUIRE(c, r != nullptr, TAPIR_ERR_INVALID, "rotary_positions: null arguments");
  OP_REQUIRE(c, r->batch >= 0 && r->tokens >= 0 && r->heads >= 1 && r->dim >= 1, TAPIR_ERR_INVALID, "rotary_positions: bad size");
  OP_REQUIRE(c, r->dim <= 2 * ROT_MAX_PAIRS, TAPIR_ERR_UNSUPPORTED, "rotary_positions: head dimension over 256");
  OP_REQUIRE(c, r->axes >= 1 && r->axes <= ROT_MAX_AXES, TAPIR_ERR_INVALID, "rotary_positions: 1 to 4 axes");
  const long most = 1L << 40;
  OP_REQUIRE(c, r->batch <= most && r->tokens <= most && (double)r->batch * r->tokens * r->heads * r->dim < 9e15, TAPIR_ERR_UNSUPPORTED,
             "rotary_positions: too many tokens");
  RotaryArgs a{};
  int at = 0, pairs = 0;
  for (int x = 0; x < r->axes; ++x) {
    const int w = r->section[x];
    OP_REQUIRE(c, w >= 0 && w % 2 == 0 && at + w <= r->dim, TAPIR_ERR_INVALID,
               "rotary_positions: sections have to be even and fit the head dimension");
    OP_REQUIRE(c, r->base[x] > 0.0 && isfinite(r->base[x]), TAPIR_ERR_INVALID, "rotary_positions: base has to be positive and finite");
    for (int i = 0; i < w / 2; ++i, ++pairs) {
      a.turns[pairs] = pow(r->base[x], -2.0 * i / w) / 6.283185307179586476925286766559;
      a.axis[pairs] = (unsigned char)x;
      a.lo[pairs] = (unsigned char)(r->interleaved ? at + 2 * i : at + i);
      a.hi[pairs] = (unsigned char)(r->interleaved ? at + 2 * i + 1 : at + i + w / 2);
    }
    at += w;
  }
  if (r->batch == 0 || r->tokens == 0) return TAPIR_OK;
  OP_REQUIRE(c, r->x && r->y && r->positions, TAPIR_ERR_INVALID, "rotary_positions: null tensor");
  OP_TRY(c, hipSetDevice(ci.device));
  const int epc = ci.dtype == TAPIR_BF16 ? 8 : 4;
  const bool bf16 = ci.dtype == TAPIR_BF16;
  if (r->dim % epc == 0 && r->x_stride[0] % epc == 0 && r->x_stride[1] % epc == 0 && r->x_stride[2] % epc == 0 && aligned16(r->x) &&
      aligned16(r->y)) {
    RotaryRowArgs v{};
    v.x = r->x; v.sb = r->x_stride[0]; v.sn = r->x_stride[1]; v.sh = r->x_stride[2];
    v.pos = r->positions; v.pb = r->positions_stride; v.y = r->y;
    v.B = r->batch; v.N = r->tokens; v.H = r->heads; v.D = r->dim; v.axes = r->axes;
    v.sign = r->inverse ? -1.f : 1.f;
    for (int i = 0; i < r->dim; ++i) v.other[i] = (unsigned char)i;
    for (int i = 0; i < pairs; ++i) {
      v.turns[a.lo[i]] = v.turns[a.hi[i]] = a.turns[i];
      v.axis[a.lo[i]] = v.axis[a.hi[i]] = a.axis[i];
      v.other[a.lo[i]] = a.hi[i];
      v.other[a.hi[i]] = a.lo[i];
    }
    const long rpb = (long)(ROT_THREADS / 64) * (64 / (r->dim / epc));   // tokens of a workgroup and step
    const long base = (r->batch * r->tokens + rpb - 1) / rpb;
    // few tokens: the heads go to workgroups of their own, ROT_HEADS at most in each, rather than one after the other
    const int cuts = (int)std::min<long>((r->heads + ROT_HEADS - 1) / ROT_HEADS, std::max<long>(1, 1024 / base));
    v.heads = (r->heads + cuts - 1) / cuts;
    const dim3 grid(stride_grid(base), (unsigned)((r->heads + v.heads - 1) / v.heads)), block(ROT_THREADS);
    if (bf16) hipLaunchKernelGGL((rotary_rows_kernel<bf16_t>), grid, block, 0, (hipStream_t)stream, v);
    else hipLaunchKernelGGL((rotary_rows_kernel<float>), grid, block, 0, (hipStream_t)stream, v);
    OP_TRY(c, hipGetLastError());
    return TAPIR_OK;
  }
  a.x = r->x; a.sb = r->x_stride[0]; a.sn = r->x_stride[1]; a.sh = r->x_stride[2];
  a.pos = r->positions; a.pb = r->positions_stride; a.y = r->y;
  a.B = r->batch; a.N = r->tokens; a.H = r->heads; a.D = r->dim; a.axes = r->axes; a.pairs = pairs;
  a.sign = r->inverse ? -1.f : 1.f;
  const long work = (a.B * a.N * (a.D - a.pairs) + ROT_THREADS - 1) / ROT_THREADS;
  const dim3 grid(stride_grid(work)), block(ROT_THREADS);
  if (bf16) hipLaunchKernelGGL((rotary_kernel<bf16_t>), grid, block, 0, (hipStream_t)stream, a);
  else hipLaunchKernelGGL((rotary_kernel<float>), grid, block, 0, (hipStream_t)stream, a);
  OP_TRY(c, hipGetLastError());
  return TAPIR_OK;
}

int tapir_cross_attention_workspace(tapir_ctx* c, const tapir_attn_args* a, int backward, uint64_t* bytes) {
  if (!c) return TAPIR_ERR_INVALID;
  OP_REQUIRE(c, a && bytes && a->batch >= 0 && a->queries >= 0 && a->keys >= 0 && a->kv_heads >= 1 && a->heads >= 1 &&
                    a->heads % a->kv_heads == 0, TAPIR_ERR_INVALID, "cross_attention: bad size");
  *bytes = sizeof(float) * attn_workspace_floats(attn_plan(a, ctx_info(c).dtype, backward != 0));
  return TAPIR_OK;
}

int tapir_cross_attention(tapir_ctx* c, const tapir_attn_args* a, void* stream) {
  if (!c) return TAPIR_ERR_INVALID;
  const CtxInfo ci = ctx_info(c);
  const int rc = attn_check(c, a, false);
  if (rc != TAPIR_OK) return rc;
  if (a->batch == 0 || a->queries == 0) return TAPIR_OK;
  const AttnPlan p = attn_plan(a, ci.dtype, false);
  const size_t floats = attn_workspace_floats(p);
  OP_REQUIRE(c, floats == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= sizeof(float) * floats),
             TAPIR_ERR_INVALID, "cross_attention: workspace missing or too small (tapir_cross_attention_workspace)");
  OP_TRY(c, hipSetDevice(ci.device));
  const AttnArgs k = attn_args(a, p);
  ATTN_DISPATCH(attn_fwd_launch, ci.dtype, p.dp, k, (hipStream_t)stream);
  OP_TRY(c, hipGetLastError());
  return TAPIR_OK;
}

int tapir_cross_attention_backward(tapir_ctx* c, const tapir_attn_args* a, void* stream) {
  if (!c) return TAPIR_ERR_INVALID;
  const CtxInfo ci = ctx_info(c);
  const int rc = attn_check(c, a, true);
  if (rc != TAPIR_OK) return rc;
  if (a->batch == 0) return TAPIR_OK;
  const AttnPlan p = attn_plan(a, ci.dtype, true);
  const size_t floats = attn_workspace_floats(p);
  OP_REQUIRE(c, floats == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= sizeof(float) * floats),
             TAPIR_ERR_INVALID, "cross_attention: workspace missing or too small (tapir_cross_attention_workspace)");
  OP_TRY(c, hipSetDevice(ci.device));
  const AttnArgs k = attn_args(a, p);
  ATTN_DISPATCH(attn_bwd_launch, ci.dtype, p.dp, k, (hipStream_t)stream);
  OP_TRY(c, hipGetLastError());
  return TAPIR_OK;
}

}  // extern "C"
