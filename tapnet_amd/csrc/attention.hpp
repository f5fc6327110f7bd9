// Cross attention of query rows to an encoder's tokens, forward and backward, one pass over the keys.
//
//   s_rk = scale q_r . k_k,  p_rk = exp(s_rk - m_r) / l_r,  l_r = sum_k exp(s_rk - m_r),  o_r = sum_k p_rk v_k
//   D_r = do_r . o_r,  dp_rk = do_r . v_k,  ds_rk = p_rk (dp_rk - D_r) scale
//   dq_r = sum_k ds_rk k_k,   dk_k = sum_r ds_rk q_r,   dv_k = sum_r p_rk do_r
//
// Rows: the G query heads that share a key head are flattened with the queries into one row axis (row = g * queries + query),
// so that a tile of rows reads every key once for all heads of the group, and the sums dk / dv of a shared head need no
// reduction of their own.  Masked keys (behind the clip's length, or cleared in the key mask) are never loaded: their rows of
// the tile are zeros and their scores -inf, so whatever the padding holds (NaN, infinities) cannot reach a result.  A row
// without any key gives zeros and passes zero gradients.
//
// Matrix products: v_mfma_f32_32x32x16_bf16 / v_mfma_f32_32x32x2_f32.  The forward pass and dq work on TRANSPOSED scores
// (rows of the product = keys, columns = query rows): a lane then holds 16 keys of ONE query row, the softmax statistics are
// per-lane scalars (one exchange with lane ^ 32), and the 8 probabilities a lane holds in consecutive registers ARE its operand
// of the next product (the order of the summed keys is free as long as both operands agree): nothing is moved between the
// products.  dk / dv use the untransposed scores for the same reason (a lane holds 16 query rows of one key).  The other
// operand of these second products is a transposed tile: ds_read_b64_tr_b16 (bf16), plain 4-byte reads (f32).
#pragma once
#include "common.hpp"

namespace tapir {

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

constexpr int AT_WAVES = 4;
constexpr int AT_THREADS = 64 * AT_WAVES;
constexpr int AT_QROWS = 32 * AT_WAVES;      // query rows of a forward / dq workgroup
constexpr int AT_KEYS = 32 * AT_WAVES;       // keys of a dk / dv workgroup
constexpr float kLog2e = 1.4426950408889634f;
constexpr float AT_SLACK = 8.f;
constexpr float AT_FAR = 0x1p24f, AT_NEAR = 0x1p10f;   // sizes of a base of the exponentials: at_exponent, attn_dkv_kernel
constexpr long AT_MAX_STRIDE = 1L << 22;   // elements from token to token: offsets within a tile of 64 tokens stay below 2^30 bytes

struct AttnArgs {
  const void *q, *k, *v, *dout;
  long qs[3], ks[3], vs[3], ds[3];     // strides in elements: clip, token, head (channels dense)
  const int* key_lengths;              // [B] or null
  const unsigned char* key_mask;       // [B, Nk] or null: nonzero = may be attended to
  void* out;                           // [B, Nq, H, D] dense
  float *out32;                        // the same unrounded (training), or null
  float *stats;                        // [B, Hkv, rows, 2]: m_r log2(e) and 1 / l_r (0, 0 for a row without keys), or null
  float *delta;                        // [B, Hkv, rows]: D_r
  void *dq, *dk, *dv;                  // dense
  float *part_o, *part_ml;             // split keys, forward: [splits, B * Hkv, rows, DP] and [B * Hkv, rows, splits, 2]
  float *part_dq, *part_dk, *part_dv;  // backward: [splits] copies of dq (keys split) and of dk, dv (rows split) in f32
  long n_dq, n_dkv;                    // elements of dq and of dk
  long Nq, Nk, rows;                   // rows = G * Nq
  int B, Hkv, G, D;
  int splits, tiles_per_split;         // key tiles of a split (forward, dq)
  int row_splits, row_steps_per_split; // row steps of a split (dk / dv)
  int row_tiles;
  float scale, scale2;                 // scale, scale * log2(e)
};

// physical 16-byte chunk of logical chunk c in row r of a tile with CH chunks a row: rows that are read together have their chunks in
// different places of a bank line.  Measured conflict cycles, of the cycles in which LDS works: a third at 32 and 64 channels (dq 0.40, dk / dv
// 0.24), 0.44 to 0.49 at 128; f32 0.18 to 0.29.  LDS works in 2 to 31 % of a compute unit's busy cycles and bounds none of these kernels.
template <int CH> __device__ __forceinline__ int at_swizzle(int r, int c) {
  if (CH >= 8) return c ^ (((r & 3) << 1) | ((r >> 2) & 1));
  return c ^ ((r & 2) | ((r >> 2) & 1));        // 64-byte rows: the row's parity picks the half of a bank line already
}

template <typename T> struct AtFrag;            // 16 bytes of a row: the operand of one k-step
template <> struct AtFrag<bf16_t> { static constexpr int EPC = 8; };
template <> struct AtFrag<float> { static constexpr int EPC = 4; };
// chunks from row to row of a tile of DP channels: the swizzle stays within a power of two or a multiple of eight
template <typename T, int DP> struct AtPitch { static constexpr int CH = DP / AtFrag<T>::EPC, V = CH % 8 == 0 || CH == 4 ? CH : 16; };
// channels from row to row of the forward pass' partial results
template <int DP> struct AtPart { static constexpr int V = DP == 96 ? 128 : DP; };

// c += a b over the elements of one 16-byte chunk per lane (lanes l and l ^ 32 hold neighbouring chunks)
__device__ __forceinline__ f32x16 at_mma(const uint4& a, const uint4& b, f32x16 c, bf16_t) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 at_mma(const uint4& a, const uint4& b, f32x16 c, float) {
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
}

// ds_read_b64_tr_b16: the 16 lanes of a group name 16 x 8 bytes (lane i: row i / 4, columns 4 (i % 4) .. +3 of a 4 x 16 block);
// lane i receives column i of the block, rows 0 .. 3.
__device__ __forceinline__ uint2 at_read_tr(const bf16_t* p) {
#ifdef TAPIR_HIPEMU
  const unsigned l = threadIdx.x & 63, i = l & 15;
  const uint64_t a = (uint64_t)(uintptr_t)p;
  uint16_t r[4];
  for (int j = 0; j < 4; ++j) {
    const int src = (int)((l & 48) + 4 * j + (i >> 2));
    const uint64_t hi = (uint32_t)__shfl((int)(a >> 32), src), lo = (uint32_t)__shfl((int)a, src);
    r[j] = ((const uint16_t*)(uintptr_t)((hi << 32) | lo))[i & 3];
  }
  return make_uint2((unsigned)r[0] | ((unsigned)r[1] << 16), (unsigned)r[2] | ((unsigned)r[3] << 16));
#else
  typedef __attribute__((ext_vector_type(4))) short s16x4;
  typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
  const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
  return __builtin_bit_cast(uint2, r);
#endif
}

// c[32 channels from d0][32 columns] += X[32 summed rows from r0][channels]^T * w, w = 16 values a lane in the layout of a
// 32 x 32 product (register i of lane half h: summed row 8 (i / 4) + 4 h + i % 4).  X: a tile of CH-chunk rows in LDS.
struct AtTr { uint2 t[4]; };     // a lane's share of X's 32 rows from r0, 32 channels from d0
template <int CH> __device__ __forceinline__ AtTr at_tr(const bf16_t* X, int r0, int d0) {
  const int l = threadIdx.x & 63, h = l >> 5, i = l & 15;
  AtTr x;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = r0 + 8 * u + 4 * h + (i >> 2), col = d0 + (l & 16) + 4 * (i & 3);
    x.t[u] = at_read_tr(X + ((long)r * CH + at_swizzle<CH>(r, col >> 3)) * 8 + (col & 7));
  }
  return x;
}
__device__ __forceinline__ void at_mma_tr(f32x16& c, const AtTr& x, const unsigned (&w)[8]) {
#pragma unroll
  for (int s = 0; s < 2; ++s)
    c = at_mma(make_uint4(x.t[2 * s].x, x.t[2 * s].y, x.t[2 * s + 1].x, x.t[2 * s + 1].y),
               make_uint4(w[4 * s], w[4 * s + 1], w[4 * s + 2], w[4 * s + 3]), c, bf16_t{});
}
template <int CH>
__device__ __forceinline__ void at_mma_tr(f32x16& c, const bf16_t* X, int r0, int d0, const unsigned (&w)[8]) {
  at_mma_tr(c, at_tr<CH>(X, r0, d0), w);
}
template <int CH>
__device__ __forceinline__ void at_mma_tr(f32x16& c, const float* X, int r0, int d0, const float (&w)[16]) {
  const int l = threadIdx.x & 63, h = l >> 5, col = d0 + (l & 31);
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + 8 * (i >> 2) + 4 * h + (i & 3);
    x[i] = X[((long)r * CH + at_swizzle<CH>(r, col >> 2)) * 4 + (col & 3)];
  }
  sched_fence();
#pragma unroll
  for (int i = 0; i < 16; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], w[i], c, 0, 0, 0);
}

// the 16 values of a lane as the operand of at_mma_tr, f32: as they are
__device__ __forceinline__ void at_operand(const f32x16& p, float (&w)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = p[i];
}
// bf16: in two parts, w + v: the 16 most significant bits and the bf16 of what is left (2^-15 together).  One rounding of p and ds
// would show: where a row attends to many tokens alike its result is a small sum of many terms, and the error of p stands beside the
// result's own rounding (1.4 to 1.5 times as far from the exact result in all; 1 query x 49152 keys); the gradients' terms cancel as well
// (1.45 to 1.7 times).  What the second part costs, forward: 1 query x 49152 keys, 8 / 2 heads x 64: 14.7 -> 15.3 us; 256 x 49152 x 4 x 64:
// 30.6 -> 34.5; 4096 x 49152 x 4 x 64: 260 -> 337 (the vector unit splits every p); gradients, 256 x 49152: 6 us of 95 for p, 10 for ds.
__device__ __forceinline__ void at_operand2(const f32x16& p, unsigned (&w)[8], unsigned (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned a = __float_as_uint(p[2 * i]) & 0xffff0000u, b = __float_as_uint(p[2 * i + 1]) & 0xffff0000u;
#ifdef TAPIR_HIPEMU
    w[i] = (a >> 16) | b;
#else
    w[i] = __builtin_amdgcn_perm(__float_as_uint(p[2 * i + 1]), __float_as_uint(p[2 * i]), 0x07060302u);   // both upper halves
#endif
    v[i] = pack_bf16x2(p[2 * i] - __uint_as_float(a), p[2 * i + 1] - __uint_as_float(b));
  }
}

// c plus the 16 values, unrounded: a sum of the rounded ones would make 1 / l_r, and with it every gradient of the row, off by up
// to a bf16 rounding where one key dominates (two chains: an addition's latency is longer than its issue)
__device__ __forceinline__ float at_sum(const f32x16& p, float c) {
  float d = p[0];
#pragma unroll
  for (int i = 1; i < 15; i += 2) { c += p[i]; d += p[i + 1]; }
  return (c + p[15]) + d;
}
template <typename T> struct AtOperand;
template <> struct AtOperand<bf16_t> { unsigned w[8]; };
template <> struct AtOperand<float> { float w[16]; };

// maximum / sum of the two values that lanes l and l ^ 32 hold
__device__ __forceinline__ void at_halves(float v, float* a, float* b) {
#ifdef TAPIR_HIPEMU
  *a = v;
  *b = __shfl_xor(v, 32);
#else
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  *a = __uint_as_float(r[0]);
  *b = __uint_as_float(r[1]);
#endif
}
__device__ __forceinline__ float at_max_halves(float v) { float a, b; at_halves(v, &a, &b); return fmaxf(a, b); }
__device__ __forceinline__ float at_sum_halves(float v) { float a, b; at_halves(v, &a, &b); return a + b; }

__device__ __forceinline__ f32x16 at_zero() {
  f32x16 z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

// 16 bytes a lane from base + off (base uniform) to LDS, lane i of the wave to `lds` + 16 i; asynchronous: dma_wait().  Written out
// because the compiler waits for all outstanding copies before every ds_read_b64_tr_b16, whose address it does not analyse: the
// next tile's copies would then not run under this tile's products.  No register is written, only LDS (M0, the copies' LDS address,
// serves nothing else in these kernels).  The wait covers M0 and a base that a vector instruction wrote into scalar registers just before.
__device__ __forceinline__ void at_copy16(const void* base, unsigned off, void* lds) {
#ifdef TAPIR_HIPEMU
  *((uint4*)lds + (threadIdx.x & 63)) = *(const uint4*)((const char*)base + off);   // (only the lanes that take part)
#else
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
               :: "s"(__builtin_amdgcn_readfirstlane((int)(uintptr_t)lds)), "v"(off), "s"(base) : "memory");
#endif
}

// ROWS x DP tile of a [token][channel] tensor -> LDS, 16-byte chunks, by the whole workgroup: thread i copies slots i, i + 256,
// ... of the tile.  The offsets of a thread's chunks from the tile's first row stay the same for all tiles of a tensor.
template <typename T, int ROWS, int DP> struct AtStage {
  static constexpr int EPC = AtFrag<T>::EPC, CH = AtPitch<T, DP>::V, N = ROWS * CH / AT_THREADS;
  static_assert(ROWS * CH % AT_THREADS == 0, "tile");
  unsigned off[N];     // bytes (token strides are below AT_MAX_STRIDE elements)

  static __device__ __forceinline__ int row(int n) { return (n * AT_THREADS + (int)threadIdx.x) / CH; }
  static __device__ __forceinline__ int chunk(int n) { const int s = n * AT_THREADS + (int)threadIdx.x; return at_swizzle<CH>(s / CH, s % CH); }
  __device__ __forceinline__ void init(long stride) {
#pragma unroll
    for (int n = 0; n < N; ++n) off[n] = (unsigned)((row(n) * stride + chunk(n) * EPC) * (long)sizeof(T));
  }
  // the thread's n-th chunk from `first` (uniform) + off, or zeros
  static __device__ __forceinline__ void put(T* lds, int n, const T* first, unsigned off, bool ok) {
    T* const to = lds + (n * AT_THREADS + (threadIdx.x >> 6) * 64) * EPC;
    if (ok) at_copy16(first, off, to);
    else *reinterpret_cast<uint4*>(to + (threadIdx.x & 63) * EPC) = make_uint4(0u, 0u, 0u, 0u);
  }
  // rows from `first` on; row r is zeros where bit r of `bits` is not set, channels from D on are zeros too
  __device__ __forceinline__ void rows(T* lds, const T* first, uint64_t bits, int D) const {
    constexpr uint64_t all = ROWS == 64 ? ~0ull : (1ull << (ROWS & 63)) - 1;
    if ((bits & all) == all && D == CH * EPC) {   // (no chunk of the pitch lies behind the channels)
#pragma unroll
      for (int n = 0; n < N; ++n) at_copy16(first, off[n], lds + (n * AT_THREADS + (threadIdx.x >> 6) * 64) * EPC);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) put(lds, n, first, off[n], ((bits >> row(n)) & 1) && chunk(n) * EPC < D);
    }
  }
};

template <typename T, int CH> __device__ __forceinline__ uint4 at_chunk(const T* X, int r, int c) {
  return *reinterpret_cast<const uint4*>(X + ((long)r * CH + at_swizzle<CH>(r, c)) * AtFrag<T>::EPC);
}

// s += (rows r + lane of the tile X) . (the lane's operand chunks b), f32: the next chunk is read before the products with this one
// are issued, and a fence keeps it so (the compiler would read each right before its products and wait; 739 x 1161 x 32 x 72,
// backward: 527 -> 453 us.  bf16, whose products take an eighth of the time, gains nothing by one chunk and spills with more)
template <typename T, int PC, int NS>
__device__ __forceinline__ void at_dot(f32x16& s, const T* X, int r, const uint4 (&b)[NS]) {
  const int l = threadIdx.x & 63, h = l >> 5;
  uint4 a[2];
  a[0] = at_chunk<T, PC>(X, r + (l & 31), h);
#pragma unroll
  for (int x = 0; x < NS; ++x) {
    if (x + 1 < NS) a[(x + 1) & 1] = at_chunk<T, PC>(X, r + (l & 31), 2 * x + 2 + h);
    sched_fence();
    s = at_mma(a[x & 1], b[x], s, T{});
  }
}

// Key validity of a tile's keys as a wave-uniform mask (bit j: key k0 + j takes part).  The mask's bytes are read one tile ahead:
// a load that is waited for here would wait for the copies in flight, too.
struct AtKeyBits {
  const unsigned char* mask;     // of the clip, or null
  long len;
  unsigned next;                 // the lane's byte of the tile that is staged next

  __device__ __forceinline__ void fetch(long k0) {
    const long key = k0 + (threadIdx.x & 63);
    next = mask != nullptr && key < len ? mask[key] : 1;
  }
  __device__ __forceinline__ uint64_t bits(long k0) const { return __ballot(k0 + (threadIdx.x & 63) < len && next != 0); }
};

__device__ __forceinline__ long at_key_len(const AttnArgs& a, int b) {
  if (a.key_lengths == nullptr) return a.Nk;
  const long n = a.key_lengths[b];
  return n < 0 ? 0 : (n > a.Nk ? a.Nk : n);
}

// 4 consecutive channels of a result row
template <typename T> __device__ __forceinline__ void at_store4(T* p, float x, float y, float z, float w);
template <> __device__ __forceinline__ void at_store4<float>(float* p, float x, float y, float z, float w) {
  *reinterpret_cast<float4*>(p) = make_float4(x, y, z, w);
}
template <> __device__ __forceinline__ void at_store4<bf16_t>(bf16_t* p, float x, float y, float z, float w) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(x, y), pack_bf16x2(z, w));
}

// keys a forward / dq step stages: 64 (bf16) or 32 (f32)
template <typename T> struct AtTile { static constexpr int KT = sizeof(T) == 2 ? 64 : 32; };
// query rows a dk / dv step stages: 64, so that the next step's copies have two blocks of products to arrive under (bf16, 64
// channels: 256 x 49152 x 4 x 64: 60 -> 51 us); f32, whose products take eight times as long: 32 where that is a copy per thread
template <typename T, int DP> struct AtRowTile { static constexpr int RT = sizeof(T) == 4 && DP > 32 ? 32 : 64; };

// ------------------------------------------------------------------------------------------------------- work distribution
// splits of a clip's keys that hold any (at least one: it writes the zeros of a clip without tokens); its key tiles that do
template <typename T> __device__ __forceinline__ unsigned at_clip_splits(const AttnArgs& a, int b) {
  if (a.key_lengths == nullptr) return a.splits;
  const unsigned tiles = (unsigned)((at_key_len(a, b) + AtTile<T>::KT - 1) / AtTile<T>::KT), per = a.tiles_per_split;
  return tiles <= per ? 1 : (tiles + per - 1) / per;
}
__device__ __forceinline__ unsigned at_clip_key_tiles(const AttnArgs& a, int b) { return (unsigned)((at_key_len(a, b) + AT_KEYS - 1) / AT_KEYS); }

// Workgroups are dealt to the 8 dies in turn; each die takes one run of consecutive units of work, so that its own L2 serves the
// keys (rows) that neighbouring units share.  Only units that hold work are counted (`active` of them): clips of different lengths
// would otherwise leave whole dies idle (3 clips of 8200, 4100 and 0 tokens: 489 -> 291 us a training step).  Returns the unit, or
// -1 - i for the i-th workgroup that is left over.
__device__ __forceinline__ int at_unit(unsigned active) {
  const unsigned n = gridDim.x, i = blockIdx.x, x = i % 8, j = i / 8;
  const unsigned q = active / 8, r = active % 8, mine = q + (x < r);
  if (j < mine) return (int)(x * q + (x < r ? x : r) + j);
  const unsigned nq = n / 8, nr = n % 8;
  return -1 - (int)(x * (nq - q) + (x < nr ? x : nr) - (x < r ? x : r) + j - mine);
}

struct AtUnit { int b, hk, split, tile; };

__device__ __forceinline__ unsigned at_uniform(unsigned v) { return (unsigned)__builtin_amdgcn_readfirstlane((int)v); }

// Units of all clips, count(clip) each: 64 clips at a time, a lane each
template <class F> __device__ __forceinline__ unsigned at_units(int B, const F& count) {
  unsigned total = 0;
  for (int c = 0; c < B; c += 64) {
    const int clip = c + (int)(threadIdx.x & 63);
    unsigned v = clip < B ? count(clip) : 0;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += (unsigned)__shfl_xor((int)v, m);
    total += at_uniform(v);
  }
  return total;
}
// the clip that unit w of them falls to; w becomes its index within the clip, n the clip's count
template <class F> __device__ __forceinline__ int at_find_clip(int B, const F& count, unsigned* w, unsigned* n) {
  const int l = threadIdx.x & 63;
  for (int c = 0; c < B; c += 64) {
    const unsigned v = c + l < B ? count(c + l) : 0;
    unsigned upto = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const unsigned before = (unsigned)__shfl((int)upto, (l - m) & 63);
      if (l >= m) upto += before;
    }
    const uint64_t behind = __ballot(upto > *w);
    if (behind != 0) {
      const int lane = (int)at_uniform((unsigned)__builtin_ctzll(behind));
      *n = at_uniform((unsigned)__shfl((int)v, lane));
      *w -= at_uniform((unsigned)__shfl((int)upto, lane)) - *n;
      return c + lane;
    }
    *w -= at_uniform((unsigned)__shfl((int)upto, 63));
  }
  return 0;   // (not reached: w is below the sum)
}

// (units fit 31 bits: 64-bit divisions of them took a third of a short workgroup's prologue)
__device__ __forceinline__ AtUnit at_decode(int b, unsigned w, unsigned tiles, unsigned splits) {
  const unsigned rest = w / tiles, hk = rest / splits;
  return AtUnit{b, (int)hk, (int)(rest - hk * splits), (int)(w - rest * tiles)};
}

// forward / dq: units ordered by clip, key head, split of the keys, row tile
template <typename T> __device__ __forceinline__ bool at_row_unit(const AttnArgs& a, AtUnit* u) {
  const unsigned per = (unsigned)(a.Hkv * a.row_tiles);
  unsigned w, splits = a.splits;
  int b;
  if (a.key_lengths == nullptr) {
    w = at_unit(gridDim.x);
    b = (int)(w / (per * splits));
    w -= b * per * splits;
  } else {
    auto count = [&](int clip) { return per * at_clip_splits<T>(a, clip); };
    const int i = at_unit(at_units(a.B, count));
    if (i < 0) return false;
    w = i;
    b = at_find_clip(a.B, count, &w, &splits);
    splits /= per;
  }
  *u = at_decode(b, w, a.row_tiles, splits);
  return true;
}

// dk / dv: units ordered by clip, key head, split of the rows, key tile.  Tiles behind a clip's length come back from the workgroups
// that are left over, as `zero`: there is nothing to sum, but dk and dv are to be written.
__device__ __forceinline__ bool at_key_unit(const AttnArgs& a, AtUnit* u, bool* zero) {
  const unsigned tiles = (unsigned)((a.Nk + AT_KEYS - 1) / AT_KEYS), per = (unsigned)(a.Hkv * a.row_splits);
  *zero = false;
  unsigned w, n = tiles, first = 0;
  int b;
  if (a.key_lengths == nullptr) {
    w = at_unit(gridDim.x);
    b = (int)(w / (per * tiles));
    w -= b * per * tiles;
  } else {
    auto count = [&](int clip) { return per * at_clip_key_tiles(a, clip); };
    const int i = at_unit(at_units(a.B, count));
    if (i < 0 && a.row_splits > 1) return false;     // (the join writes the zeros)
    *zero = i < 0;
    w = i < 0 ? -1 - i : i;
    if (i < 0) b = at_find_clip(a.B, [&](int clip) { return per * (tiles - at_clip_key_tiles(a, clip)); }, &w, &n);
    else b = at_find_clip(a.B, count, &w, &n);
    n /= per;
    first = i < 0 ? tiles - n : 0;
  }
  *u = at_decode(b, w, n, a.row_splits);
  u->tile += first;
  return true;
}

// waves per SIMD that the register allocation aims at
template <typename T, int DP> struct AtWaves {
  static constexpr bool BF16 = sizeof(T) == 2;
  static constexpr int FWD = DP == 32 ? 4 : DP == 64 ? 3 : DP == 96 ? 2 : (BF16 ? 2 : 1);
  static constexpr int DQ = DP == 32 ? 4 : DP == 64 ? (BF16 ? 3 : 2) : BF16 ? 2 : 1;
  static constexpr int DKV = DP == 32 ? (BF16 ? 3 : 2) : DP == 64 ? 2 : 1;
};

// The exponent of p: s scale2 - m.  A fused multiply-add knows s scale2 beyond the bits of m, which is the rounded product of the
// largest s: the largest p is 2^r, r up to half of m's last bit, and cancels from the normalised p.  From 2^31 on r would leave the
// range of f32 (the sum was inf or 0): there, and already from AT_FAR on, the product is rounded first, as m was.
__device__ __forceinline__ float at_exponent(float s, float scale2, float m) {
#pragma clang fp contract(off)
  const float product = s * scale2, rounded = product - m;
  return fabsf(m) >= AT_FAR ? rounded : fmaf(s, scale2, -m);
}

// 1 / l_r.  A row without keys: 0, its result and gradients are zeros.  A row that has keys but no positive sum -- all its scores are
// -inf, or one is NaN or +inf -- has no softmax: NaN, for its result and for every gradient that it enters.
__device__ __forceinline__ float at_inverse(float sum, bool keys) { return sum > 0.f ? 1.f / sum : keys ? NAN : 0.f; }

// ---------------------------------------------------------------------------------------------------------------- forward
// A workgroup: AT_QROWS query rows of one key head, `tiles_per_split` key tiles; two LDS buffers, the next tile's copies in
// flight under the current tile's products.  A score costs the vector unit a multiply-add, an exponential (two issue slots), half a
// maximum, an addition and three operations that split it in two parts (and, subtract, half a conversion, half a permutation): bound by
// that (0.74 of the vector unit's cycles) next to three products (0.45 of the matrix unit's).  Three waves a SIMD at 64 channels hold the
// operands (158 registers; at four they spill: 373 us for 337).  4096 x 49152 x 4 x 64, bf16: 334-337 us with the join, 0.92 PFLOP/s
// executed (the kernel alone 337 to 427 us, median 348, under the profiler's trace); f32 2 x 256 x 4096 x 8 x 32: 28.6 us, 75 TFLOP/s of 151.
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, (AtWaves<T, DP>::FWD)) void attn_fwd_kernel(AttnArgs a) {
  constexpr int EPC = AtFrag<T>::EPC, CH = DP / EPC, PC = AtPitch<T, DP>::V, KT = AtTile<T>::KT, NB = DP / 32;
  __shared__ __attribute__((aligned(16))) T kt[2][KT * PC * EPC];
  __shared__ __attribute__((aligned(16))) T vt[2][KT * PC * EPC];
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, h = l >> 5;
  AtUnit unit;
  if (!at_row_unit<T>(a, &unit)) return;
  const int b = unit.b, hk = unit.hk, split = unit.split;
  const unsigned row = (unsigned)(unit.tile * AT_QROWS + wave * 32 + (l & 31));
  const bool live = row < a.rows;
  const unsigned rr = live ? row : 0, in_group = rr / (unsigned)a.Nq;
  const int head = hk * a.G + (int)in_group;
  const long query = rr - in_group * (unsigned)a.Nq;
  const long len = at_key_len(a, b);
  const int t0 = split * a.tiles_per_split;
  const long n_tiles = (len + KT - 1) / KT;
  const int t1 = (int)(n_tiles < (long)t0 + a.tiles_per_split ? n_tiles : (long)t0 + a.tiles_per_split);
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];

  uint4 qf[CH / 2];
  const T* qp = (const T*)a.q + b * a.qs[0] + query * a.qs[1] + head * a.qs[2];
#pragma unroll
  for (int s = 0; s < CH / 2; ++s) {
    const int c = 2 * s + h;
    qf[s] = live && c * EPC < a.D ? ldg16(qp + c * EPC) : make_uint4(0, 0, 0, 0);
  }
  f32x16 o[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) o[d] = at_zero();
  float base = -INFINITY, sum = 0.f;   // base: of the exponentials, in powers of two
  uint64_t some = 0;                   // (of any tile) there are keys at all

  AtStage<T, KT, DP> sk, sv;
  sk.init(a.ks[1]);
  sv.init(a.vs[1]);
  AtKeyBits valid{a.key_mask ? a.key_mask + (long)b * a.Nk : nullptr, len, 1};
  uint64_t bits = 0;
  auto stage = [&](int t, int buf) {
    const long k0 = (long)t * KT;
    bits = valid.bits(k0);
    sk.rows(kt[buf], kp + k0 * a.ks[1], bits, a.D);
    sv.rows(vt[buf], vp + k0 * a.vs[1], bits, a.D);
    valid.fetch(k0 + KT);
  };
  valid.fetch((long)t0 * KT);
  if (t0 < t1) stage(t0, 0);
#pragma unroll
  for (int x = 0; x < CH / 2; ++x) pin(qf[x]);   // (waited for here, not behind the copies of every step)
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const uint64_t cur = bits;
    some |= cur;
    dma_wait<0>();
    __syncthreads();
    if (t + 1 < t1) stage(t + 1, buf ^ 1);
    f32x16 s[KT / 32];
    float top = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      s[kb] = at_zero();
#pragma unroll
      for (int x = 0; x < CH / 2; ++x) s[kb] = at_mma(at_chunk<T, PC>(kt[buf], kb * 32 + (l & 31), 2 * x + h), qf[x], s[kb], T{});
      const unsigned mb = (unsigned)(cur >> (32 * kb));
      if (mb != 0xffffffffu) {
        const unsigned mine = mb >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1 ? s[kb][i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[kb][i]);
    }
    // The base of the exponentials need not be the running maximum itself: it stays until a score is AT_SLACK powers of two above
    // it (sums and products stay below 2^AT_SLACK per key, far from f32's range), which spares nearly all rescaling of o.
    top = at_max_halves(top) * a.scale2;
    const bool move = top > base + AT_SLACK;          // (base -inf: every finite score moves it)
    if (__ballot(move) != 0) {
      const float alpha = move ? fast_exp2(base - top) : 1.f;
      if (move) base = top;
      sum *= alpha;
#pragma unroll
      for (int d = 0; d < NB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
    }
    const float off = base == -INFINITY ? 0.f : base;
    const bool far = __ballot(fabsf(off) >= AT_FAR) != 0;
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      if (far) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = fast_exp2(at_exponent(s[kb][i], a.scale2, off));
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = fast_exp2(fmaf(s[kb][i], a.scale2, -off));
      }
      sum = at_sum(s[kb], sum);
      if constexpr (sizeof(T) == 2) {
        unsigned w[8], v[8];
        at_operand2(s[kb], w, v);
#pragma unroll
        for (int d = 0; d < NB; ++d) {
          const AtTr x = at_tr<PC>(vt[buf], kb * 32, d * 32);
          at_mma_tr(o[d], x, w);
          at_mma_tr(o[d], x, v);
        }
      } else {
        AtOperand<T> p;
        at_operand(s[kb], p.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) at_mma_tr<PC>(o[d], vt[buf], kb * 32, d * 32, p.w);
      }
    }
  }
  sum = at_sum_halves(sum);
  if (!live) return;
  const long bh = (long)b * a.Hkv + hk;
  if (a.splits > 1) {
    float* po = a.part_o + (((long)split * a.B * a.Hkv + bh) * a.rows + row) * AtPart<DP>::V;
#pragma unroll
    for (int d = 0; d < NB; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        at_store4<float>(po + d * 32 + 8 * i + 4 * h, o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
    // (keys whose scores are all -inf: their sum of nothing is marked, for the join to tell it from a split without keys)
    if (h == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * ((bh * a.rows + row) * a.splits + split)) = make_float2(base, some != 0 && sum == 0.f ? 1.f : sum);
    return;
  }
  const float inv = at_inverse(sum, some != 0);
  const long at = (((long)b * a.Nq + query) * a.Hkv * a.G + head) * a.D;
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = d * 32 + 8 * i + 4 * h;
      if (c < a.D) {
        const float x = o[d][4 * i] * inv, y = o[d][4 * i + 1] * inv, z = o[d][4 * i + 2] * inv, u = o[d][4 * i + 3] * inv;
        at_store4<T>((T*)a.out + at + c, x, y, z, u);
        if (a.out32 && (const void*)a.out32 != a.out) at_store4<float>(a.out32 + at + c, x, y, z, u);
      }
    }
  if (a.stats && h == 0) *reinterpret_cast<float2*>(a.stats + 2 * (bh * a.rows + row)) = make_float2(base == -INFINITY ? 0.f : base, inv);
}

// joins the key splits:  o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.  WPR waves a row; the lanes of a wave are DP / 4
// groups of channels times the splits that they add in turn.  Bound by reading the partial results (4096 x 49152: 25 MB, 9.5 us; one
// query: 4-5 us, where one wave a row going through the splits one by one took 45 us).
template <typename T, int DP, int WPR>
__global__ __launch_bounds__(AT_THREADS) void attn_join_kernel(AttnArgs a) {
  constexpr int CG = DP / 4, SG = 64 / CG;      // channel groups, splits a wave adds at a time
  __shared__ __attribute__((aligned(16))) float red[WPR == 1 ? 1 : AT_WAVES][WPR == 1 ? 4 : DP + 4];
  const long bhs = (long)a.B * a.Hkv, total = bhs * a.rows;
  const int l = threadIdx.x & 63, w = WPR == 1 ? 0 : threadIdx.x >> 6;
  const long r = (long)blockIdx.x * (AT_WAVES / WPR) + (WPR == 1 ? threadIdx.x >> 6 : 0);
  if (r >= total) return;                       // (WPR > 1: the whole workgroup)
  const long bh = r / a.rows, row = r % a.rows, b = bh / a.Hkv, hk = bh % a.Hkv;
  const int splits = at_clip_splits<T>(a, (int)b);
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + r * a.splits;
  float top = -INFINITY;
  for (int s = l; s < splits; s += 64) top = fmaxf(top, ml[s].x);
  top = wave_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  bool keys = true;
  if (top == -INFINITY) {                       // no finite score: a row without keys, or one whose splits are marked
    bool mine = false;
    for (int s = l; s < splits; s += 64) mine = mine || ml[s].y != 0.f;
    keys = __ballot(mine) != 0;
  }
  const int c = (l % CG) * 4, g = l / CG;
  float sum = 0.f;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = w * SG + g; s < splits; s += WPR * SG) {
    const float2 e = ml[s];
    const float f = fast_exp2(e.x - base);
    const tapir_f32x4 v = ldg_f4(a.part_o + ((long)s * total + r) * DP + c);
    sum = fmaf(f, e.y, sum);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = fmaf(f, v[i], x[i]);
  }
#pragma unroll
  for (int m = CG; m < 64; m <<= 1) {
    sum += __shfl_xor(sum, m);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] += __shfl_xor(x[i], m);
  }
  if (WPR > 1) {
    if (g == 0) *reinterpret_cast<float4*>(&red[w][c]) = make_float4(x[0], x[1], x[2], x[3]);
    if (l == 0) red[w][DP] = sum;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (int q = 1; q < WPR; ++q) {
      sum += red[q][DP];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += red[q][c + i];
    }
  }
  const float inv = at_inverse(sum, keys);
  const long at = ((b * a.Nq + row % a.Nq) * a.Hkv * a.G + hk * a.G + row / a.Nq) * a.D;
  if (g == 0 && c < a.D) {
    at_store4<T>((T*)a.out + at + c, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    if (a.out32 && (const void*)a.out32 != a.out) at_store4<float>(a.out32 + at + c, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
  }
  if (a.stats && l == 0) *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(base, inv);
}

// --------------------------------------------------------------------------------------------------------------- backward
// dq (and D_r on the way): the forward kernel's loop with p from the saved statistics; 1 / l_r is a factor of the whole row and
// joins it at the end.  Keys are split like the forward pass': with few rows there are too few row tiles to fill the chip (256 rows of
// 4 heads are 8 workgroups: 1.2 ms unsplit).  Bound by matrix and vector instructions in turn (S, dP, two parts of dQ: 256 x 49152 x
// 4 x 64, bf16: 40 us, 0.65 PFLOP/s executed; f32 2 x 256 x 4096 x 8 x 32: 40 us, 80 TFLOP/s; matrix unit 0.35 and 0.60 busy).
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, (AtWaves<T, DP>::DQ)) void attn_dq_kernel(AttnArgs a) {
  constexpr int EPC = AtFrag<T>::EPC, CH = DP / EPC, PC = AtPitch<T, DP>::V, KT = AtTile<T>::KT, NB = DP / 32;
  constexpr bool BF16 = sizeof(T) == 2;
  __shared__ __attribute__((aligned(16))) T kt[2][KT * PC * EPC];
  __shared__ __attribute__((aligned(16))) T vt[2][KT * PC * EPC];
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, h = l >> 5;
  AtUnit unit;
  if (!at_row_unit<T>(a, &unit)) return;
  const int b = unit.b, hk = unit.hk, split = unit.split;
  const unsigned row = (unsigned)(unit.tile * AT_QROWS + wave * 32 + (l & 31));
  const bool live = row < a.rows;
  const unsigned rr = live ? row : 0, in_group = rr / (unsigned)a.Nq;
  const int head = hk * a.G + (int)in_group;
  const long query = rr - in_group * (unsigned)a.Nq;
  const long len = at_key_len(a, b);
  const int t0 = split * a.tiles_per_split;
  const long n_tiles = (len + KT - 1) / KT;
  const int t1 = (int)(n_tiles < (long)t0 + a.tiles_per_split ? n_tiles : (long)t0 + a.tiles_per_split);
  const T* kp = (const T*)a.k + b * a.ks[0] + hk * a.ks[2];
  const T* vp = (const T*)a.v + b * a.vs[0] + hk * a.vs[2];
  const long bh = (long)b * a.Hkv + hk;
  const long at = (((long)b * a.Nq + query) * a.Hkv * a.G + head) * a.D;

  uint4 qf[CH / 2], gf[CH / 2];
  const T* qp = (const T*)a.q + b * a.qs[0] + query * a.qs[1] + head * a.qs[2];
  const T* gp = (const T*)a.dout + b * a.ds[0] + query * a.ds[1] + head * a.ds[2];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < CH / 2; ++s) {
    const int c = 2 * s + h;
    const bool in = live && c * EPC < a.D;
    qf[s] = in ? ldg16(qp + c * EPC) : make_uint4(0, 0, 0, 0);
    gf[s] = in ? ldg16(gp + c * EPC) : make_uint4(0, 0, 0, 0);
    if (in) {
#pragma unroll
      for (int e = 0; e < EPC; ++e) delta = fmaf(Elem<T>::ld(gp + c * EPC + e), a.out32[at + c * EPC + e], delta);
    }
  }
  delta = at_sum_halves(delta);
  float row_max = a.stats[2 * (bh * a.rows + rr)], row_inv = a.stats[2 * (bh * a.rows + rr) + 1];
  if (live && h == 0 && split == 0) a.delta[bh * a.rows + row] = delta;
  f32x16 o[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) o[d] = at_zero();

  AtStage<T, KT, DP> sk, sv;
  sk.init(a.ks[1]);
  sv.init(a.vs[1]);
  f32x16 minus_delta;      // bf16: what the products with dout begin at
#pragma unroll
  for (int i = 0; i < 16; ++i) minus_delta[i] = -delta;
  AtKeyBits valid{a.key_mask ? a.key_mask + (long)b * a.Nk : nullptr, len, 1};
  uint64_t bits = 0;
  auto stage = [&](int t, int buf) {
    const long k0 = (long)t * KT;
    bits = valid.bits(k0);
    sk.rows(kt[buf], kp + k0 * a.ks[1], bits, a.D);
    sv.rows(vt[buf], vp + k0 * a.vs[1], bits, a.D);
    valid.fetch(k0 + KT);
  };
  valid.fetch((long)t0 * KT);
  if (t0 < t1) stage(t0, 0);
#pragma unroll
  for (int x = 0; x < CH / 2; ++x) { pin(qf[x]); pin(gf[x]); }
  pin(row_max);
  pin(row_inv);
  const bool far = __ballot(fabsf(row_max) >= AT_FAR) != 0;
  const float factor = far ? 1.f : a.scale2, offset = far ? 0.f : row_max;
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    const uint64_t cur = bits;
    dma_wait<0>();
    __syncthreads();
    if (t + 1 < t1) stage(t + 1, buf ^ 1);
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      f32x16 s = at_zero(), g = BF16 ? minus_delta : at_zero();
      if constexpr (sizeof(T) == 4 && DP > 64) {
        at_dot<T, PC>(s, kt[buf], kb * 32, qf);
        at_dot<T, PC>(g, vt[buf], kb * 32, gf);
      } else {
#pragma unroll
        for (int x = 0; x < CH / 2; ++x) {
          s = at_mma(at_chunk<T, PC>(kt[buf], kb * 32 + (l & 31), 2 * x + h), qf[x], s, T{});
          g = at_mma(at_chunk<T, PC>(vt[buf], kb * 32 + (l & 31), 2 * x + h), gf[x], g, T{});
        }
      }
      if (far) {
        const float m = a.stats[2 * (bh * a.rows + (row < a.rows ? row : 0))];    // (read again: a register less on the usual way)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = at_exponent(s[i], a.scale2, m);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], factor, -offset)) * (BF16 ? g[i] : g[i] - delta);
      const unsigned mb = (unsigned)(cur >> (32 * kb));
      if (mb != 0xffffffffu) {
        const unsigned mine = mb >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (mine >> (8 * (i >> 2) + (i & 3))) & 1 ? s[i] : 0.f;
      }
      if constexpr (BF16) {
        unsigned w[8], v[8];
        at_operand2(s, w, v);
#pragma unroll
        for (int d = 0; d < NB; ++d) {
          const AtTr x = at_tr<PC>(kt[buf], kb * 32, d * 32);
          at_mma_tr(o[d], x, w);
          at_mma_tr(o[d], x, v);
        }
      } else {
        AtOperand<T> p;
        at_operand(s, p.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) at_mma_tr<PC>(o[d], kt[buf], kb * 32, d * 32, p.w);
      }
    }
  }
  if (!live) return;
  const float f = row_inv * a.scale;
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = d * 32 + 8 * i + 4 * h;
      if (c < a.D) {
        const float x = o[d][4 * i] * f, y = o[d][4 * i + 1] * f, z = o[d][4 * i + 2] * f, u = o[d][4 * i + 3] * f;
        if (a.splits > 1) at_store4<float>(a.part_dq + split * a.n_dq + at + c, x, y, z, u);
        else at_store4<T>((T*)a.dq + at + c, x, y, z, u);
      }
    }
}

// D_r where dq is not wanted: two lanes a row, the sums in the order of attn_dq_kernel
template <typename T>
__global__ __launch_bounds__(AT_THREADS) void attn_delta_kernel(AttnArgs a) {
  constexpr int EPC = AtFrag<T>::EPC;
  const int l = threadIdx.x & 63;
  const long total = (long)a.B * a.Hkv * a.rows, r = ((long)blockIdx.x * AT_WAVES + (threadIdx.x >> 6)) * 32 + (l & 31);
  const bool live = r < total;
  const long rr = live ? r : 0, bh = rr / a.rows, row = rr % a.rows, b = bh / a.Hkv, head = bh % a.Hkv * a.G + row / a.Nq, query = row % a.Nq;
  const T* gp = (const T*)a.dout + b * a.ds[0] + query * a.ds[1] + head * a.ds[2];
  const float* op = a.out32 + ((b * a.Nq + query) * a.Hkv * a.G + head) * a.D;
  float delta = 0.f;
  for (int c = l >> 5; live && c * EPC < a.D; c += 2)
#pragma unroll
    for (int e = 0; e < EPC; ++e) delta = fmaf(Elem<T>::ld(gp + c * EPC + e), op[c * EPC + e], delta);
  delta = at_sum_halves(delta);
  if (live && l < 32) a.delta[r] = delta;
}

// dk, dv: a workgroup AT_KEYS keys of one key head, all query rows of the group's heads (or a split of them), RT at a time.
// Six products a step in bf16 (S, dP and two parts each of dV and dK).  K and V stay in registers as operands, dK and dV as sums: two
// waves a SIMD at 64 channels, one at 128.  Bound by matrix instructions for many rows (4096 x 49152: 1.0 PFLOP/s executed with dq), by
// loading and storing its keys for few (256 rows are four steps; 49152 x 4 x 64: 64 us, matrix unit 0.31 busy).
template <typename T, int DP>
__global__ __launch_bounds__(AT_THREADS, (AtWaves<T, DP>::DKV)) void attn_dkv_kernel(AttnArgs a) {
  constexpr int EPC = AtFrag<T>::EPC, CH = DP / EPC, PC = AtPitch<T, DP>::V, NB = DP / 32, RT = AtRowTile<T, DP>::RT;
  __shared__ __attribute__((aligned(16))) T qt[2][RT * PC * EPC];
  __shared__ __attribute__((aligned(16))) T gt[2][RT * PC * EPC];
  // what the rows' products start from and are multiplied by.  bf16: the products begin at -log2(e) L_r / scale2 and -D_r (L_r =
  // m_r + log l_r), so that p = exp2(scale2 s) and ds = p dp remain; f32: m_r, D_r and 1 / l_r apart, because one number L_r would
  // be rounded at its own size (2^-21 at 10, a relative error of 5 u of the whole row).
  constexpr bool BF16 = sizeof(T) == 2;
  // bf16: where m_r is large (AT_NEAR), the products' sums would be rounded at the size of L_r and p be off by more than a bf16
  // rounding: such steps, marked in `far`, form the scores again from zero and take m_r and log2(1 / l_r) apart, too (the test for it: 1 us of 276
  // and 1.5 of 114 a training step).
  __shared__ __attribute__((aligned(16))) float ld[2][BF16 ? 4 : 3][RT];
  __shared__ unsigned far[2];
  const int wave = threadIdx.x >> 6, l = threadIdx.x & 63, h = l >> 5;
  AtUnit unit;
  bool zero;
  if (!at_key_unit(a, &unit, &zero)) return;
  const int b = unit.b, hk = unit.hk, split = unit.split;
  const int kt = unit.tile;
  const long key = (long)kt * AT_KEYS + wave * 32 + (l & 31);
  const long len = at_key_len(a, b);
  bool in = key < len;
  if (in && a.key_mask != nullptr) in = a.key_mask[(long)b * a.Nk + key] != 0;
  const long bh = (long)b * a.Hkv + hk;
  uint4 kf[CH / 2], vf[CH / 2];
  const T* kp = (const T*)a.k + b * a.ks[0] + (in ? key : 0) * a.ks[1] + hk * a.ks[2];
  const T* vp = (const T*)a.v + b * a.vs[0] + (in ? key : 0) * a.vs[1] + hk * a.vs[2];
#pragma unroll
  for (int s = 0; s < CH / 2; ++s) {
    const int c = 2 * s + h;
    kf[s] = in && c * EPC < a.D ? ldg16(kp + c * EPC) : make_uint4(0, 0, 0, 0);
    vf[s] = in && c * EPC < a.D ? ldg16(vp + c * EPC) : make_uint4(0, 0, 0, 0);
  }
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (int d = 0; d < NB; ++d) { dk[d] = at_zero(); dv[d] = at_zero(); }
  const int t0 = split * a.row_steps_per_split, n_steps = zero ? 0 : (int)((a.rows + RT - 1) / RT);
  const int t1 = n_steps < t0 + a.row_steps_per_split ? n_steps : t0 + a.row_steps_per_split;
  // a step whose rows belong to one query head takes the same offsets as any other; where heads of fewer than RT queries meet
  // within a step, each chunk works its own row out
  const float unscale = 1.f / a.scale2;
  typedef AtStage<T, RT, DP> Stage;
  Stage sq, sg;
  sq.init(a.qs[1]);
  sg.init(a.ds[1]);
  const T* const qb = (const T*)a.q + b * a.qs[0] + (long)hk * a.G * a.qs[2];
  const T* const gb = (const T*)a.dout + b * a.ds[0] + (long)hk * a.G * a.ds[2];
  const int Nq = (int)a.Nq, n_rows = (int)a.rows;
  int head0 = 0, query0 = t0 * RT;   // of the next step's first row
  if (query0 >= Nq && t0 < t1) { head0 = (unsigned)query0 / (unsigned)Nq; query0 -= head0 * Nq; }
  const double per_query = 1.0 / (double)a.Nq;
  float2 row_stat = make_float2(0.f, 0.f);     // m_r and 1 / l_r, or D_r, of a row of the step that is staged next
  const float* const row_stats = a.stats + 2 * bh * a.rows;
  const float* const row_delta = a.delta + bh * a.rows;
  auto fetch = [&](int r0) {
    const int row = r0 + (int)(threadIdx.x & (RT - 1));
    row_stat = make_float2(0.f, 0.f);
    if (row < n_rows) {
      if (threadIdx.x < RT) row_stat = *reinterpret_cast<const float2*>(row_stats + 2 * (long)row);
      else if (threadIdx.x < 2 * RT) row_stat.x = row_delta[row];
    }
  };
  auto put_stats = [&](int buf) {
    const uint64_t large = __ballot(threadIdx.x < RT && fabsf(row_stat.x) >= (BF16 ? AT_NEAR : AT_FAR));
    if (threadIdx.x == 0) far[buf] = large != 0;      // (the rows are the first wave's)
    if (threadIdx.x < RT) {
      if (BF16) {
        const float l = log2f(row_stat.y);                        // (-inf for a row without keys: p = 0)
        ld[buf][0][threadIdx.x] = (l - row_stat.x) * unscale;
        ld[buf][BF16 ? 2 : 0][threadIdx.x] = row_stat.x;
        ld[buf][BF16 ? 3 : 0][threadIdx.x] = l;
      }
      else { ld[buf][0][threadIdx.x] = row_stat.x; ld[buf][BF16 ? 0 : 2][threadIdx.x] = row_stat.y; }
    } else if (threadIdx.x < 2 * RT) {
      ld[buf][1][threadIdx.x - RT] = BF16 ? -row_stat.x : row_stat.x;
    }
  };
  auto copy = [&](int t, int buf) {
    const int r0 = t * RT, left = n_rows - r0;
    if (query0 + RT <= Nq || (left < RT && query0 + left <= Nq)) {
      const uint64_t rows = left >= 64 ? ~0ull : (1ull << left) - 1;
      sq.rows(qt[buf], qb + head0 * a.qs[2] + query0 * a.qs[1], rows, a.D);
      sg.rows(gt[buf], gb + head0 * a.ds[2] + query0 * a.ds[1], rows, a.D);
    } else {
#pragma unroll
      for (int n = 0; n < Stage::N; ++n) {
        const int row = r0 + Stage::row(n);
        // row / Nq: the half keeps the quotient 0.5 / Nq away from whole numbers, far more than its rounding (rows < 2^31)
        const int head = (int)(((double)row + 0.5) * per_query), query = row - head * Nq;
        const bool ok = row < n_rows && Stage::chunk(n) * EPC < a.D;
        const T* const qp = qb + query * a.qs[1] + head * a.qs[2] + Stage::chunk(n) * EPC;
        const T* const gp = gb + query * a.ds[1] + head * a.ds[2] + Stage::chunk(n) * EPC;
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u), qv = ok ? ldg16(qp) : zero, gv = ok ? ldg16(gp) : zero;
        const int slot = (n * AT_THREADS + (int)threadIdx.x) * EPC;
        *reinterpret_cast<uint4*>(qt[buf] + slot) = qv;
        *reinterpret_cast<uint4*>(gt[buf] + slot) = gv;
      }
    }
    query0 += RT;
    if (query0 >= Nq) { const int more = (unsigned)query0 / (unsigned)Nq; head0 += more; query0 -= more * Nq; }
  };
  if (t0 < t1) {
    fetch(t0 * RT);
    copy(t0, 0);
    put_stats(0);
    fetch((t0 + 1) * RT);
  }
#pragma unroll
  for (int x = 0; x < CH / 2; ++x) { pin(kf[x]); pin(vf[x]); }
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    dma_wait<0>();
    __syncthreads();
    if (t + 1 < t1) {
      put_stats(buf ^ 1);         // (waits for the statistics: before the copies are under way)
      copy(t + 1, buf ^ 1);
      fetch((t + 2) * RT);
    }
    const bool large = at_uniform(far[buf]) != 0;
    const float factor = large ? 1.f : a.scale2;
    if constexpr (BF16) {
      // Operands are read from LDS a phase before the products that take them, and the fences keep it so: left to itself the
      // compiler reads each right before its product and waits (3 x 1000 x 8200 x 2 x 128: 119 -> 107 us).  64 and 96 channels
      // read the second block late: its operands did not fit the registers of two waves (115 -> 108 us for 64)
      uint4 qa[CH / 2], ga[CH / 2];
      auto read = [&](int rb) {
#pragma unroll
        for (int x = 0; x < CH / 2; ++x) {
          qa[x] = at_chunk<T, PC>(qt[buf], rb + (l & 31), 2 * x + h);
          ga[x] = at_chunk<T, PC>(gt[buf], rb + (l & 31), 2 * x + h);
        }
      };
      read(0);
#pragma unroll
      for (int rb = 0; rb < RT; rb += 32) {
        if ((DP == 64 || DP == 96) && rb > 0) read(rb);
        f32x16 s, g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const tapir_f32x4 L = *reinterpret_cast<const tapir_f32x4*>(&ld[buf][0][rb + 8 * i + 4 * h]);
          const tapir_f32x4 E = *reinterpret_cast<const tapir_f32x4*>(&ld[buf][1][rb + 8 * i + 4 * h]);
#pragma unroll
          for (int j = 0; j < 4; ++j) { s[4 * i + j] = L[j]; g[4 * i + j] = E[j]; }
        }
        AtTr gx[NB], qx[NB];
#pragma unroll
        for (int d = 0; d < NB; ++d) gx[d] = at_tr<PC>(gt[buf], rb, d * 32);
        sched_fence();
#pragma unroll
        for (int x = 0; x < CH / 2; ++x) {
          s = at_mma(qa[x], kf[x], s, T{});
          g = at_mma(ga[x], vf[x], g, T{});
        }
#pragma unroll
        for (int d = 0; d < NB; ++d) qx[d] = at_tr<PC>(qt[buf], rb, d * 32);
        if ((DP == 32 || DP == 128) && rb + 32 < RT) read(rb + 32);
        sched_fence();
        if (large) {
          s = at_zero();
#pragma unroll
          for (int x = 0; x < CH / 2; ++x) s = at_mma(at_chunk<T, PC>(qt[buf], rb + (l & 31), 2 * x + h), kf[x], s, T{});
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = rb + 8 * (i >> 2) + 4 * h + (i & 3);
            s[i] = at_exponent(s[i], a.scale2, ld[buf][BF16 ? 2 : 0][r]) + ld[buf][BF16 ? 3 : 0][r];
          }
        }
        AtOperand<T> p, e, f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = fast_exp2(s[i] * factor);
        at_operand2(s, p.w, f.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) at_mma_tr(dv[d], gx[d], p.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) at_mma_tr(dv[d], gx[d], f.w);
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] *= s[i];
        at_operand2(g, e.w, f.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) at_mma_tr(dk[d], qx[d], e.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) at_mma_tr(dk[d], qx[d], f.w);
      }
    } else {
#pragma unroll
      for (int rb = 0; rb < RT; rb += 32) {
        f32x16 s = at_zero(), g = at_zero();
        at_dot<T, PC>(s, qt[buf], rb, kf);
        at_dot<T, PC>(g, gt[buf], rb, vf);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const tapir_f32x4 M = *reinterpret_cast<const tapir_f32x4*>(&ld[buf][0][rb + 8 * i + 4 * h]);
          const tapir_f32x4 E = *reinterpret_cast<const tapir_f32x4*>(&ld[buf][1][rb + 8 * i + 4 * h]);
          const tapir_f32x4 I = *reinterpret_cast<const tapir_f32x4*>(&ld[buf][2][rb + 8 * i + 4 * h]);
          if (large) {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[4 * i + j] = at_exponent(s[4 * i + j], a.scale2, M[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[4 * i + j] = fmaf(s[4 * i + j], a.scale2, -M[j]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[4 * i + j] = fast_exp2(s[4 * i + j]) * I[j];
            g[4 * i + j] = s[4 * i + j] * (g[4 * i + j] - E[j]);
          }
        }
        AtOperand<T> p, e;
        at_operand(s, p.w);
        at_operand(g, e.w);
#pragma unroll
        for (int d = 0; d < NB; ++d) {
          at_mma_tr<PC>(dv[d], gt[buf], rb, d * 32, p.w);
          at_mma_tr<PC>(dk[d], qt[buf], rb, d * 32, e.w);
        }
      }
    }
  }
  if (key >= a.Nk) return;
  const long at = (((long)b * a.Nk + key) * a.Hkv + hk) * a.D;
#pragma unroll
  for (int d = 0; d < NB; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = d * 32 + 8 * i + 4 * h;
      if (c < a.D) {
        float x[4], y[4];   // (a masked key: zeros, also where dout holds something that is not finite)
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = in ? dk[d][4 * i + j] * a.scale : 0.f; y[j] = in ? dv[d][4 * i + j] : 0.f; }
        if (a.row_splits > 1) {
          at_store4<float>(a.part_dk + split * a.n_dkv + at + c, x[0], x[1], x[2], x[3]);
          at_store4<float>(a.part_dv + split * a.n_dkv + at + c, y[0], y[1], y[2], y[3]);
        } else {
          at_store4<T>((T*)a.dk + at + c, x[0], x[1], x[2], x[3]);
          at_store4<T>((T*)a.dv + at + c, y[0], y[1], y[2], y[3]);
        }
      }
    }
}

// adds the splits' shares of a gradient, in order (4 elements a thread; every row has a multiple of 8)
template <typename T>
__device__ __forceinline__ void at_add_shares(T* out, const float* part, long n, int shares, long i) {
  tapir_f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < shares; ++p) s += ldg_f4(part + p * n + i);
  at_store4<T>(out + i, s[0], s[1], s[2], s[3]);
}
template <typename T>
__global__ __launch_bounds__(AT_THREADS) void attn_join_grads_kernel(AttnArgs a) {
  const long nq = a.part_dq ? a.n_dq : 0, nk = a.part_dk ? a.n_dkv : 0;
  const long token = (long)a.Hkv * a.D, clip_q = a.rows * token, clip_k = a.Nk * token;   // elements
  for (long i = 4 * ((long)blockIdx.x * AT_THREADS + threadIdx.x); i < nq + 2 * nk; i += 4L * gridDim.x * AT_THREADS) {
    if (i < nq) {
      at_add_shares((T*)a.dq, a.part_dq, a.n_dq, at_clip_splits<T>(a, a.key_lengths ? (int)(i / clip_q) : 0), i);
      continue;
    }
    const bool of_v = i >= nq + nk;
    const long at = i - nq - (of_v ? nk : 0);
    const bool gone = a.key_lengths && at % clip_k / token >= at_key_len(a, (int)(at / clip_k));
    at_add_shares((T*)(of_v ? a.dv : a.dk), of_v ? a.part_dv : a.part_dk, a.n_dkv, gone ? 0 : a.row_splits, at);
  }
}

}  // namespace tapir
