// attention_op.h -- attention with its backward pass on caller-owned tensors: the kernels, as templates over the element type
// and the padded head size (attention_f32.hip, attention_f16.hip and attention_bf16.hip instantiate them).
//
// x_ij = scale q_i . k_j over the visible keys, lse_i = log sum_j exp x_ij, p_ij = exp(x_ij - lse_i), o_i = sum_j p_ij v_j, and
// with delta_i = do_i . o_i:  ds_ij = p_ij (do_i . v_j - delta_i),  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
// dv_j = sum_i p_ij do_i.  The probabilities are recomputed from lse, nothing of size rows x keys is ever in memory.
//
// Rows.  The query rows of one key head are the pairs (i, g), i < q_len, g < group, walked as "row" i * group + g: the heads
// that share a key head share its tiles, a lone token still fills `group` rows, and the sums of dk and dv over a group run in a
// fixed order inside one workgroup.  No atomics: two runs give the same bits.
//
// Layout of a product.  Everything is 32 x 32 tiles on the 16-deep matrix instruction of the 16-bit types (fp32: eight 2-deep
// ones over the same registers).  Lane l holds elements k = 8 (l / 32) + 0..7 of row (column) l % 32 of an operand and column
// l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4 of a result.  A result is used as the next product's right operand without leaving
// its registers: result rows 16 t + 8 (e / 4) + 4 (l / 32) + e % 4, e < 8, are taken as the k slots 8 (l / 32) + e, and the left
// operand, read transposed from LDS, follows the same order.  Forward and dq therefore compute the transposed scores (a lane
// holds one query row: its maximum and sum need one exchange between the half waves), dk / dv the straight ones.
#pragma once
#include "operator_common.h"

#include <algorithm>
#include <type_traits>

namespace urf {

struct AttnView { void *p; long long b, r, h; };   // base, strides in elements: batch, row, head

struct AttnArgs {
  AttnView q, k, v, o, dout, dq, dk, dv;
  const int *q_lens, *k_lens;    // rows in use per sequence (null = all)
  float *lse;                    // [B][Hq][Lq], natural logarithm
  float *delta;                  // [B][Hq][Lq] (backward)
  float *norm_do, *norm_v;       // |do_i| [B][Hq][Lq], |v_j| [B][Hk][Lk] (backward, f16)
  float *part_o, *part_ml;       // forward over split keys: [split][B * Hk][Lq * G][DP] and (maximum, sum)
  float *part_kv, *part_q;       // backward in parts: dk then dv [split][B * Hk][Lk][DP]; dq [split][B * Hk][Lq * G][DP]
  int B, Hq, Hk, G, Lq, Lk, D;
  int causal;
  int splits;                    // forward: key ranges
  int tiles;                     // its row tiles per (sequence, key head)
  int kv_tiles, kv_splits, q_tiles, q_splits;   // backward: tiles of 128 keys / rows, and ranges of the other side
  int few_tiles;                 // backward: tiles of 128 rows per (sequence, key head) that may hold rows of few keys
  float scale, scale2;           // scale, scale * log2(e)
};

// ------------------------------------------------------------------ element types
template <typename T> struct Elem;
template <> struct Elem<__bf16> {
  typedef b16x8 Frag;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<_Float16> {
  typedef h16x8 Frag;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<float> {
  typedef f32x8 Frag;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
  }
};

// eight values of a result as an operand: the one rounding of the probabilities (and of ds) to the inputs' type, as the matrix
// instruction takes them; sums, maxima and every accumulator stay in fp32
template <typename T> __device__ __forceinline__ typename Elem<T>::Frag to_frag(const f32x16 &c, int t) {
  typename Elem<T>::Frag f;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = (T)c[8 * t + e];
  return f;
}

// ------------------------------------------------------------------ LDS tiles
// A tile is rows of 64 or 128 elements (head sizes padded to 32, 64, 96 or 128), row r's 16-byte chunk c at chunk position
// c ^ swizzle(r).  16-bit types: eight consecutive
// lanes of a row-wise fragment read (eight rows, one chunk) and the half wave of a transposed read (four rows, four chunks)
// each fall into distinct banks.
template <typename T, int DP> struct Tile {
  static constexpr int kPer = 16 / (int)sizeof(T);          // elements of a chunk
  static constexpr int kPitch = DP <= 64 ? 64 : 128;
  static constexpr int kChunks = kPitch / kPer;
  static constexpr int kBytes = kPitch * (int)sizeof(T);    // of a row
  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (sizeof(T) == 4) return (((r >> 2) & 1) << 3) | ((r & 3) << 1);
    else if constexpr (kBytes == 256) return ((r & 3) << 2) | ((r >> 2) & 3);
    else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ char *at(char *tile, int r, int c) { return tile + r * kBytes + ((c ^ swizzle(r)) << 4); }
  // Elements 16 kc + 8 half .. + 7 of row r0 + r: `base` = row_base(r, half), once; r0 a multiple of 16 (the swizzle's period), so
  // that a read costs one xor of the address, the rest is its immediate offset.
  static __device__ __forceinline__ unsigned row_base(int r, int half) {
    return r * kBytes + (((sizeof(T) == 2 ? half : 2 * half) ^ swizzle(r)) << 4);
  }
  // (`base` may include an offset into LDS that is a multiple of 512 bytes; `tile` + r0 rows should be constant)
  static __device__ __forceinline__ typename Elem<T>::Frag row(const char *tile, unsigned base, int r0, int kc) {
    const char *p = tile + r0 * kBytes;
    if constexpr (sizeof(T) == 2) {
      return *(const typename Elem<T>::Frag *)(p + (base ^ (kc << 5)));
    } else {
      const f32x4 a = *(const f32x4 *)(p + (base ^ (kc << 6))), b = *(const f32x4 *)(p + (base ^ (kc << 6) ^ 16));
      f32x8 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
      return f;
    }
  }
  // Column 32 dt + l % 32 of rows r0 + {4 half + 0..3, 8 + 4 half + 0..3}, r0 a multiple of 16: the left operand of a product over
  // rows.  16-bit types: the 16 lanes of a group read four rows of 16 elements, four elements a lane, and get one column of four
  // rows each.
  struct ColBase {
    unsigned a, b;
    __device__ __forceinline__ ColBase operator+(unsigned off) const { return {a + off, b + off}; }
  };
  static __device__ __forceinline__ ColBase col_base(int lane) {
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, r = 4 * half + (i >> 2), c = 2 * ((lane >> 4) & 1) + ((i >> 1) & 1);
      return {(unsigned)(r * kBytes + ((c ^ swizzle(r)) << 4) + 8 * (i & 1)), (unsigned)((r + 8) * kBytes + ((c ^ swizzle(r + 8)) << 4) + 8 * (i & 1))};
    } else {
      const int d = lane & 31, r = 4 * half;               // rows r + 0..3 differ in the swizzle's bits 5 and 6 of the address
      return {(unsigned)(r * kBytes + (((d >> 2) ^ swizzle(r)) << 4) + 4 * (d & 3)), (unsigned)((r + 8) * kBytes + (((d >> 2) ^ swizzle(r + 8)) << 4) + 4 * (d & 3))};
    }
  }
  static __device__ __forceinline__ typename Elem<T>::Frag column(const char *tile, const ColBase &base, int r0, int dt) {
    const char *p = tile + r0 * kBytes;
    typename Elem<T>::Frag f;
    if constexpr (sizeof(T) == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + (base.a ^ (dt << 6))));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(p + (base.b ^ (dt << 6))));
      typedef T T4 __attribute__((ext_vector_type(4)));
      const T4 x = __builtin_bit_cast(T4, a), y = __builtin_bit_cast(T4, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) { f[e] = x[e]; f[4 + e] = y[e]; }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        f[e] = *(const float *)(p + (e & 3) * kBytes + ((e < 4 ? base.a : base.b) ^ (dt << 7) ^ ((e & 3) << 5)));
    }
    return f;
  }
};

// Copies tiles of R consecutive rows into LDS, one after the other, through registers: load() fetches the next tile, store() writes
// it.  Rows outside [low, end) and chunks beyond the head size become zero -- what lies behind a
// sequence's end may be anything, NaN included, and never enters a product.  Every thread walks pointers of its own: an (i, g) row advances by R rows without a
// division.
template <typename T, int DP, int R> struct Stage {
  typedef Tile<T, DP> TL;
  static constexpr int kN = R * TL::kChunks / 256;
  static_assert(R * TL::kChunks % 256 == 0, "whole chunks per thread");
  u32x4 x[kN];
  const T *p[kN];
  int g[kN], row, group;            // row of chunk 0, from `low` on; chunk n is 256 / kChunks * n rows further
  long long step, wrap;
  bool inner;                       // the chunk lies within the head size
  __device__ __forceinline__ void start(const T *head, long long srow, long long shead, int grp, int first, int D, int tid, int low = 0) {
    group = grp;
    row = first + tid / TL::kChunks;
    const int c = tid % TL::kChunks;
    inner = c * TL::kPer < D;
    step = (long long)(R / grp) * srow + (long long)(R % grp) * shead;
    wrap = srow - (long long)grp * shead;
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int r = row + 256 / TL::kChunks * n, i = grp == 1 ? r : r / grp;
      g[n] = r - i * grp;
      p[n] = head + (long long)i * srow + (long long)g[n] * shead + c * TL::kPer;
    }
    row -= low;
  }
  // count = end - low, not negative.  DOWN: the tiles are walked towards the first row
  template <bool DOWN = false> __device__ __forceinline__ void load(int count) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      x[n] = u32x4{0, 0, 0, 0};
      if (inner && (unsigned)(row + 256 / TL::kChunks * n) < (unsigned)count) x[n] = *(const u32x4 *)p[n];
      p[n] += DOWN ? -step : step;
      if (group > 1) {
        g[n] += DOWN ? -(R % group) : R % group;
        if (DOWN ? g[n] < 0 : g[n] >= group) { g[n] += DOWN ? group : -group; p[n] += DOWN ? -wrap : wrap; }
      }
    }
    row += DOWN ? -R : R;
  }
  __device__ __forceinline__ void store(char *tile, int tid) const {
    char *p = TL::at(tile, tid / TL::kChunks, tid % TL::kChunks);
#pragma unroll
    for (int n = 0; n < kN; ++n) *(u32x4 *)(p + n * (256 / TL::kChunks) * TL::kBytes) = x[n];
  }
};

// operand fragments of one row straight from memory (the row a lane keeps for the whole kernel); zero where there is none
template <typename T> __device__ __forceinline__ typename Elem<T>::Frag load_frag(const T *row, bool valid, int kc, int half, int D) {
  typename Elem<T>::Frag f = {};
  const int d = 16 * kc + 8 * half;
  if (valid && d < D) {
    if constexpr (sizeof(T) == 2) {
      f = *(const typename Elem<T>::Frag *)(row + d);
    } else {
      const f32x4 a = *(const f32x4 *)(row + d), b = *(const f32x4 *)(row + d + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
    }
  }
  return f;
}

template <typename T> __device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  *(T4 *)p = T4{(T)a, (T)b, (T)c, (T)d};
}

// a lane's column of a transposed accumulator (row `p` of the output): four consecutive elements at a time; 0 where nothing was `seen`,
// whatever the others' keys left there (0 times infinity)
template <typename T, int DP> __device__ __forceinline__ void store_rows(T *p, const f32x16 *acc, float f, bool seen, int D, int half) {
  auto of = [&](float x) { return seen ? x * f : 0.0f; };
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * dt + 2 * r + 4 * half;
      if (d < D) store4<T>(p + d, of(acc[dt][r]), of(acc[dt][r + 1]), of(acc[dt][r + 2]), of(acc[dt][r + 3]));
    }
}

// in a branch: keeps the compiler from turning the branch into selects that every tile pays for
__device__ __forceinline__ void stay_a_branch() { asm volatile(""); }

__device__ __forceinline__ int clamp_len(const int *lens, int b, int most) {
  return lens ? min(max(lens[b], 0), most) : most;      // lengths come from device memory: never trusted beyond the tensor
}

// ------------------------------------------------------------------ forward
// workgroups of four waves per CU that the registers are kept for (fp32 rows of 128: twice the registers of everything)
template <typename T, int DP> constexpr int kBlocksPerCu = sizeof(T) == 2 || DP <= 64 ? 2 : 1;
constexpr float kSlack = 6.0f;      // log2: probabilities may grow by 64 before the maximum moves
// f16: probabilities start from 2^9, not from 1 (up to 2^15 with the slack): many small ones, which may be most of a row together, are
// rounded to its subnormal numbers 2^9 times later (300000 keys of 2^-25 of the largest's probability: those behind it were lost altogether)
template <typename T> constexpr int kLift = std::is_same<T, _Float16>::value ? 9 : 0;
// A row's lse and what its accumulators are divided by, from its maximum (log2 units, less kLift) and sum.  The sum is 0 for a row that saw
// no key and no other; a NaN, which a NaN or an infinite score leaves in it, goes into both.  (The logarithm is taken of the sum
// without the lift: near 9 its rounding would be most of the lse's error.)
template <typename T> __device__ __forceinline__ float row_lse(float m, float l) {
  return l == 0.0f ? -INFINITY : ((m + kLift<T>) + log2f(l * (1.0f / (1 << kLift<T>)))) * kLn2;
}
__device__ __forceinline__ float row_inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
// One workgroup: SPLIT = 0: 128 rows, 32 per wave, over tiles of 64 keys; SPLIT = 1: 32 rows, each of the four waves a quarter of
// a 128-key tile, joined through LDS at the end (few rows: more workgroups, more loads in flight).  The key range may be cut in
// `splits` parts, joined by attn_join_kernel.
// Bound: long rows, matrix instructions and exponentials of two waves per SIMD (2 x 16 heads of 4096 x 4096 x 128, causal, bf16: 137 GFLOP in
// 159 us, 864 TFLOP/s, 0.75 of what a large library product reaches).  Heads of 64, up to 1024 keys (16 x 4 heads, a quarter of the rows
// unused, bf16): 36 us, 370 TFLOP/s; 64 keys take a workgroup 2 us, of which neither exponentials nor loads alone are worth more than
// 0.3 (36.5 us -> 30.9 without the former, 32.0 without the latter).  fp32, 4 x 4 heads of 1000 x 1000 x 64: 4.1 GFLOP in 47 us, 87 TFLOP/s of 153.
// Single tokens, the keys' bytes (32 sequences of up to 16384 keys, 8 key heads of 128, bf16: 1.63 GB in 290 us, 5.6 TB/s).
template <typename T, int DP, int SPLIT>
__global__ void __launch_bounds__(256, (kBlocksPerCu<T, DP>)) attn_forward_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  constexpr int kKeys = SPLIT ? 128 : 64, kRows = SPLIT ? 32 : 128, kKc = DP / 16, kDt = DP / 32, kSub = SPLIT ? 1 : 2;
  extern __shared__ __align__(16) char lds[];
  constexpr int kTile = kKeys * TL::kBytes;                // k, then v; SPLIT = 0: two buffers, one barrier per tile
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const unsigned wave_rows = SPLIT ? 32 * wave * TL::kBytes : 0;       // SPLIT: the wave's own keys of a tile
  const unsigned row_base = TL::row_base(col, half) + wave_rows;
  const typename TL::ColBase col_base = TL::col_base(lane) + wave_rows;
  int tile, group;
  xcd_group_map(blockIdx.x, a.tiles * a.splits, a.B * a.Hk, tile, group);
  const int split = tile % a.splits;
  tile = a.tiles - 1 - tile / a.splits;                    // causal: the longest tiles first
  const int b = group / a.Hk, hk = group % a.Hk;
  const int nq = clamp_len(a.q_lens, b, a.Lq), nk = clamp_len(a.k_lens, b, a.Lk);
  const int row = tile * kRows + (SPLIT ? 0 : 32 * wave) + col, i = row / a.G, g = row - i * a.G;
  const bool inside = row < a.Lq * a.G, active = i < nq;
  // keys [0, seen) are visible to this lane's row, [0, block_end) to any row of the workgroup
  const int seen = !active ? 0 : a.causal ? min(nk, max(0, i + 1 + nk - nq)) : nk;
  const int i_last = min(nq, (min((tile + 1) * kRows, a.Lq * a.G) - 1) / a.G + 1) - 1, i_first = tile * kRows / a.G;
  int block_end = i_first >= nq ? 0 : a.causal ? min(nk, max(0, i_last + 1 + nk - nq)) : nk;
  const int full_end = a.causal ? min(nk, max(0, i_first + 1 + nk - nq)) : nk;     // every active row sees the keys below it
  const bool all_active = (i_last + 1) * a.G >= (tile + 1) * kRows;               // no row of the tile lies behind nq
  int begin = 0;
  if (a.splits > 1) {
    const int t = (block_end + kKeys - 1) / kKeys, per = (t + a.splits - 1) / a.splits;
    begin = min(block_end, split * per * kKeys);
    block_end = min(block_end, (split + 1) * per * kKeys);
  }
  const T *qrow = (const T *)a.q.p + (long long)b * a.q.b + (long long)i * a.q.r + (long long)(hk * a.G + g) * a.q.h;
  const T *kh = (const T *)a.k.p + (long long)b * a.k.b + (long long)hk * a.k.h;
  const T *vh = (const T *)a.v.p + (long long)b * a.v.b + (long long)hk * a.v.h;
  Frag q[kKc];
#pragma unroll
  for (int kc = 0; kc < kKc; ++kc) q[kc] = load_frag<T>(qrow, active, kc, half, a.D);
  f32x16 acc[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) acc[dt] = f32x16{};
  float m = -INFINITY, l = 0.0f;          // running maximum (log2 units; f16: 2^9 below it) and this half wave's share of the sum
  Stage<T, DP, kKeys> ks, vs;
  ks.start(kh, a.k.r, 0, 1, begin, a.D, tid);
  vs.start(vh, a.v.r, 0, 1, begin, a.D, tid);
  ks.load(block_end);
  vs.load(block_end);
  ks.store(lds, tid);
  vs.store(lds + kTile, tid);
  int buffer = 0;
  for (int key0 = begin; key0 < block_end; key0 += kKeys) {
    lds_barrier();                        // this tile is written, the other buffer (if any) has been read
    const unsigned at = buffer * 2 * kTile;
    const bool more = key0 + kKeys < block_end;
    if (more) {
      ks.load(block_end);
      vs.load(block_end);
    }
    f32x16 s[kSub];
    // the matrix instructions first, whichever wave of the SIMD has them ready: the other's exponentials fill the gaps (169 -> 155 us
    // for 2 x 16 heads of 4096 x 4096 x 128, causal, bf16)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      s[u] = f32x16{};
#pragma unroll
      for (int kc = 0; kc < kKc; ++kc) s[u] = Elem<T>::mma(TL::row(lds, row_base + at, 32 * u, kc), q[kc], s[u]);
    }
    __builtin_amdgcn_s_setprio(0);
    if (key0 + kKeys > min(full_end, block_end) || !all_active) {
      stay_a_branch();
      const int end = min(seen, block_end);
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        const int k0 = key0 + (SPLIT ? 32 * wave : 32 * u) + 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 8 * (r >> 2) + (r & 3) >= end) s[u][r] = -INFINITY;
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    // The running maximum only has to keep the exponentials in range: it moves when some row of the wave has grown by more than
    // 2^kSlack, so that the accumulators are rescaled once or twice per row, not once per tile, and the half waves' maxima are
    // brought together only then.
    if (__any(top * a.scale2 > m + (kSlack + kLift<T>))) {
      const float mn = fmaxf(m, fmaf(fmaxf(top, __shfl_xor(top, 32, 64)), a.scale2, -kLift<T>)), alpha = mn == -INFINITY ? 1.0f : exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) acc[dt] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.0f : m;           // nothing visible yet: all the exponentials are 0
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], a.scale2, -mu));
        sum += s[u][r];
      }
    l += sum;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag p = to_frag<T>(s[u], t);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) acc[dt] = Elem<T>::mma(TL::column(lds + kTile, col_base + at, 32 * u + 16 * t, dt), p, acc[dt]);
      }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (!SPLIT) buffer ^= 1;
    if (more) {
      if constexpr (SPLIT) lds_barrier();
      ks.store(lds + buffer * 2 * kTile, tid);
      vs.store(lds + buffer * 2 * kTile + kTile, tid);
    }
  }
  l += __shfl_xor(l, 32, 64);
  if constexpr (SPLIT) {                  // join the four waves: the maxima and sums, then the scaled accumulators
    float *ml = (float *)lds, *part = ml + 4 * 32 * 2;                     // part: [wave][DP][32]
    lds_barrier();
    if (half == 0) { ml[(wave * 32 + col) * 2] = m; ml[(wave * 32 + col) * 2 + 1] = l; }
    lds_barrier();
    float mm = -INFINITY, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[(w * 32 + col) * 2]);
    const float mu = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
    for (int w = 0; w < 4; ++w) ll += ml[(w * 32 + col) * 2 + 1] * exp2f(ml[(w * 32 + col) * 2] - mu);
    const float f = exp2f(m - mu);
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) part[(wave * DP + 32 * dt + 8 * (r >> 2) + 4 * half + (r & 3)) * 32 + col] = acc[dt][r] * f;
    lds_barrier();
    m = mm; l = ll;
    // wave w keeps the column groups [w * DP / 4, (w + 1) * DP / 4) of all 32 rows
    constexpr int kOwn = DP / 8;          // values of a lane: its half of the wave's DP / 4 columns
    float ov[kOwn];
#pragma unroll
    for (int e = 0; e < kOwn; ++e) {
      const int d = wave * (DP / 4) + half * kOwn + e;
      ov[e] = ((part[d * 32 + col] + part[(DP + d) * 32 + col]) + part[(2 * DP + d) * 32 + col]) + part[(3 * DP + d) * 32 + col];
    }
    const int d0 = wave * (DP / 4) + half * kOwn;
    if (!inside) return;
    if (a.splits > 1) {
      const long long prow = ((long long)split * a.B * a.Hk + group) * ((long long)a.Lq * a.G) + row;
#pragma unroll
      for (int e = 0; e < kOwn; e += 4) store4<float>(a.part_o + prow * DP + d0 + e, ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
      if (wave == 0 && half == 0) { a.part_ml[prow * 2] = m; a.part_ml[prow * 2 + 1] = l; }
    } else {
      const float inv = row_inverse(l);
      T *orow = (T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)(hk * a.G + g) * a.o.h;
#pragma unroll
      for (int e = 0; e < kOwn; ++e) ov[e] = l == 0.0f ? 0.0f : ov[e] * inv;
#pragma unroll
      for (int e = 0; e < kOwn; e += 4)
        if (d0 + e < a.D) store4<T>(orow + d0 + e, ov[e], ov[e + 1], ov[e + 2], ov[e + 3]);
      if (wave == 0 && half == 0) a.lse[((long long)b * a.Hq + hk * a.G + g) * a.Lq + i] = row_lse<T>(m, l);
    }
  } else if (inside) {
    const float inv = row_inverse(l);
    store_rows<T, DP>((T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)(hk * a.G + g) * a.o.h, acc, inv, l != 0.0f, a.D, half);
    if (half == 0) a.lse[((long long)b * a.Hq + hk * a.G + g) * a.Lq + i] = row_lse<T>(m, l);
  }
}

// Joins the key ranges: a wave per row; fixed order over the ranges.  Bound by latency (1024 rows of 128 in eight ranges: 7 us).
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
  const int lane = threadIdx.x & 63, rows = a.Lq * a.G;
  const unsigned w = blockIdx.x * 4 + (threadIdx.x >> 6);       // (rows of all heads: below 2^28)
  if (w >= (unsigned)(a.B * a.Hk * rows)) return;
  const int group = w / rows, row = w - group * rows, b = group / a.Hk, hk = group % a.Hk, i = row / a.G, g = row - i * a.G;
  const long long step = (long long)a.B * a.Hk * rows, base = w;
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[(base + s * step) * 2]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const float mu = m == -INFINITY ? 0.0f : m;
  constexpr int kN = (DP + 63) / 64;       // columns lane and lane + 64
  float l = 0.0f, o[kN];
#pragma unroll
  for (int e = 0; e < kN; ++e) o[e] = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const long long p = base + s * step;
    const float f = exp2f(a.part_ml[p * 2] - mu);
    l += a.part_ml[p * 2 + 1] * f;
#pragma unroll
    for (int e = 0; e < kN; ++e)
      if (lane + 64 * e < DP) o[e] += a.part_o[p * DP + lane + 64 * e] * f;
  }
  const float inv = row_inverse(l);
  T *orow = (T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)(hk * a.G + g) * a.o.h;
#pragma unroll
  for (int e = 0; e < kN; ++e)
    if (lane + 64 * e < a.D) orow[lane + 64 * e] = (T)(l == 0.0f ? 0.0f : o[e] * inv);
  if (lane == 0) a.lse[((long long)b * a.Hq + hk * a.G + g) * a.Lq + i] = row_lse<T>(m, l);
}

// ------------------------------------------------------------------ backward
// The range of f16 in the backward pass's second products.  Probabilities are about 1 / keys and gradients of any size, so that p and ds
// as they are would be rounded among f16's subnormal numbers, in steps of 2^-24 (8192 keys, do ~ 1e-3: dq and dk off by 0.011 of their
// norm, one rounding of the results 0.0009), and large ones beyond its largest.  p <= 1 is taken times 2^14, ds times a power of two that
// brings its bound |do_i| |v_j| + |delta_i| (the largest among the rows and keys of a workgroup for dk, of a row for dq) to 2^14..2^15:
// a subtraction becomes an fma, an exponent is shifted, and the results are multiplied by the inverse in fp32.  Terms down to 2^-29 of
// the bound have all of f16's bits.  The norms are made beside delta.  (us, 16 x 4 heads of 1024 x 1024 x 64 / 2 x 16 heads of 4096 x 4096 x
// 128, causal: 88 / 604, without any of it 82 / 588.  Following the largest term seen so far, as the forward pass does, needs no norms, but
// its branch stands between the products: 92 / 735.)
template <typename T> constexpr bool kScaled = std::is_same<T, _Float16>::value;
constexpr int kProbShift = 14;
template <typename T> constexpr float kDvScale = kScaled<T> ? 1.0f / (1 << kProbShift) : 1.0f;
// the exponent of the power of two for ds below `bound`
__device__ __forceinline__ int grad_shift(float bound) { return min(14 + 127 - (__float_as_int(bound) >> 23), 60); }
__device__ __forceinline__ float finite_max(float m, float x) { return x < INFINITY ? fmaxf(m, x) : m; }       // (x >= 0 or NaN)
// over the workgroup; `lds`: 16 bytes that nothing else uses until the caller's next barrier
__device__ __forceinline__ float block_max(float m, float *lds) {
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  lds_barrier();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  lds_barrier();
  return fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
}

// Rows that see up to 64 keys, 16-bit types: delta_i = sum_j p_ij (do_i . v_j) in fp32.  o was rounded, and where few keys share a row that
// error is as large as the gradients' own rounding (4 keys: dq and dk off by 2.05 of what one rounding costs, 15: 1.74, 30: 1.59; two
// roundings, of ds and of the result, are 1.41).  With more keys o's entries are small beside v's, and do . o is as good.
constexpr int kFewKeys = 64;
// the keys of row i of nq, if these are few, or 0
__device__ __forceinline__ int few_keys(int i, int nq, int nk, int causal) {
  const int seen = i >= nq ? 0 : causal ? min(nk, max(0, i + 1 + nk - nq)) : nk;
  return seen <= kFewKeys ? seen : 0;
}
template <typename T, int DP> __device__ __forceinline__ void attn_few_keys(const AttnArgs &a, int id, char *lds) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const unsigned row_base = TL::row_base(col, half);
  const int group = id / a.few_tiles, tile = id - group * a.few_tiles, b = group / a.Hk, hk = group % a.Hk;
  const int nq = clamp_len(a.q_lens, b, a.Lq), nk = clamp_len(a.k_lens, b, a.Lk);
  const int i_first = max(tile * 128 / a.G, a.causal ? nq - nk : 0), i_last = min(nq, (min((tile + 1) * 128, a.Lq * a.G) - 1) / a.G + 1) - 1;
  if (i_first > i_last || few_keys(i_first, nq, nk, a.causal) == 0) return;        // the first row that sees a key sees the fewest
  const int end = a.causal ? min(min(nk, kFewKeys), i_last + 1 + nk - nq) : nk;
  const int row = tile * 128 + 32 * wave + col, i = row / a.G, g = row - i * a.G, h = hk * a.G + g, few = few_keys(i, nq, nk, a.causal);
  const T *qrow = (const T *)a.q.p + (long long)b * a.q.b + (long long)i * a.q.r + (long long)h * a.q.h;
  const T *drow = (const T *)a.dout.p + (long long)b * a.dout.b + (long long)i * a.dout.r + (long long)h * a.dout.h;
  constexpr int kTile = kFewKeys * TL::kBytes;
  {
    Stage<T, DP, kFewKeys> x;
    x.start((const T *)a.k.p + (long long)b * a.k.b + (long long)hk * a.k.h, a.k.r, 0, 1, 0, a.D, tid);
    x.load(end);
    x.store(lds, tid);
    x.start((const T *)a.v.p + (long long)b * a.v.b + (long long)hk * a.v.h, a.v.r, 0, 1, 0, a.D, tid);
    x.load(end);
    x.store(lds + kTile, tid);
  }
  const long long at = ((long long)b * a.Hq + h) * a.Lq + i;
  const float lse = few ? a.lse[at] : -INFINITY, ls = lse == -INFINITY ? INFINITY : lse * kLog2e;
  lds_barrier();
  float delta = 0.0f;
#pragma unroll
  for (int u = 0; u < kFewKeys / 32; ++u) {
    f32x16 s = {}, dp = {};
#pragma unroll
    for (int kc = 0; kc < DP / 16; ++kc) {
      s = Elem<T>::mma(TL::row(lds, row_base, 32 * u, kc), load_frag<T>(qrow, few, kc, half, a.D), s);
      dp = Elem<T>::mma(TL::row(lds + kTile, row_base, 32 * u, kc), load_frag<T>(drow, few, kc, half, a.D), dp);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      if (32 * u + 4 * half + 8 * (r >> 2) + (r & 3) < few)
        delta = few == 1 ? dp[r] : fmaf(__builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -ls)), dp[r], delta);      // (one key: no gradient, not its rounding's)
  }
  delta += __shfl_xor(delta, 32, 64);
  if (few && half == 0) a.delta[at] = delta;
}

// delta_i = do_i . o_i of the other rows: L lanes per row, 16 bytes of each tensor at a time; 8 where that is a row of 64 16-bit elements, 16
// otherwise.  FEW: the first workgroups do the rows of few keys; 0 where none can have few.
// Bound by memory: 2 x 4096 rows of 16 heads of 128, bf16, 67 MB each of o and do in 13 us, 15.8 with the rows of few keys (10.3 and 8.5
// TB/s: what the forward pass wrote is in the last-level cache).
template <typename T, int DP, int L, bool FEW>
__global__ void __launch_bounds__(256, FEW ? 4 : 0) attn_delta_kernel(AttnArgs a) {
  extern __shared__ __align__(16) char lds[];
  unsigned block = blockIdx.x;
  if constexpr (FEW) {
    const unsigned few_blocks = a.few_tiles * a.B * a.Hk;
    if (block < few_blocks) return attn_few_keys<T, DP>(a, block, lds);
    block -= few_blocks;
  }
  constexpr int kPer = 16 / (int)sizeof(T);
  constexpr bool kNorms = kScaled<T>;
  constexpr unsigned kRows = 256 / L;
  const int c = threadIdx.x % L;
  if constexpr (kNorms) {
    const unsigned do_blocks = (a.B * a.Lq * a.Hq + kRows - 1) / kRows, v_rows = a.B * a.Lk * a.Hk;
    if (block >= do_blocks) {                              // rows (b, j, h) of v
      const unsigned v_blocks = gridDim.x - (blockIdx.x - block) - do_blocks;
      for (unsigned u = (block - do_blocks) * kRows + threadIdx.x / L; u < v_rows; u += v_blocks * kRows) {
        const unsigned uh = u / a.Hk;
        const int h = u - uh * a.Hk, b = uh / a.Lk, j = uh - b * a.Lk;
        float s = 0.0f;
        if (j < clamp_len(a.k_lens, b, a.Lk)) {
          const T *v = (const T *)a.v.p + (long long)b * a.v.b + (long long)j * a.v.r + (long long)h * a.v.h;
          typedef T TV __attribute__((ext_vector_type(kPer)));
          for (int e = c * kPer; e < a.D; e += L * kPer) {
            const TV x = *(const TV *)(v + e);
#pragma unroll
            for (int n = 0; n < kPer; ++n) s = fmaf((float)x[n], (float)x[n], s);
          }
        }
#pragma unroll
        for (int x = L / 2; x >= 1; x >>= 1) s += __shfl_xor(s, x, L);
        if (c == 0) a.norm_v[((long long)b * a.Hk + h) * a.Lk + j] = sqrtf(s);
      }
      return;
    }
  }
  const unsigned u = block * kRows + threadIdx.x / L;
  const unsigned uh = u / a.Hq;                            // row (b, i, h), (b, i)
  const bool inside = u < (unsigned)(a.B * a.Lq * a.Hq);
  const int h = u - uh * a.Hq, b = inside ? uh / a.Lq : 0, i = uh - b * a.Lq;
  float s = 0.0f, ss = 0.0f;
  if (inside && i < clamp_len(a.q_lens, b, a.Lq)) {
    const T *o = (const T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)h * a.o.h;
    const T *d = (const T *)a.dout.p + (long long)b * a.dout.b + (long long)i * a.dout.r + (long long)h * a.dout.h;
    typedef T TV __attribute__((ext_vector_type(kPer)));
    for (int e = c * kPer; e < a.D; e += L * kPer) {
      const TV x = *(const TV *)(o + e), y = *(const TV *)(d + e);
#pragma unroll
      for (int n = 0; n < kPer; ++n) {
        s = fmaf((float)x[n], (float)y[n], s);
        if (kNorms) ss = fmaf((float)y[n], (float)y[n], ss);
      }
    }
  }
#pragma unroll
  for (int x = L / 2; x >= 1; x >>= 1) {
    s += __shfl_xor(s, x, L);
    if (kNorms) ss += __shfl_xor(ss, x, L);
  }
  if (inside && c == 0) {
    if (!FEW || !few_keys(i, clamp_len(a.q_lens, b, a.Lq), clamp_len(a.k_lens, b, a.Lk), a.causal)) a.delta[((long long)b * a.Hq + h) * a.Lq + i] = s;
    if (kNorms) a.norm_do[((long long)b * a.Hq + h) * a.Lq + i] = sqrtf(ss);
  }
}

// Tiles of 64 rows (keys) where the registers allow it: half the barriers, and the second half's products run beside the first
// half's exponentials (16 x 4 heads of 1024 x 1024 x 64, bf16: 84 us with 32 rows, 79 with 64; longer heads have no registers for it).
template <typename T, int DP> constexpr int kBackwardSub = sizeof(T) == 2 && DP <= 64 ? 2 : 1;

// dk and dv of 128 keys, 32 per wave.  k stays in registers, v in LDS: with both in registers the accumulators leave room for one
// wave per SIMD only, and nothing runs beside its waits.  The query rows, cut in `splits` ranges of whole tiles, are walked
// from the last one down, range by range over all key tiles: the workgroups that run together read the same rows at about the same
// time, and the first of them brings a row into the XCD's L2 for the others, causal or not.
template <typename T, int DP> __device__ __forceinline__ void attn_backward_kv(const AttnArgs &a, int id, char *lds) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  constexpr int kSub = kBackwardSub<T, DP>, kRows = 32 * kSub, kKc = DP / 16, kDt = DP / 32;
  constexpr int kTile = kRows * TL::kBytes, kBuffer = 2 * kTile + 512;         // q, do, lse (log2 units) and delta of the rows; two buffers
  char *const vt = lds + 2 * kBuffer;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const unsigned row_base = TL::row_base(col, half), v_base = row_base + 32 * wave * TL::kBytes;
  const typename TL::ColBase col_base = TL::col_base(lane);
  int tile, group;
  xcd_group_map(id, a.kv_tiles * a.kv_splits, a.B * a.Hk, tile, group);
  const int split = tile / a.kv_tiles;                                           // 0: the last rows
  tile -= split * a.kv_tiles;
  const int b = group / a.Hk, hk = group % a.Hk;
  const int nq = clamp_len(a.q_lens, b, a.Lq), nk = clamp_len(a.k_lens, b, a.Lk);
  const int key = tile * 128 + 32 * wave + col;
  // rows [begin, rows) see some key of the workgroup; causal: key j is seen by i >= j - (nk - nq), which is row >= first_row, and
  // from row `diagonal` on every row sees every key
  int rows = tile * 128 < nk ? nq * a.G : 0;
  const int first_row = a.causal ? min(nq, max(0, key - (nk - nq))) * a.G : 0;
  const int i_min = a.causal ? min(nq, max(0, tile * 128 - (nk - nq))) : 0, diagonal = a.causal ? min(nq, max(0, tile * 128 + 127 - (nk - nq))) * a.G : 0;
  const int low = a.causal ? max(0, nq - nk) * a.G : 0;      // rows below it see no key at all: as if they were not there
  int begin = min(i_min * a.G, rows) / kRows * kRows;
  {
    const int t = (nq * a.G + kRows - 1) / kRows, per = (t + a.kv_splits - 1) / a.kv_splits * kRows, from = (t * kRows) - (split + 1) * per;
    begin = max(begin, from);
    rows = min(rows, from + per);
  }
  f32x16 dk[kDt], dv[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) dk[dt] = dv[dt] = f32x16{};
  float factor = 1.0f;                    // f16: of ds, beside the probabilities'
  if (begin < rows) {
    if constexpr (kScaled<T>) {
      float most_do = 0.0f, most_delta = 0.0f, most_v = 0.0f;
      const int i0 = max(begin, low) / a.G, i1 = (rows + a.G - 1) / a.G;
      for (int g = 0; g < a.G; ++g) {
        const long long at = ((long long)b * a.Hq + hk * a.G + g) * a.Lq;
        for (int i = i0 + tid; i < i1; i += 256) {
          most_do = finite_max(most_do, a.norm_do[at + i]);
          most_delta = finite_max(most_delta, fabsf(a.delta[at + i]));
        }
      }
      if (tid < 128 && tile * 128 + tid < nk) most_v = finite_max(0.0f, a.norm_v[((long long)b * a.Hk + hk) * a.Lk + tile * 128 + tid]);
      most_do = block_max(most_do, (float *)lds);
      most_delta = block_max(most_delta, (float *)lds);
      most_v = block_max(most_v, (float *)lds);
      lds_barrier();
      factor = ldexpf(1.0f, grad_shift(most_do * most_v + most_delta) - kProbShift);
    }
    const T *krow = (const T *)a.k.p + (long long)b * a.k.b + (long long)key * a.k.r + (long long)hk * a.k.h;
    Frag k[kKc];
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc) k[kc] = load_frag<T>(krow, key < nk, kc, half, a.D);
    {
      Stage<T, DP, 32> vs;
      vs.start((const T *)a.v.p + (long long)b * a.v.b + (long long)hk * a.v.h, a.v.r, 0, 1, tile * 128, a.D, tid);
      for (int n = 0; n < 4; ++n) {
        vs.load(nk);
        vs.store(vt + n * 32 * TL::kBytes, tid);
      }
    }
    int r0 = (rows - 1) / kRows * kRows;
    Stage<T, DP, kRows> qs, ds;
    qs.start((const T *)a.q.p + (long long)b * a.q.b + (long long)hk * a.G * a.q.h, a.q.r, a.q.h, a.G, r0, a.D, tid, low);
    ds.start((const T *)a.dout.p + (long long)b * a.dout.b + (long long)hk * a.G * a.dout.h, a.dout.r, a.dout.h, a.G, r0, a.D, tid, low);
    // threads 0 .. kRows - 1 carry the rows' lse, the next kRows their delta
    int stat_row = r0 + (tid & (kRows - 1)), stat_i = stat_row / a.G, stat_g = stat_row - stat_i * a.G;
    const float *stat = (tid < kRows ? a.lse : a.delta) + ((long long)b * a.Hq + hk * a.G) * a.Lq;
    float stat_next = 0.0f;
    auto load = [&]() {
      qs.template load<true>(max(0, rows - low));
      ds.template load<true>(max(0, rows - low));
      if (tid < 2 * kRows) {
        // no such row, or one that sees nothing: probabilities 0
        stat_next = tid < kRows ? INFINITY : 0.0f;
        if (stat_row < rows && stat_row >= low) {
          const float x = stat[(long long)stat_g * a.Lq + stat_i];
          stat_next = tid < kRows ? (x == -INFINITY ? INFINITY : x * kLog2e - (kScaled<T> ? kProbShift : 0)) : kScaled<T> ? x * factor : x;
        }
        stat_row -= kRows;
        stat_i -= kRows / a.G;
        stat_g -= kRows % a.G;
        if (stat_g < 0) { stat_g += a.G; --stat_i; }
      }
    };
    auto store = [&](char *to) {
      qs.store(to, tid);
      ds.store(to + kTile, tid);
      if (tid < 2 * kRows) ((float *)(to + 2 * kTile))[tid] = stat_next;
    };
    load();
    store(lds);
    int buffer = 0;
    for (; r0 >= begin; r0 -= kRows) {
      lds_barrier();                      // this tile is written, the other buffer has been read
      const unsigned at = buffer * kBuffer;
      const bool more = r0 > begin;
      if (more) load();
      f32x16 s[kSub], dp[kSub];
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        s[u] = dp[u] = f32x16{};
#pragma unroll
        for (int kc = 0; kc < kKc; ++kc) {
          s[u] = Elem<T>::mma(TL::row(lds, row_base + at, 32 * u, kc), k[kc], s[u]);
          dp[u] = Elem<T>::mma(TL::row(lds + kTile, row_base + at, 32 * u, kc), TL::row(vt, v_base, 0, kc), dp[u]);
        }
      }
      if (r0 < diagonal) {                // causal: some row of the tile does not see some key of the workgroup
        stay_a_branch();
        const int low = first_row - r0 - 4 * half;
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * u + 8 * (r >> 2) + (r & 3) < low) s[u][r] = -INFINITY;
      }
      const float *lt = (const float *)(lds + 2 * kTile + at) + 4 * half;
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 ls = *(const f32x4 *)(lt + 32 * u + 8 * r4), de = *(const f32x4 *)(lt + kRows + 32 * u + 8 * r4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * r4 + e;
            s[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], a.scale2, -ls[e]));
            dp[u][r] = s[u][r] * (kScaled<T> ? fmaf(dp[u][r], factor, -de[e]) : dp[u][r] - de[e]);
          }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const Frag p = to_frag<T>(s[u], t), d = to_frag<T>(dp[u], t);
#pragma unroll
          for (int dt = 0; dt < kDt; ++dt) {
            dv[dt] = Elem<T>::mma(TL::column(lds + kTile, col_base + at, 32 * u + 16 * t, dt), p, dv[dt]);
            dk[dt] = Elem<T>::mma(TL::column(lds, col_base + at, 32 * u + 16 * t, dt), d, dk[dt]);
          }
        }
      }
      buffer ^= 1;
      if (more) store(lds + buffer * kBuffer);
    }
  }
  if (key >= a.Lk) return;
  const bool used = key < nk;             // behind the sequence's end a column held no key
  const float of_dk = kScaled<T> ? a.scale * (kDvScale<T> / factor) : a.scale, of_dv = kDvScale<T>;
  if (a.kv_splits > 1) {
    const long long at = ((long long)split * a.B * a.Hk + group) * a.Lk + key, other = (long long)a.kv_splits * a.B * a.Hk * a.Lk * DP;
    store_rows<float, DP>(a.part_kv + at * DP, dk, of_dk, used, DP, half);
    store_rows<float, DP>(a.part_kv + other + at * DP, dv, of_dv, used, DP, half);
  } else {
    store_rows<T, DP>((T *)a.dk.p + (long long)b * a.dk.b + (long long)key * a.dk.r + (long long)hk * a.dk.h, dk, of_dk, used, a.D, half);
    store_rows<T, DP>((T *)a.dv.p + (long long)b * a.dv.b + (long long)key * a.dv.r + (long long)hk * a.dv.h, dv, of_dv, used, a.D, half);
  }
}

// dq of 128 rows, 32 per wave, whose q and do rows stay in registers; walks the keys (or one of `splits` ranges).
template <typename T, int DP> __device__ __forceinline__ void attn_backward_q(const AttnArgs &a, int id, char *lds) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  constexpr int kSub = kBackwardSub<T, DP>, kKeys = 32 * kSub, kKc = DP / 16, kDt = DP / 32;
  constexpr int kTile = kKeys * TL::kBytes;                // k, then v; two buffers
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  const unsigned row_base = TL::row_base(col, half);
  const typename TL::ColBase col_base = TL::col_base(lane);
  int tile, group;
  xcd_group_map(id, a.q_tiles * a.q_splits, a.B * a.Hk, tile, group);
  const int split = tile % a.q_splits;
  tile = a.q_tiles - 1 - tile / a.q_splits;
  const int b = group / a.Hk, hk = group % a.Hk;
  const int nq = clamp_len(a.q_lens, b, a.Lq), nk = clamp_len(a.k_lens, b, a.Lk);
  const int row = tile * 128 + 32 * wave + col, i = row / a.G, g = row - i * a.G;
  const bool inside = row < a.Lq * a.G;
  const int seen = i >= nq ? 0 : a.causal ? min(nk, max(0, i + 1 + nk - nq)) : nk;
  const bool active = seen > 0;
  const int i_last = min(nq, (min((tile + 1) * 128, a.Lq * a.G) - 1) / a.G + 1) - 1, i_first = tile * 128 / a.G;
  int block_end = i_first >= nq ? 0 : a.causal ? min(nk, max(0, i_last + 1 + nk - nq)) : nk;
  const int full_end = a.causal ? min(nk, max(0, i_first + 1 + nk - nq)) : nk;
  int begin = 0;
  {
    const int n = (block_end + kKeys - 1) / kKeys, per = (n + a.q_splits - 1) / a.q_splits;
    begin = min(block_end, split * per * kKeys);
    block_end = min(block_end, begin + per * kKeys);
  }
  const int h = hk * a.G + g;
  const T *qrow = (const T *)a.q.p + (long long)b * a.q.b + (long long)i * a.q.r + (long long)h * a.q.h;
  const T *drow = (const T *)a.dout.p + (long long)b * a.dout.b + (long long)i * a.dout.r + (long long)h * a.dout.h;
  const T *kh = (const T *)a.k.p + (long long)b * a.k.b + (long long)hk * a.k.h;
  const T *vh = (const T *)a.v.p + (long long)b * a.v.b + (long long)hk * a.v.h;
  Frag q[kKc], d[kKc];
#pragma unroll
  for (int kc = 0; kc < kKc; ++kc) { q[kc] = load_frag<T>(qrow, active, kc, half, a.D); d[kc] = load_frag<T>(drow, active, kc, half, a.D); }
  const long long at = ((long long)b * a.Hq + h) * a.Lq + i;
  // a row that sees nothing: probabilities 0
  const float lse = active ? a.lse[at] : -INFINITY, ls = lse == -INFINITY ? INFINITY : lse * kLog2e, de = active ? a.delta[at] : 0.0f;
  float up = 0.0f;                        // f16: ds is taken times 2^up
  if constexpr (kScaled<T>) {
    float most_v = 0.0f;
    const float *norm_v = a.norm_v + ((long long)b * a.Hk + hk) * a.Lk;
    for (int j = begin + tid; j < block_end; j += 256) most_v = finite_max(most_v, norm_v[j]);
    most_v = block_max(most_v, (float *)lds);
    lds_barrier();
    if (active) up = grad_shift(finite_max(0.0f, a.norm_do[at]) * most_v + finite_max(0.0f, fabsf(de)));
  }
  f32x16 dq[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) dq[dt] = f32x16{};
  Stage<T, DP, kKeys> ks, vs;
  ks.start(kh, a.k.r, 0, 1, begin, a.D, tid);
  vs.start(vh, a.v.r, 0, 1, begin, a.D, tid);
  ks.load(block_end);
  vs.load(block_end);
  ks.store(lds, tid);
  vs.store(lds + kTile, tid);
  int buffer = 0;
  for (int key0 = begin; key0 < block_end; key0 += kKeys) {
    lds_barrier();
    const unsigned at = buffer * 2 * kTile;
    const bool more = key0 + kKeys < block_end;
    if (more) {
      ks.load(block_end);
      vs.load(block_end);
    }
    f32x16 s[kSub], dp[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      s[u] = dp[u] = f32x16{};
#pragma unroll
      for (int kc = 0; kc < kKc; ++kc) {
        s[u] = Elem<T>::mma(TL::row(lds, row_base + at, 32 * u, kc), q[kc], s[u]);
        dp[u] = Elem<T>::mma(TL::row(lds + kTile, row_base + at, 32 * u, kc), d[kc], dp[u]);
      }
    }
    if (key0 + kKeys > min(full_end, block_end)) {
      stay_a_branch();
      const int end = min(seen, block_end) - key0 - 4 * half;
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * u + 8 * (r >> 2) + (r & 3) >= end) s[u][r] = -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[u][r] = __builtin_amdgcn_exp2f(fmaf(s[u][r], a.scale2, up - ls)) * (dp[u][r] - de);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag x = to_frag<T>(dp[u], t);
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) dq[dt] = Elem<T>::mma(TL::column(lds, col_base + at, 32 * u + 16 * t, dt), x, dq[dt]);
      }
    }
    buffer ^= 1;
    if (more) {
      ks.store(lds + buffer * 2 * kTile, tid);
      vs.store(lds + buffer * 2 * kTile + kTile, tid);
    }
  }
  if (!inside) return;
  const float of_dq = kScaled<T> ? ldexpf(a.scale, -(int)up) : a.scale;
  if (a.q_splits > 1)
    store_rows<float, DP>(a.part_q + (((long long)split * a.B * a.Hk + group) * ((long long)a.Lq * a.G) + row) * DP, dq, of_dq, active, DP, half);
  else
    store_rows<T, DP>((T *)a.dq.p + (long long)b * a.dq.b + (long long)i * a.dq.r + (long long)h * a.dq.h, dq, of_dq, active, a.D, half);
}

// Both in one launch: the first workgroups make dk and dv, the others dq, so that neither leaves CUs idle at its end.  Seven products of
// rows x keys where five are necessary (the scores and do . v twice): dq made by the first workgroups too would need atomics or its
// partial sums in memory, one for every 128 keys.
// Bound: matrix instructions, exponentials and LDS reads in turn, two waves per SIMD (2 x 16 heads of 4096 x 4096 x 128, causal, bf16: 481
// GFLOP executed in 553 us, 870 TFLOP/s; 16 x 4 heads of 1024 x 1024 x 64: 590; fp32, 4 x 4 heads of 1000 x 1000 x 64: 14.3 GFLOP in 126 us, 114 of 153).
template <typename T, int DP>
__global__ void __launch_bounds__(256, (kBlocksPerCu<T, DP>)) attn_backward_kernel(AttnArgs a) {
  extern __shared__ __align__(16) char lds[];
  const int kv_blocks = a.kv_tiles * a.kv_splits * a.B * a.Hk;
  if ((int)blockIdx.x < kv_blocks) attn_backward_kv<T, DP>(a, blockIdx.x, lds);
  else attn_backward_q<T, DP>(a, blockIdx.x - kv_blocks, lds);
}

// The gradients that were made in parts: the sums of the parts, in their order.  Four elements a thread, over the rows of dk and dv
// (group, key) and of dq (group, row = i * G + g) as far as they have parts.  Bound by memory.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_sum_kernel(AttnArgs a) {
  const long long u = (long long)blockIdx.x * 256 + threadIdx.x;
  long long r = u / (DP / 4);
  const int d = (int)(u - r * (DP / 4)) * 4, groups = a.B * a.Hk;
  const long long kv_rows = a.kv_splits > 1 ? (long long)groups * a.Lk : 0, q_rows = a.q_splits > 1 ? (long long)groups * a.Lq * a.G : 0;
  if (r >= 2 * kv_rows + q_rows || d >= a.D) return;
  const bool is_q = r >= 2 * kv_rows, is_v = !is_q && r >= kv_rows;
  const float *part = is_q ? a.part_q : a.part_kv + (is_v ? a.kv_splits * kv_rows * DP : 0);
  const AttnView out = is_q ? a.dq : is_v ? a.dv : a.dk;
  const long long all = is_q ? q_rows : kv_rows;
  const int splits = is_q ? a.q_splits : a.kv_splits, rows = is_q ? a.Lq * a.G : a.Lk, per_i = is_q ? a.G : 1;
  r -= is_q ? 2 * kv_rows : is_v ? kv_rows : 0;
  f32x4 s = *(const f32x4 *)(part + r * DP + d);
  for (int n = 1; n < splits; n += 3) {        // three loads in flight (8.4 million sums of three parts: 19.7 -> 18.4 us)
    f32x4 x[3];
#pragma unroll
    for (int e = 0; e < 3; ++e) x[e] = *(const f32x4 *)(part + (min(n + e, splits - 1) * all + r) * DP + d);
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (n + e < splits) s += x[e];
  }
  const int group = (unsigned)r / (unsigned)rows, row = (int)r - group * rows, b = group / a.Hk, hk = group % a.Hk, i = row / per_i, g = row - i * per_i;
  store4<T>((T *)out.p + (long long)b * out.b + (long long)i * out.r + (long long)(hk * per_i + g) * out.h + d, s[0], s[1], s[2], s[3]);
}

// ------------------------------------------------------------------ launches
// dynamic LDS above 64 KiB has to be allowed once per kernel and device
inline hipError_t allow_lds(DeviceOnce &once, const void *kernel, int bytes) {
  if (bytes <= 64 * 1024 || !once.need()) return hipSuccess;
  const hipError_t rc = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (rc == hipSuccess) once.mark();
  return rc;
}

template <typename T, int DP> hipError_t attn_forward_dp(AttnArgs a, int narrow, hipStream_t st) {
  const int rows = a.Lq * a.G, kRows = narrow ? 32 : 128, kKeys = narrow ? 128 : 64;
  a.tiles = (rows + kRows - 1) / kRows;
  const int tile_bytes = (narrow ? 2 : 4) * kKeys * Tile<T, DP>::kBytes, join_bytes = narrow ? (4 * 32 * 2 + 4 * 32 * DP) * 4 : 0;
  const int lds = tile_bytes > join_bytes ? tile_bytes : join_bytes;
  const unsigned grid = (unsigned)a.tiles * a.splits * a.B * a.Hk;
  auto kernel = narrow ? attn_forward_kernel<T, DP, 1> : attn_forward_kernel<T, DP, 0>;
  static DeviceOnce once[2];
  hipError_t rc = allow_lds(once[narrow], (const void *)kernel, lds);
  if (rc != hipSuccess) return rc;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), lds, st, a);
  rc = hipGetLastError();
  if (rc != hipSuccess || a.splits == 1) return rc;
  const long long waves = (long long)a.B * a.Hk * rows;
  hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T, int DP> hipError_t attn_backward_dp(AttnArgs a, hipStream_t st) {
  const long long rows = (long long)a.B * a.Lq * a.Hq, v_rows = kScaled<T> ? (long long)a.B * a.Lk * a.Hk : 0;
  constexpr int kLanes = DP * sizeof(T) <= 128 ? 8 : 16, kPerBlock = 256 / kLanes;
  const long long v_blocks = std::min((v_rows + kPerBlock - 1) / kPerBlock, 1ll << 22);
  constexpr int kBytes = Tile<T, DP>::kBytes;
  // rows of few keys: none unless the keys are few, a length that only the device knows may be, or a causal call begins with few
  const long long begin = (long long)a.Lk - a.Lq + 1;      // causal, all in use: the keys of row 0
  const bool unknown = a.k_lens || (a.causal && a.q_lens);
  const long long few_rows = sizeof(T) == 4 || a.Lk == 0 ? 0 : unknown || a.Lk <= kFewKeys ? a.Lq
                           : a.causal && begin <= kFewKeys ? std::min<long long>(a.Lq, kFewKeys + 1 - begin) : 0;
  a.few_tiles = (int)((few_rows * a.G + 127) / 128);
  const unsigned delta_grid = (unsigned)((long long)a.few_tiles * a.B * a.Hk + (rows + kPerBlock - 1) / kPerBlock + v_blocks);
  if constexpr (sizeof(T) == 2) {
    if (a.few_tiles) hipLaunchKernelGGL((attn_delta_kernel<T, DP, kLanes, true>), dim3(delta_grid), dim3(256), 2 * kFewKeys * kBytes, st, a);
  }
  if (!a.few_tiles) hipLaunchKernelGGL((attn_delta_kernel<T, DP, kLanes, false>), dim3(delta_grid), dim3(256), 0, st, a);
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  static DeviceOnce once;
  const int lds = 128 * kBytes + 4 * 32 * kBackwardSub<T, DP> * kBytes + 1024;
  rc = allow_lds(once, (const void *)attn_backward_kernel<T, DP>, lds);
  if (rc != hipSuccess) return rc;
  a.kv_tiles = (a.Lk + 127) / 128;
  a.q_tiles = (a.Lq * a.G + 127) / 128;
  const unsigned grid = (unsigned)(a.kv_tiles * a.kv_splits + a.q_tiles * a.q_splits) * a.B * a.Hk;
  hipLaunchKernelGGL((attn_backward_kernel<T, DP>), dim3(grid), dim3(256), lds, st, a);
  rc = hipGetLastError();
  const long long sums = (long long)a.B * a.Hk * ((a.kv_splits > 1 ? 2ll * a.Lk : 0) + (a.q_splits > 1 ? (long long)a.Lq * a.G : 0)) * (DP / 4);
  if (rc != hipSuccess || sums == 0) return rc;
  hipLaunchKernelGGL((attn_sum_kernel<T, DP>), dim3((unsigned)((sums + 255) / 256)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T> hipError_t attn_forward_t(const AttnArgs &a, int narrow, hipStream_t st) {
  return a.D <= 32 ? attn_forward_dp<T, 32>(a, narrow, st) : a.D <= 64 ? attn_forward_dp<T, 64>(a, narrow, st)
       : a.D <= 96 ? attn_forward_dp<T, 96>(a, narrow, st) : attn_forward_dp<T, 128>(a, narrow, st);
}
template <typename T> hipError_t attn_backward_t(const AttnArgs &a, hipStream_t st) {
  return a.D <= 32 ? attn_backward_dp<T, 32>(a, st) : a.D <= 64 ? attn_backward_dp<T, 64>(a, st)
       : a.D <= 96 ? attn_backward_dp<T, 96>(a, st) : attn_backward_dp<T, 128>(a, st);
}

}  // namespace urf
