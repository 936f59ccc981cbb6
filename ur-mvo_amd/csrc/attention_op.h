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

namespace urf {

struct AttnView { void *p; long long b, r, h; };   // base, strides in elements: batch, row, head

struct AttnArgs {
  AttnView q, k, v, o, dout, dq, dk, dv;
  const int *q_lens, *k_lens;    // rows in use per sequence (null = all)
  float *lse;                    // [B][Hq][Lq], natural logarithm
  float *delta;                  // [B][Hq][Lq] (backward)
  float *part_o, *part_ml;       // forward over split keys: [split][B * Hk][rows padded to 32][DP] and (maximum, sum)
  int B, Hq, Hk, G, Lq, Lk, D;
  int causal;
  int splits;                    // key ranges of the forward kernel
  int tiles;                     // row (key) tiles per (sequence, key head)
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
// A tile is rows x DP elements, row r's 16-byte chunk c at chunk position c ^ swizzle(r).  16-bit types: eight consecutive
// lanes of a row-wise fragment read (eight rows, one chunk) and the half wave of a transposed read (four rows, four chunks)
// each fall into distinct banks.
template <typename T, int DP> struct Tile {
  static constexpr int kPer = 16 / (int)sizeof(T);          // elements of a chunk
  static constexpr int kChunks = DP / kPer;
  static constexpr int kBytes = DP * (int)sizeof(T);        // of a row
  static __device__ __forceinline__ int swizzle(int r) {
    if constexpr (sizeof(T) == 4) return (((r >> 2) & 1) << 3) | ((r & 3) << 1);
    else if constexpr (kBytes == 256) return ((r & 3) << 2) | ((r >> 2) & 3);
    else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  }
  static __device__ __forceinline__ const char *at(const char *tile, int r, int c) { return tile + r * kBytes + ((c ^ swizzle(r)) << 4); }
  static __device__ __forceinline__ char *at(char *tile, int r, int c) { return tile + r * kBytes + ((c ^ swizzle(r)) << 4); }
  // elements 16 kc + 8 half .. + 7 of row r
  static __device__ __forceinline__ typename Elem<T>::Frag row(const char *tile, int r, int kc, int half) {
    if constexpr (sizeof(T) == 2) {
      return *(const typename Elem<T>::Frag *)at(tile, r, 2 * kc + half);
    } else {
      const f32x4 a = *(const f32x4 *)at(tile, r, 4 * kc + 2 * half), b = *(const f32x4 *)at(tile, r, 4 * kc + 2 * half + 1);
      f32x8 f;
#pragma unroll
      for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
      return f;
    }
  }
  // column 32 dt + l % 32 of rows r0 + 16 t + {4 half + 0..3, 8 + 4 half + 0..3}: the left operand of a product over rows
  static __device__ __forceinline__ typename Elem<T>::Frag column(const char *tile, int r0, int dt, int lane) {
    const int half = lane >> 5;
    typename Elem<T>::Frag f;
    if constexpr (sizeof(T) == 2) {
      // the 16 lanes of a group read four rows of 16 elements, four elements a lane, and get one column of four rows each
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 lds4;
      const int i = lane & 15, r = r0 + 4 * half + (i >> 2), c = 4 * dt + 2 * ((lane >> 4) & 1) + ((i >> 1) & 1);
      const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(at(tile, r, c) + 8 * (i & 1)));
      const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4 *)(at(tile, r + 8, c) + 8 * (i & 1)));
      typedef T T4 __attribute__((ext_vector_type(4)));
      const T4 x = __builtin_bit_cast(T4, a), y = __builtin_bit_cast(T4, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) { f[e] = x[e]; f[4 + e] = y[e]; }
    } else {
      const int d = 32 * dt + (lane & 31);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int r = r0 + 8 * (e >> 2) + 4 * half + (e & 3);
        f[e] = *(const float *)(at(tile, r, d >> 2) + 4 * (d & 3));
      }
    }
    return f;
  }
};

// Copies R rows (from `first`, valid below `end`) of one head into a tile: chunks beyond the head size and rows at or behind
// `end` become zero -- what lies behind a sequence's end may be anything, NaN included, and never enters a product.
// `group` > 1 walks (i, g) rows of a query tensor.  Two halves: the loads into registers, and the LDS writes.
template <typename T, int DP, int R> struct Stage {
  typedef Tile<T, DP> TL;
  static constexpr int kN = R * TL::kChunks / 256;
  u32x4 x[kN];
  __device__ __forceinline__ void load(const T *head, long long srow, long long shead, int group, int first, int end, int D, int tid) {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int u = tid + 256 * n, r = first + u / TL::kChunks, c = u % TL::kChunks;
      x[n] = u32x4{0, 0, 0, 0};
      if (r < end && c * TL::kPer < D) {
        const int i = group == 1 ? r : r / group, g = group == 1 ? 0 : r - i * group;
        x[n] = *(const u32x4 *)(head + (long long)i * srow + (long long)g * shead + c * TL::kPer);
      }
    }
  }
  __device__ __forceinline__ void store(char *tile, int tid) const {
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const int u = tid + 256 * n;
      *(u32x4 *)TL::at(tile, u / TL::kChunks, u % TL::kChunks) = x[n];
    }
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

__device__ __forceinline__ int clamp_len(const int *lens, int b, int most) {
  return lens ? min(max(lens[b], 0), most) : most;      // lengths come from device memory: never trusted beyond the tensor
}

// ------------------------------------------------------------------ forward
// One workgroup: SPLIT = 0: 128 rows, 32 per wave, over tiles of 64 keys; SPLIT = 1: 32 rows, each of the four waves a quarter of
// a 128-key tile, joined through LDS at the end (few rows: more workgroups, more loads in flight).  The key range may be cut in
// `splits` parts, joined by attn_join_kernel.
template <typename T, int DP, int SPLIT>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) attn_forward_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  constexpr int kKeys = SPLIT ? 128 : 64, kRows = SPLIT ? 32 : 128, kKc = DP / 16, kDt = DP / 32, kSub = SPLIT ? 1 : 2;
  extern __shared__ __align__(16) char lds[];
  char *kt = lds, *vt = lds + kKeys * TL::kBytes;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
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
  float m = -INFINITY, l = 0.0f;          // running maximum (log2 units) and this half wave's share of the sum
  Stage<T, DP, kKeys> ks, vs;
  ks.load(kh, a.k.r, 0, 1, begin, min(nk, block_end), a.D, tid);
  vs.load(vh, a.v.r, 0, 1, begin, min(nk, block_end), a.D, tid);
  for (int key0 = begin; key0 < block_end; key0 += kKeys) {
    lds_barrier();                        // the previous tile has been read
    ks.store(kt, tid);
    vs.store(vt, tid);
    lds_barrier();
    if (key0 + kKeys < block_end) {
      ks.load(kh, a.k.r, 0, 1, key0 + kKeys, min(nk, block_end), a.D, tid);
      vs.load(vh, a.v.r, 0, 1, key0 + kKeys, min(nk, block_end), a.D, tid);
    }
    f32x16 s[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      s[u] = f32x16{};
      const int r0 = SPLIT ? 32 * wave : 32 * u;
#pragma unroll
      for (int kc = 0; kc < kKc; ++kc) s[u] = Elem<T>::mma(TL::row(kt, r0 + col, kc, half), q[kc], s[u]);
    }
    const bool edge = key0 + kKeys > min(full_end, block_end) || !all_active;
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      const int k0 = key0 + (SPLIT ? 32 * wave : 32 * u) + 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] *= a.scale2;
        if (edge && k0 + 8 * (r >> 2) + (r & 3) >= min(seen, block_end)) s[u][r] = -INFINITY;
        top = fmaxf(top, s[u][r]);
      }
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mn = fmaxf(m, top), mu = mn == -INFINITY ? 0.0f : mn;      // nothing visible yet: all the exponentials are 0
    const float alpha = exp2f(m - mu);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = __builtin_amdgcn_exp2f(s[u][r] - mu);
        sum += s[u][r];
      }
    l = l * alpha + sum;
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt) acc[dt] *= alpha;
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Frag p = to_frag<T>(s[u], t);
        const int r0 = (SPLIT ? 32 * wave : 32 * u) + 16 * t;
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) acc[dt] = Elem<T>::mma(TL::column(vt, r0, dt, lane), p, acc[dt]);
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
    if (a.splits > 1) {
      const long long prow = ((long long)split * a.B * a.Hk + group) * (a.tiles * 32) + row;
#pragma unroll
      for (int e = 0; e < kOwn; ++e) a.part_o[prow * DP + d0 + e] = ov[e];
      if (wave == 0 && half == 0) { a.part_ml[prow * 2] = m; a.part_ml[prow * 2 + 1] = l; }
    } else if (inside) {
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      T *orow = (T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)(hk * a.G + g) * a.o.h;
#pragma unroll
      for (int e = 0; e < kOwn; e += 4)
        if (d0 + e < a.D) store4<T>(orow + d0 + e, ov[e] * inv, ov[e + 1] * inv, ov[e + 2] * inv, ov[e + 3] * inv);
      if (wave == 0 && half == 0) a.lse[((long long)b * a.Hq + hk * a.G + g) * a.Lq + i] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
    }
  } else if (inside) {
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    T *orow = (T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)(hk * a.G + g) * a.o.h;
#pragma unroll
    for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * dt + 2 * r + 4 * half;
        if (d < a.D) store4<T>(orow + d, acc[dt][r] * inv, acc[dt][r + 1] * inv, acc[dt][r + 2] * inv, acc[dt][r + 3] * inv);
      }
    if (half == 0) a.lse[((long long)b * a.Hq + hk * a.G + g) * a.Lq + i] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
  }
}

// Joins the key ranges: a wave per row, a lane for two columns; fixed order over the ranges.
template <typename T, int DP>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnArgs a) {
  const int lane = threadIdx.x & 63, rows = a.Lq * a.G;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (long long)a.B * a.Hk * rows) return;
  const int group = (int)(w / rows), row = (int)(w % rows), b = group / a.Hk, hk = group % a.Hk, i = row / a.G, g = row - i * a.G;
  const long long step = (long long)a.B * a.Hk * (a.tiles * 32), base = (long long)group * (a.tiles * 32) + row;
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[(base + s * step) * 2]);
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
  const float mu = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, o[DP / 64];
#pragma unroll
  for (int e = 0; e < DP / 64; ++e) o[e] = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const long long p = base + s * step;
    const float f = exp2f(a.part_ml[p * 2] - mu);
    l += a.part_ml[p * 2 + 1] * f;
#pragma unroll
    for (int e = 0; e < DP / 64; ++e) o[e] += a.part_o[p * DP + lane * (DP / 64) + e] * f;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  T *orow = (T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)(hk * a.G + g) * a.o.h;
#pragma unroll
  for (int e = 0; e < DP / 64; ++e)
    if (lane * (DP / 64) + e < a.D) orow[lane * (DP / 64) + e] = (T)(o[e] * inv);
  if (lane == 0) a.lse[((long long)b * a.Hq + hk * a.G + g) * a.Lq + i] = l > 0.0f ? (m + log2f(l)) * kLn2 : -INFINITY;
}

// ------------------------------------------------------------------ backward
// delta_i = do_i . o_i: sixteen lanes per row
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(AttnArgs a) {
  constexpr int kPer = 16 / (int)sizeof(T);
  const long long u = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);      // row (b, i, h)
  const int c = threadIdx.x & 15;
  const bool inside = u < (long long)a.B * a.Lq * a.Hq;
  const int h = (int)(u % a.Hq), i = (int)(u / a.Hq % a.Lq), b = inside ? (int)(u / a.Hq / a.Lq) : 0;
  float s = 0.0f;
  if (inside && i < clamp_len(a.q_lens, b, a.Lq)) {
    const T *o = (const T *)a.o.p + (long long)b * a.o.b + (long long)i * a.o.r + (long long)h * a.o.h;
    const T *d = (const T *)a.dout.p + (long long)b * a.dout.b + (long long)i * a.dout.r + (long long)h * a.dout.h;
    typedef T TV __attribute__((ext_vector_type(kPer)));
    for (int e = c * kPer; e < a.D; e += 16 * kPer) {
      const TV x = *(const TV *)(o + e), y = *(const TV *)(d + e);
#pragma unroll
      for (int n = 0; n < kPer; ++n) s = fmaf((float)x[n], (float)y[n], s);
    }
  }
#pragma unroll
  for (int x = 8; x >= 1; x >>= 1) s += __shfl_xor(s, x, 16);
  if (inside && c == 0) a.delta[((long long)b * a.Hq + h) * a.Lq + i] = s;
}

// dk and dv of 128 keys, 32 per wave, whose k and v rows stay in registers; walks the query rows in tiles of 32.
template <typename T, int DP>
__global__ void __launch_bounds__(256, 1) attn_backward_kv_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  constexpr int kRows = 32, kKc = DP / 16, kDt = DP / 32;
  extern __shared__ __align__(16) char lds[];
  char *qt = lds, *dt_ = lds + kRows * TL::kBytes;
  float *lt = (float *)(lds + 2 * kRows * TL::kBytes), *et = lt + kRows;      // lse (log2 units) and delta of the rows
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  int tile, group;
  xcd_group_map(blockIdx.x, a.tiles, a.B * a.Hk, tile, group);
  const int b = group / a.Hk, hk = group % a.Hk;
  const int nq = clamp_len(a.q_lens, b, a.Lq), nk = clamp_len(a.k_lens, b, a.Lk);
  const int key = tile * 128 + 32 * wave + col;
  const bool inside = key < a.Lk, active = key < nk;
  const T *qh = (const T *)a.q.p + (long long)b * a.q.b + (long long)hk * a.G * a.q.h;
  const T *dh = (const T *)a.dout.p + (long long)b * a.dout.b + (long long)hk * a.G * a.dout.h;
  const T *krow = (const T *)a.k.p + (long long)b * a.k.b + (long long)key * a.k.r + (long long)hk * a.k.h;
  const T *vrow = (const T *)a.v.p + (long long)b * a.v.b + (long long)key * a.v.r + (long long)hk * a.v.h;
  Frag k[kKc], v[kKc];
#pragma unroll
  for (int kc = 0; kc < kKc; ++kc) { k[kc] = load_frag<T>(krow, active, kc, half, a.D); v[kc] = load_frag<T>(vrow, active, kc, half, a.D); }
  f32x16 dk[kDt], dv[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) dk[dt] = dv[dt] = f32x16{};
  // rows [row_first, rows) see some key of the workgroup; causal: key j is seen by i >= j - (nk - nq)
  const int rows = tile * 128 < nk ? nq * a.G : 0;
  const int i_min = a.causal ? max(0, tile * 128 - (nk - nq)) : 0;
  const int row_first = min((long long)i_min * a.G, (long long)rows) / kRows * kRows;
  Stage<T, DP, kRows> qs, ds;
  float lse_next = 0.0f;
  auto load = [&](int r0) {
    qs.load(qh, a.q.r, a.q.h, a.G, r0, rows, a.D, tid);
    ds.load(dh, a.dout.r, a.dout.h, a.G, r0, rows, a.D, tid);
    if (tid < 2 * kRows) {
      const int r = r0 + (tid & (kRows - 1)), i = r / a.G, g = r - i * a.G;
      lse_next = 0.0f;
      if (r < rows) {
        const long long at = ((long long)b * a.Hq + hk * a.G + g) * a.Lq + i;
        lse_next = tid < kRows ? a.lse[at] * kLog2e : a.delta[at];
      }
    }
  };
  if (row_first < rows) load(row_first);
  for (int r0 = row_first; r0 < rows; r0 += kRows) {
    lds_barrier();
    qs.store(qt, tid);
    ds.store(dt_, tid);
    if (tid < 2 * kRows) lt[tid] = lse_next;
    lds_barrier();
    if (r0 + kRows < rows) load(r0 + kRows);
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc) {
      s = Elem<T>::mma(TL::row(qt, col, kc, half), k[kc], s);
      dp = Elem<T>::mma(TL::row(dt_, col, kc, half), v[kc], dp);
    }
    // some row of the tile does not see some key of the workgroup (or there is no such row)
    const bool edge = r0 + kRows > rows || tile * 128 + 128 > nk || (a.causal && tile * 128 + 127 > r0 / a.G + nk - nq);
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x4 ls = *(const f32x4 *)(lt + 8 * r4 + 4 * half), de = *(const f32x4 *)(et + 8 * r4 + 4 * half);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * r4 + e;
        float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -ls[e]));
        if (edge) {
          const int row = r0 + 8 * r4 + 4 * half + e, i = row / a.G;
          if (!(row < rows && active && (!a.causal || key <= i + nk - nq))) p = 0.0f;
        }
        s[r] = p;
        dp[r] = p * (dp[r] - de[e]);
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag p = to_frag<T>(s, t), d = to_frag<T>(dp, t);
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) {
        dv[dt] = Elem<T>::mma(TL::column(dt_, 16 * t, dt, lane), p, dv[dt]);
        dk[dt] = Elem<T>::mma(TL::column(qt, 16 * t, dt, lane), d, dk[dt]);
      }
    }
  }
  if (!inside) return;
  T *dkrow = (T *)a.dk.p + (long long)b * a.dk.b + (long long)key * a.dk.r + (long long)hk * a.dk.h;
  T *dvrow = (T *)a.dv.p + (long long)b * a.dv.b + (long long)key * a.dv.r + (long long)hk * a.dv.h;
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * dt + 2 * r + 4 * half;
      if (d < a.D) {
        store4<T>(dkrow + d, dk[dt][r] * a.scale, dk[dt][r + 1] * a.scale, dk[dt][r + 2] * a.scale, dk[dt][r + 3] * a.scale);
        store4<T>(dvrow + d, dv[dt][r], dv[dt][r + 1], dv[dt][r + 2], dv[dt][r + 3]);
      }
    }
}

// dq of 128 rows, 32 per wave, whose q and do rows stay in registers; walks the keys in tiles of 32.
template <typename T, int DP>
__global__ void __launch_bounds__(256, 1) attn_backward_q_kernel(AttnArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Frag Frag;
  constexpr int kKeys = 32, kKc = DP / 16, kDt = DP / 32;
  extern __shared__ __align__(16) char lds[];
  char *kt = lds, *vt = lds + kKeys * TL::kBytes;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
  int tile, group;
  xcd_group_map(blockIdx.x, a.tiles, a.B * a.Hk, tile, group);
  tile = a.tiles - 1 - tile;
  const int b = group / a.Hk, hk = group % a.Hk;
  const int nq = clamp_len(a.q_lens, b, a.Lq), nk = clamp_len(a.k_lens, b, a.Lk);
  const int row = tile * 128 + 32 * wave + col, i = row / a.G, g = row - i * a.G;
  const bool inside = row < a.Lq * a.G, active = i < nq;
  const int seen = !active ? 0 : a.causal ? min(nk, max(0, i + 1 + nk - nq)) : nk;
  const int i_last = min(nq, (min((tile + 1) * 128, a.Lq * a.G) - 1) / a.G + 1) - 1, i_first = tile * 128 / a.G;
  const int block_end = i_first >= nq ? 0 : a.causal ? min(nk, max(0, i_last + 1 + nk - nq)) : nk;
  const int full_end = a.causal ? min(nk, max(0, i_first + 1 + nk - nq)) : nk;
  const bool all_active = (i_last + 1) * a.G >= (tile + 1) * 128;
  const int h = hk * a.G + g;
  const T *qrow = (const T *)a.q.p + (long long)b * a.q.b + (long long)i * a.q.r + (long long)h * a.q.h;
  const T *drow = (const T *)a.dout.p + (long long)b * a.dout.b + (long long)i * a.dout.r + (long long)h * a.dout.h;
  const T *kh = (const T *)a.k.p + (long long)b * a.k.b + (long long)hk * a.k.h;
  const T *vh = (const T *)a.v.p + (long long)b * a.v.b + (long long)hk * a.v.h;
  Frag q[kKc], d[kKc];
#pragma unroll
  for (int kc = 0; kc < kKc; ++kc) { q[kc] = load_frag<T>(qrow, active, kc, half, a.D); d[kc] = load_frag<T>(drow, active, kc, half, a.D); }
  const long long at = ((long long)b * a.Hq + h) * a.Lq + i;
  const float ls = active ? a.lse[at] * kLog2e : 0.0f, de = active ? a.delta[at] : 0.0f;
  f32x16 dq[kDt];
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt) dq[dt] = f32x16{};
  Stage<T, DP, kKeys> ks, vs;
  ks.load(kh, a.k.r, 0, 1, 0, block_end, a.D, tid);
  vs.load(vh, a.v.r, 0, 1, 0, block_end, a.D, tid);
  for (int key0 = 0; key0 < block_end; key0 += kKeys) {
    lds_barrier();
    ks.store(kt, tid);
    vs.store(vt, tid);
    lds_barrier();
    if (key0 + kKeys < block_end) {
      ks.load(kh, a.k.r, 0, 1, key0 + kKeys, block_end, a.D, tid);
      vs.load(vh, a.v.r, 0, 1, key0 + kKeys, block_end, a.D, tid);
    }
    f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc) {
      s = Elem<T>::mma(TL::row(kt, col, kc, half), q[kc], s);
      dp = Elem<T>::mma(TL::row(vt, col, kc, half), d[kc], dp);
    }
    const bool edge = key0 + kKeys > full_end || !all_active;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.scale2, -ls));
      if (edge && key0 + 8 * (r >> 2) + 4 * half + (r & 3) >= seen) p = 0.0f;
      dp[r] = p * (dp[r] - de);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const Frag x = to_frag<T>(dp, t);
#pragma unroll
      for (int dt = 0; dt < kDt; ++dt) dq[dt] = Elem<T>::mma(TL::column(kt, 16 * t, dt, lane), x, dq[dt]);
    }
  }
  if (!inside) return;
  T *out = (T *)a.dq.p + (long long)b * a.dq.b + (long long)i * a.dq.r + (long long)h * a.dq.h;
#pragma unroll
  for (int dt = 0; dt < kDt; ++dt)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int e = 32 * dt + 2 * r + 4 * half;
      if (e < a.D) store4<T>(out + e, dq[dt][r] * a.scale, dq[dt][r + 1] * a.scale, dq[dt][r + 2] * a.scale, dq[dt][r + 3] * a.scale);
    }
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
  const int tile_bytes = 2 * kKeys * Tile<T, DP>::kBytes, join_bytes = narrow ? (4 * 32 * 2 + 4 * 32 * DP) * 4 : 0;
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
  const long long rows = (long long)a.B * a.Lq * a.Hq;
  hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a);
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  const int lds = 2 * 32 * Tile<T, DP>::kBytes;
  a.tiles = (a.Lk + 127) / 128;
  hipLaunchKernelGGL((attn_backward_kv_kernel<T, DP>), dim3((unsigned)a.tiles * a.B * a.Hk), dim3(256), lds + 256, st, a);
  rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  a.tiles = (a.Lq * a.G + 127) / 128;
  hipLaunchKernelGGL((attn_backward_q_kernel<T, DP>), dim3((unsigned)a.tiles * a.B * a.Hk), dim3(256), lds, st, a);
  return hipGetLastError();
}

template <typename T> hipError_t attn_forward_t(const AttnArgs &a, int narrow, hipStream_t st) {
  return a.D <= 64 ? attn_forward_dp<T, 64>(a, narrow, st) : attn_forward_dp<T, 128>(a, narrow, st);
}
template <typename T> hipError_t attn_backward_t(const AttnArgs &a, hipStream_t st) {
  return a.D <= 64 ? attn_backward_dp<T, 64>(a, st) : attn_backward_dp<T, 128>(a, st);
}

}  // namespace urf
