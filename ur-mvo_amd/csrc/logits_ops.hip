// logits_ops.hip -- operators over rows of scores (logits, log-assignments) on caller-owned tensors: log probabilities of given
// candidates with entropy and top alternatives, distillation from a teacher's top alternatives, and their gradients.
//
// With c = scale log2(e), m = max z and x_v = c (z_v - m):  S = sum 2^x_v,  lse = scale m + ln S,  and the entropy is
// (log2 S - A / S) ln 2 with A = sum 2^x_v x_v: one pass over the row, every lane with a running maximum of its own that rescales its
// sums when it grows.  (The difference comes before the product: scores at the lowest value of their type stay in range.)  The
// gradients need lse only and are one more pass: read a score, write its gradient.
// All of it is bound by memory: a score is read once per pass, 16 bytes a lane and load, four loads in flight per lane.  bf16: 2048 rows of
// 131072, 537 MB: log probabilities 121 us (4.4 TB/s, the entropy's operations beside it; fp32, 819 MB: 144 us, 5.7 TB/s), distillation 104
// (5.2 TB/s), a gradient 181 (1.07 GB, 5.9 TB/s); a large copy reaches 4.8 TB/s, a large sum 4.0.
//
// A row belongs to W waves (1, 4 or 16, one workgroup): 1 where the rows are short, 16 where there are too few rows to fill the
// chip with 4.  A few long rows (the next token of some sequences) are cut in parts, a workgroup of 4 each, whose sums and
// alternatives a second kernel joins.  Of many short rows a wave takes two, one per half (L = 32 lanes a row): what is done once per row
// -- joining the lanes, sorting, the row's results -- is most of the work there.  Sums are joined in a fixed order.  Rows may start at any
// element: the vectors begin at the row's first boundary, and the scores before and behind them are one more step.
//
// "Listed" candidates (targets, a teacher's alternatives): at most 64 a row, one per lane of every wave.  A wave asks by ballot
// whether any lies among the elements it is about to handle, which is rare in a long row, and only then looks whose they are.
// Their gradients are added to the element's own before its one rounding, in the list's order, so that a candidate listed twice
// gets both; there are no atomics and no second write.
#include "operator_common.h"

#include <math.h>

namespace urf {

static_assert(URF_TOP_MAX == 64, "one listed candidate per lane");
constexpr int kUnroll = 4;               // 16-byte loads in flight per lane
constexpr double kLog2eDouble = 1.4426950408889634;
constexpr int kMostParts = 32;           // of a row
constexpr int kShort = 2048;             // classes of an fp32 row whose gradient is normalised by the row's own sum (exact_lse)
constexpr int kKept = kShort / 256;      // vectors of it per lane of a wave
constexpr float kNothing = -0x1p100f;    // a row whose largest scaled score is below it allows nothing (masks of -inf or the lowest value)
constexpr float kFloor = -1.0e4f;        // 2^kFloor is 0: a masked score (-inf) adds 0 * kFloor to A, not 0 * inf

struct RowsArgs {
  const void *z;                 // [R] rows of V scores
  long long stride;              // elements between rows
  int R, V;
  float c;                       // scale * log2(e)
  float scale;                   // 1 / temperature for the distillation
  // log probabilities
  const int *targets; int N;     // [R][N]
  int K;                         // alternatives (log_probs), listed per row (distillation)
  float *log_prob, *entropy, *lse, *top_log_prob;
  int *top_index;
  // distillation
  const int *t_index; const float *t_value;      // [R][K]
  float *loss, *log_tail;
  // gradients
  const float *g1, *g2;          // d_log_prob [R][N] (or d_loss [R]); d_entropy [R]
  void *dz; long long dz_stride;
  int per_row;                   // gradients: waves per row
  // log probabilities of rows in parts: per row and part K keys, then a Stat
  int parts;
  unsigned long long *part_keys; struct Stat *part_stats;
};

// ------------------------------------------------------------------ rows
template <typename T> struct Row {
  static constexpr int kPer = 16 / (int)sizeof(T);
  typedef T Vec __attribute__((ext_vector_type(kPer)));
  typedef T LooseVec __attribute__((ext_vector_type(kPer), aligned(sizeof(T))));      // gradients whose rows begin elsewhere
  // scores before the first boundary: of 64 bytes, what the memory pipeline takes four lanes' vectors as (2048 rows of 100003 bf16
  // scores: 98 us, 104 from the rows' first elements on), or of 16 where the lanes of a row are too few to take up to 31 scores before it
  // and 7 behind the last vector
  template <int L> static __device__ __forceinline__ int head(const T *z, int V) {
    constexpr int kTo = L == 64 ? 63 : 15;
    return min(V, (int)(-(uintptr_t)z & kTo) / (int)sizeof(T));
  }
  static __device__ __forceinline__ void load(const T *p, float (&f)[kPer]) { spread(*(const Vec *)p, f); }
  static __device__ __forceinline__ void spread(const Vec &v, float (&f)[kPer]) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) f[e] = (float)v[e];
  }
  // kUnroll steps from step b on: the vectors below `end` steps and V scores; the others are -inf.  (z, V: from the first boundary on)
  template <int L> static __device__ __forceinline__ void fetch(const T *z, int b, int end, int V, int lane, Vec (&v)[kUnroll]) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int first = (b + u) * L * kPer + lane * kPer;
#pragma unroll
      for (int e = 0; e < kPer; ++e) v[u][e] = (T)-INFINITY;
      if (b + u < end && first + kPer <= V) v[u] = *(const Vec *)(z + first);
    }
  }
};

typedef unsigned long long u64;
// the value of lane ^ x, x a power of two, in the vector pipe (the LDS crossbar's latency is several times that)
__device__ __forceinline__ int lane_xor(int v, int x) {
  const int lane = threadIdx.x;
  switch (x) {
    case 1: return __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, false);
    case 2: return __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, false);
    case 4: return __builtin_amdgcn_update_dpp(0, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false), 0x1B, 0xf, 0xf, false);   // ^7, then ^3
    case 8: return __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, false);
    case 16: { const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false); return (lane & 16) ? r[0] : r[1]; }
    default: { const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false); return (lane & 32) ? r[0] : r[1]; }
  }
}
__device__ __forceinline__ float lane_xor(float v, int x) { return __int_as_float(lane_xor(__float_as_int(v), x)); }
__device__ __forceinline__ double lane_xor(double v, int x) {
  const long long u = __double_as_longlong(v);
  return __longlong_as_double(((long long)lane_xor((int)(u >> 32), x) << 32) | (unsigned)lane_xor((int)u, x));
}

// over the L lanes of a row
template <int L> __device__ __forceinline__ float row_max(float v) {
#pragma unroll
  for (int x = L / 2; x >= 1; x >>= 1) v = fmaxf(v, lane_xor(v, x));
  return v;
}
template <int L, typename F> __device__ __forceinline__ F row_sum(F v) {
#pragma unroll
  for (int x = L / 2; x >= 1; x >>= 1) v += lane_xor(v, x);
  return v;
}
// the lanes' votes on their row's question
template <int L> __device__ __forceinline__ u64 row_ballot(bool v) {
  const u64 all = __ballot(v);
  return L == 64 ? all : (threadIdx.x & 32) ? all >> 32 : all & 0xffffffffu;
}

// running maximum (of the scores) and sums of a lane, a wave, a row
struct Stat { float m, s, a; };
__device__ __forceinline__ Stat join(Stat p, Stat q, float c) {
  const float m = fmaxf(p.m, q.m), mu = m == -INFINITY ? 0.0f : m;
  const float xp = (p.m - mu) * c, xq = (q.m - mu) * c, fp = exp2f(xp), fq = exp2f(xq);
  // c (z - m) = c (z - p.m) + c (p.m - m)
  return {m, p.s * fp + q.s * fq, fmaf(p.s, fmaxf(xp, kFloor), p.a) * fp + fmaf(q.s, fmaxf(xq, kFloor), q.a) * fq};
}
template <int L> __device__ __forceinline__ Stat lanes_join(Stat v, float c) {
  const float m = row_max<L>(v.m), x = (v.m - (m == -INFINITY ? 0.0f : m)) * c, f = exp2f(x);
  return {m, row_sum<L>(v.s * f), row_sum<L>(fmaf(v.s, fmaxf(x, kFloor), v.a) * f)};
}

// ------------------------------------------------------------------ top alternatives
// The pass over a row only notes, per lane, its largest score and where it was (three instructions per 16 bytes).  The K-th largest
// of the lanes' best scores bounds the K-th largest of the row from below, so that afterwards only lanes whose best is not below it
// -- about K of the row's 64, 256 or 1024 -- have their scores read again, cooperatively, and only scores that are not below it
// are candidates: about K again.  They are sorted 64 at a time.  (2048 rows of 100003 bf16 scores: 88 us without alternatives, 96 with 4,
// 116 with 20, 161 with 64.  Keeping a list during the pass costs more than the pass: 129 -> 190 us at the time.)
// Keys: the score as an ordered integer above, the complement of its index below (equal scores: the lower index wins); 0 = none.
__device__ __forceinline__ u64 key_of(float z, int index) {
  const unsigned u = __float_as_uint(z + 0.0f);           // -0 counts as 0
  const unsigned o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((u64)o << 32) | (unsigned)~index;
}
__device__ __forceinline__ float key_score(u64 k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ u64 shfl64(u64 v, int src, int width) {
  return ((u64)(unsigned)__shfl((int)(v >> 32), src, width) << 32) | (unsigned)__shfl((int)(unsigned)v, src, width);
}
// the lanes (of 64) that keep the larger of themselves and their partner lane ^ x, in runs of n that alternate in direction
constexpr u64 keepers(int n, int x) {
  u64 mask = 0;
  for (int l = 0; l < 64; ++l) mask |= (u64)(((l & n) == 0) == ((l & x) == 0)) << l;
  return mask;
}
template <int N, int X> __device__ __forceinline__ u64 exchange(u64 v) {
  constexpr u64 larger = keepers(N, X);
  const u64 o = ((u64)(unsigned)lane_xor((int)(v >> 32), X) << 32) | (unsigned)lane_xor((int)(unsigned)v, X);
  return __builtin_amdgcn_inverse_ballot_w64(__ballot(v > o) ^ ~larger) ? v : o;
}
template <int N, int X> __device__ __forceinline__ u64 merge_steps(u64 v) {
  v = exchange<N, X>(v);
  if constexpr (X > 1) v = merge_steps<N, X / 2>(v);
  return v;
}
// over the L lanes of a row, descending (N = L at the end: every lane's bit L is taken as 0, all runs descend)
template <int L, int N = 2> __device__ __forceinline__ u64 sort_desc(u64 v) {
  v = merge_steps<N == L ? 64 : N, N / 2>(v);
  if constexpr (N < L) v = sort_desc<L, 2 * N>(v);
  return v;
}
// both descending: the L largest of the two, descending
template <int L> __device__ __forceinline__ u64 merge_desc(u64 a, u64 b, int lane) {
  const u64 r = shfl64(b, L - 1 - lane, L);
  return merge_steps<64, L / 2>(a > r ? a : r);
}

// ------------------------------------------------------------------ listed candidates
// `mine` = this lane's listed index or -1, `hits` = the lanes whose index lies in the range at hand, f = elements first + 0 .. n - 1
template <int L, int n> __device__ __forceinline__ void hide_listed(float *f, int first, int mine, u64 hits) {
  while (__any(hits != 0)) {
    const int src = hits ? (int)__ffsll((long long)hits) - 1 : 0, index = __shfl(mine, src, L), at = hits ? index - first : -1;
    hits &= hits - 1;
#pragma unroll
    for (int e = 0; e < n; ++e)
      if (e == at) f[e] = -INFINITY;
  }
}

// what the pass of a wave (or half of one) over its share of a row leaves in a lane, beside the sums
struct Share {
  int head;          // scores before the first vector: the vectors' scores are counted from there
  int b0, b1;        // the share: steps of L vectors of 16 bytes
  float best;        // the lane's largest score (whole vectors), and the first step it was in (-1: the lane has no vector)
  int best_at;
  float extra;       // what is left of the row before and behind the vectors: one score a lane of part 0, its index or -1
  int extra_at;
};

// One pass of a wave over its share of a row.  TOP: notes the lanes' best scores; TAIL: leaves the listed candidates out, so that a
// tail far below them keeps its own maximum.
template <typename T, int W, int L, bool ENTROPY, bool TOP, bool TAIL>
__device__ __forceinline__ Stat row_pass(const T *z, int V, float c, int part, int parts, int lane, int mine, Share &sh) {
  typedef Row<T> RW;
  constexpr int kPer = RW::kPer, kStep = L * kPer;
  Stat st = {-INFINITY, 0.0f, 0.0f};
  auto absorb = [&](const float *f, int n) {
    float top = f[0];
#pragma unroll
    for (int e = 1; e < n; ++e) top = fmaxf(top, f[e]);
    const float m = fmaxf(st.m, top), mu = m == -INFINITY ? 0.0f : m;
    const float x0 = (st.m - mu) * c, f0 = __builtin_amdgcn_exp2f(x0);
    if (ENTROPY) st.a = fmaf(st.s, fmaxf(x0, kFloor), st.a) * f0;
    st.s *= f0;
    st.m = m;
#pragma unroll
    for (int e = 0; e < n; ++e) {
      const float x = (f[e] - mu) * c, p = __builtin_amdgcn_exp2f(x);
      st.s += p;
      if (ENTROPY) st.a = fmaf(p, fmaxf(x, kFloor), st.a);
    }
    return top;
  };
  const int head = RW::template head<L>(z, V), tail = (V - head) % kPer, all = V;
  const T *row = z;
  z += head;
  V -= head;
  sh.head = head;
  const int steps = (V / kPer + L - 1) / L;
  sh.b0 = (int)((long long)steps * part / parts);
  sh.b1 = (int)((long long)steps * (part + 1) / parts);
  sh.best = -INFINITY;
  sh.best_at = sh.b0 < sh.b1 && sh.b0 * kStep + (lane + 1) * kPer <= V ? sh.b0 : -1;
  typename RW::Vec now[kUnroll], next[kUnroll];
  if (W > 1) RW::template fetch<L>(z, sh.b0, sh.b1, V, lane, now);
  for (int b = sh.b0; b < sh.b1; b += kUnroll) {
    // long rows: the next scores are in flight while these are taken in; short ones are one or two steps
    if (W > 1) RW::template fetch<L>(z, b + kUnroll, sh.b1, V, lane, next);
    else RW::template fetch<L>(z, b, sh.b1, V, lane, now);
    float f[kUnroll][kPer];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (b + u < sh.b1) {
        const int base = head + (b + u) * kStep, first = base + lane * kPer;
        RW::spread(now[u], f[u]);
        if (TAIL) {
          const u64 hits = row_ballot<L>(mine >= base && mine < base + kStep);
          if (__any(hits != 0)) hide_listed<L, kPer>(f[u], first, mine, hits);
        }
        const float top = absorb(f[u], kPer);
        if (TOP && top > sh.best) { sh.best = top; sh.best_at = b + u; }
      }
    if (W > 1)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) now[u] = next[u];
  }
  sh.extra = -INFINITY;
  sh.extra_at = part || lane >= head + tail ? -1 : lane < head ? lane : all - tail + lane - head;
  if (part == 0 && head + tail) {
    if (sh.extra_at >= 0) sh.extra = (float)row[sh.extra_at];
    if (TAIL) {
      const u64 hits = row_ballot<L>(mine >= 0 && (mine < head || mine >= all - tail));
      if (__any(hits != 0)) hide_listed<L, 1>(&sh.extra, sh.extra_at, mine, hits);
    }
    absorb(&sh.extra, 1);
  }
  return st;
}

// The row's 64 largest keys of the waves' sorted lists, in wave 0 and in its part of the LDS (64 keys per wave).
template <int W> __device__ __forceinline__ u64 lists_join(u64 list, int wave, int lane, u64 *lds) {
  if constexpr (W > 1) {
    lds_barrier();
    lds[wave * 64 + lane] = list;
    lds_barrier();
    for (int n = W / 2; n >= 1; n >>= 1) {
      if (wave < n) {
        list = merge_desc<64>(list, lds[(wave + n) * 64 + lane], lane);
        lds[wave * 64 + lane] = list;
      }
      lds_barrier();
    }
  }
  return list;
}

// The alternatives of a row, descending, one key per lane, in wave 0 (K <= L).  LDS: 64 keys per wave to join, 2.5 L keys of the
// row's own lanes.  What loops, loops for both rows of a wave together.
template <typename T, int W, int L>
__device__ __forceinline__ u64 top_alternatives(const T *z, int V, int K, const Share &sh, int wave, int lane, u64 *lds, u64 *own_lds) {
  typedef Row<T> RW;
  constexpr int kPer = RW::kPer, kStep = L * kPer;
  const int head = sh.head;
  z += head;
  V -= head;
  float f[kPer];
  u64 best = sh.extra_at >= 0 ? key_of(sh.extra, sh.extra_at) : 0;
  if (sh.best_at >= 0) {
    const int first = sh.best_at * kStep + lane * kPer;
    RW::load(z + first, f);
    int at = 0;
#pragma unroll
    for (int e = kPer - 1; e >= 0; --e)
      if (f[e] == sh.best) at = e;
    const u64 k = key_of(sh.best, head + first + at);
    best = k > best ? k : best;
  }
  u64 list = lists_join<W>(sort_desc<L>(best), wave, lane, lds);
  u64 bound = shfl64(list, K - 1, L);
  if constexpr (W > 1) bound = lds[K - 1];                 // wave 0's list
  // the winners' scores, (winner, step) pairs spread over the lanes
  const u64 winners = row_ballot<L>(sh.best_at >= 0 && best >= bound), below = (1ull << lane) - 1;
  u64 *wait = own_lds;
  int *who = (int *)(own_lds + 2 * L);
  if ((winners >> lane) & 1) who[__popcll(winners & below)] = lane;
  __builtin_amdgcn_wave_barrier();
  list = 0;
  int count = 0;
  // takes in a candidate per lane (0 = none); sorts and merges whenever L wait, or what there is
  auto take = [&](u64 key, bool all) {
    const u64 pass = row_ballot<L>(key && key >= bound);
    if ((pass >> lane) & 1) wait[count + __popcll(pass & below)] = key;
    count += __popcll(pass);
    while (__any(count >= L || (all && count > 0))) {
      __builtin_amdgcn_wave_barrier();
      list = merge_desc<L>(list, sort_desc<L>(lane < count ? wait[lane] : 0), lane);
      const u64 rest = lane + L < count ? wait[lane + L] : 0;
      __builtin_amdgcn_wave_barrier();
      wait[lane] = rest;
      __builtin_amdgcn_wave_barrier();
      count = max(0, count - L);
      const u64 kth = shfl64(list, K - 1, L);
      bound = kth > bound ? kth : bound;
    }
  };
  const int ns = sh.b1 - sh.b0, pairs = __popcll(winners) * ns;
  for (int i0 = 0; __any(i0 < pairs); i0 += L) {
    const int i = i0 + lane, w = i / max(ns, 1), first = (sh.b0 + i - w * ns) * kStep + (i < pairs ? who[w] : 0) * kPer;
    const bool valid = i < pairs && first + kPer <= V;
    if (valid) RW::load(z + first, f);
#pragma unroll 1
    for (int e = 0; e < kPer; ++e) {
      take(valid ? key_of(f[0], head + first + e) : 0, false);
#pragma unroll
      for (int x = 0; x + 1 < kPer; ++x) f[x] = f[x + 1];
    }
  }
  take(sh.extra_at >= 0 ? key_of(sh.extra, sh.extra_at) : 0, true);
  return lists_join<W>(list, wave, lane, lds);
}

// joins the parts of a row, in every wave
template <int W, int L> __device__ __forceinline__ Stat row_join(Stat st, float c, int wave, int lane, Stat *lds) {
  st = lanes_join<L>(st, c);
  if constexpr (W > 1) {
    if (lane == 0) lds[wave] = st;
    lds_barrier();
    st = lds[0];
#pragma unroll
    for (int w = 1; w < W; ++w) st = join(st, lds[w], c);
  }
  return st;
}

// ------------------------------------------------------------------ forward kernels
// which row, wave of the row and lane of the row a thread is
template <int W, int L> struct Place {
  static constexpr int kRows = W > 1 ? 1 : 256 / L;        // of a workgroup
  const int lane = threadIdx.x & (L - 1), slot = W > 1 ? 0 : threadIdx.x / L, wave = W > 1 ? threadIdx.x >> 6 : 0;
  const int row = blockIdx.x * kRows + slot;
};

// what is done once per row, by its first wave; `list`: its alternatives
template <typename T, bool TOP> __device__ __forceinline__ void finish_log_probs(const RowsArgs &a, int r, const Stat &st, u64 list, int lane) {
  const T *z = (const T *)a.z + (long long)r * a.stride;
  // a NaN or +inf score leaves no distribution: everything is NaN and the alternatives are -1.  A row that allows nothing: lse
  // -inf, entropy 0, every log probability -inf.
  const bool broken = !(st.s >= 0.0f) || st.m == INFINITY, empty = st.m * a.scale < kNothing && !broken;
  const float ls = logf(st.s), nan = __uint_as_float(0x7fc00000u);
  if (lane == 0) {
    a.lse[r] = broken ? nan : empty ? -INFINITY : (float)((double)st.m * a.scale + ls);
    a.entropy[r] = broken ? nan : empty ? 0.0f : fmaf(-st.a / st.s, kLn2, ls);
  }
  auto log_prob = [&](float x) { return broken ? nan : empty || x == -INFINITY ? -INFINITY : fmaf(x - st.m, a.scale, -ls); };
  if (lane < a.N) {
    const int t = a.targets[(long long)r * a.N + lane];
    a.log_prob[(long long)r * a.N + lane] = t >= 0 && t < a.V ? log_prob((float)z[t]) : 0.0f;
  }
  if (TOP && lane < a.K) {
    a.top_index[(long long)r * a.K + lane] = broken ? -1 : (int)~(unsigned)list;
    a.top_log_prob[(long long)r * a.K + lane] = log_prob(key_score(list));
  }
}

template <typename T, int W, int L, bool TOP>
__global__ void __launch_bounds__(W == 16 ? 1024 : 256) log_probs_kernel(RowsArgs a) {
  constexpr int kWaves = W == 16 ? 16 : 4;
  __shared__ Stat stats[kWaves];
  __shared__ u64 keys[TOP ? (64 + 160) * kWaves : 1];
  const Place<W, L> place;
  const int lane = place.lane, wave = place.wave, r = place.row;
  if (r >= a.R) return;                                    // (of a wave with one row to do, the other half is gone)
  const T *z = (const T *)a.z + (long long)r * a.stride;
  Share sh;
  Stat st = row_pass<T, W, L, true, TOP, false>(z, a.V, a.c, wave, W, lane, -1, sh);
  st = row_join<W, L>(st, a.c, wave, lane, stats);
  u64 list = 0;
  if constexpr (TOP) list = top_alternatives<T, W, L>(z, a.V, a.K, sh, wave, lane, keys, keys + 64 * kWaves + 5 * L / 2 * (threadIdx.x / L));
  if (wave) return;
  finish_log_probs<T, TOP>(a, r, st, list, lane);
}

// A row in parts, and their join: a workgroup per row, lane p of a wave holds part p's sums, a wave merges the lists of every
// fourth part.
template <typename T, bool TOP>
__global__ void __launch_bounds__(256) log_probs_part_kernel(RowsArgs a) {
  __shared__ Stat stats[4];
  __shared__ u64 keys[TOP ? (64 + 160) * 4 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x / a.parts, part = blockIdx.x - r * a.parts;
  const T *z = (const T *)a.z + (long long)r * a.stride;
  Share sh;
  Stat st = row_pass<T, 4, 64, true, TOP, false>(z, a.V, a.c, 4 * part + wave, 4 * a.parts, lane, -1, sh);
  st = row_join<4, 64>(st, a.c, wave, lane, stats);
  u64 list = 0;
  if constexpr (TOP) list = top_alternatives<T, 4, 64>(z, a.V, a.K, sh, wave, lane, keys, keys + 64 * 4 + 160 * wave);
  if (wave) return;
  if (lane == 0) a.part_stats[blockIdx.x] = st;
  if (TOP && lane < a.K) a.part_keys[(long long)blockIdx.x * a.K + lane] = list;
}
template <typename T, bool TOP>
__global__ void __launch_bounds__(256) log_probs_join_kernel(RowsArgs a) {
  __shared__ u64 keys[TOP ? 64 * 4 : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x;
  Stat st = {-INFINITY, 0.0f, 0.0f};
  if (lane < a.parts) st = a.part_stats[r * a.parts + lane];
  u64 list = 0;
  if constexpr (TOP) {
    u64 lists[kMostParts / 4];                              // parts wave, wave + 4, ...
#pragma unroll
    for (int i = 0; i < kMostParts / 4; ++i) {
      const int p = wave + 4 * i;
      lists[i] = p < a.parts && lane < a.K ? a.part_keys[((long long)r * a.parts + p) * a.K + lane] : 0;
    }
#pragma unroll
    for (int n = kMostParts / 8; n >= 1; n >>= 1)
#pragma unroll
      for (int i = 0; i < n; ++i)
        if (wave + 4 * (i + n) < a.parts) lists[i] = merge_desc<64>(lists[i], lists[i + n], lane);
    list = lists_join<4>(lists[0], wave, lane, keys);
  }
  if (wave) return;
  finish_log_probs<T, TOP>(a, r, lanes_join<64>(st, a.c), list, lane);
}

// the teacher's side of a row: lane k holds alternative k (index -1 where there is none), its probability and log probability
// (in 64 bits: what is left of 1, and of teacher and student where they agree, is a difference)
struct Teacher { int index; double p, lp, mass, rest; };
template <bool TAIL, int L>
__device__ __forceinline__ Teacher teacher_of(const RowsArgs &a, int r, int lane) {
  Teacher t = {-1, 0.0, 0.0, 0.0, 0.0};
  double v = -INFINITY;
  if (lane < a.K) {
    t.index = a.t_index[(long long)r * a.K + lane];
    if (t.index < 0 || t.index >= a.V) t.index = -1;
    else v = a.t_value[(long long)r * a.K + lane];
  }
  if (TAIL) {
    t.lp = v;
    t.p = exp(v);
    const double sum = row_sum<L>(t.p);
    t.rest = fmax(1.0 - sum, 0.0);
    if (t.rest < 0x1p-20) t.rest = 0.0;                   // below the rounding of the listed probabilities: there is no rest
    t.mass = sum + t.rest;
  } else {
    v *= (double)a.scale;
    const float m = row_max<L>((float)v);
    const float e = m == -INFINITY ? 0.0f : expf((float)(v - m)), sum = row_sum<L>(e);
    t.p = sum == 0.0f ? 0.0f : e / sum;
    t.lp = v - m - logf(sum);
    t.mass = sum == 0.0f ? 0.0 : sum == sum ? 1.0 : sum;
  }
  return t;
}

// the student's side of a row: its largest score, the sum of the exponentials from there and its logarithm, the logarithm of the
// unlisted share, the score in this lane's listed place and the logarithm of the teacher's rest
struct Student { float m, zk; double all, log_all, tail, log_rest; };
// `st`: of the row, TAIL: without the listed candidates.  A few operations per row, in 64 bits: a divergence close to zero is a
// difference of far larger terms.
template <typename T, bool TAIL, int L>
__device__ __forceinline__ Student student_of(const RowsArgs &a, const T *z, const Teacher &t, const Stat &st, int lane) {
  Student q;
  const bool used = t.index >= 0;
  q.zk = used ? (float)z[t.index] : -INFINITY;
  q.m = st.m;                                             // of the whole row
  double sum = st.s, listed = 0.0;
  if (TAIL) {
    // the pass left the listed candidates out: add each of them once
    bool first = used;
    for (int k = 0; k < a.K; ++k) {
      const int other = __shfl(t.index, k, L);
      if (k < lane && other == t.index) first = false;
    }
    q.m = fmaxf(q.m, row_max<L>(q.zk));
    const float mu = q.m == -INFINITY ? 0.0f : q.m;
    listed = row_sum<L>(first ? (double)exp2f((q.zk - mu) * a.c) : 0.0);
    sum = st.s * exp2f((st.m - mu) * a.c);
  }
  q.all = sum + listed;
  // the logarithms, each in a lane of its own: of the sum, of the unlisted share of it, of the teacher's rest.  Where the unlisted
  // share is too small for the sum's scale, its own maximum counts.
  const bool far = TAIL && sum < 0x1p-100 * q.all;
  const double logs = log(lane == 0 ? q.all : lane == 1 ? (far ? (double)st.s : listed < sum ? 1.0 - listed / q.all : sum / q.all) : t.rest);
  q.log_all = __shfl(logs, 0, L);
  q.tail = q.log_rest = 0.0;
  if (TAIL) {
    q.tail = __shfl(logs, 1, L);
    if (far) q.tail += (st.m - (double)q.m) * a.scale - q.log_all;
    q.log_rest = __shfl(logs, 2, L);
  }
  return q;
}

template <typename T, int W, int L, bool TAIL>
__global__ void __launch_bounds__(W == 16 ? 1024 : 256) distill_kernel(RowsArgs a) {
  __shared__ Stat stats[W];
  const Place<W, L> place;
  const int lane = place.lane, wave = place.wave, r = place.row;
  if (r >= a.R) return;
  const T *z = (const T *)a.z + (long long)r * a.stride;
  const Teacher t = teacher_of<TAIL, L>(a, r, lane);
  Share sh;
  Stat st = row_pass<T, W, L, false, false, TAIL>(z, a.V, a.c, wave, W, lane, t.index, sh);
  st = row_join<W, L>(st, a.c, wave, lane, stats);
  if (wave) return;
  const Student q = student_of<T, TAIL, L>(a, z, t, st, lane);
  const float nan = __uint_as_float(0x7fc00000u);
  const bool broken = !(q.all >= 0.0) || q.m == INFINITY, empty = q.m * a.scale < kNothing && !broken;
  const double lq = q.zk == -INFINITY ? -INFINITY : ((double)q.zk - q.m) * a.scale - q.log_all;
  double loss = row_sum<L>(t.p != 0.0 ? t.p * (t.lp - lq) : 0.0);
  if (TAIL && t.rest > 0.0) loss += t.rest * (q.log_rest - q.tail);
  if (empty) loss = t.mass != 0.0 ? INFINITY : 0.0;       // the student allows nothing
  if (lane == 0) {
    a.loss[r] = broken ? nan : (float)loss;
    a.lse[r] = broken ? nan : empty ? -INFINITY : (float)((double)q.m * a.scale + q.log_all);
    if (TAIL) a.log_tail[r] = broken ? nan : empty ? -INFINITY : (float)q.tail;
  }
}

// ------------------------------------------------------------------ gradients
// dz = coefficient * exp(scale z - shift) [ * (1 + ...) ] + what the listed candidates add; one read, one write per score
struct GradRow {
  float shift, slo;  // lse (or lse and the tail's log probability), and what the float lacks (fp32 scores)
  float coef;        // of the probability
  float h, ent2;     // ENTROPY: -h p (log2 p + ent2), in log2 units
  float lshift, lslo, lcoef;   // TAIL: of a listed candidate's probability
  int mine;          // this lane's listed index (-1: none) and what it adds
  float add;
};

__device__ __forceinline__ void set_shift(float &hi, float &lo, double shift) {
  hi = (float)shift;
  lo = (float)(shift - (double)hi);
}

// a short row, read once for its sum and its gradient: its vectors, and the score that a lane takes before or behind them
template <typename T> struct Kept {
  typename Row<T>::Vec v[kKept];
  float extra;
};
template <typename T> __device__ __forceinline__ Kept<T> keep_row(const T *z, int V, int lane) {
  typedef Row<T> RW;
  constexpr int kPer = RW::kPer;
  const int head = RW::template head<64>(z, V), tail = (V - head) % kPer, at = lane >= head + tail ? -1 : lane < head ? lane : V - tail + lane - head;
  Kept<T> k;
#pragma unroll
  for (int s = 0; s < kKept; ++s) {
    const int first = (s * 64 + lane) * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) k.v[s][e] = (T)-INFINITY;
    if (first + kPer <= V - head) k.v[s] = *(const typename RW::Vec *)(z + head + first);
  }
  k.extra = at >= 0 ? (float)z[at] : -INFINITY;
  return k;
}

// STREAM: written past the caches (a template: the compiler joins two stores that differ in this only).  KEEP: the row is in `kept`, 1: its
// scores, 2: its probabilities, which coef and lcoef are of
template <typename T, bool ENTROPY, bool TAIL, bool STREAM, int KEEP>
__device__ __forceinline__ void grad_pass(const T *z, T *dz, int V, float scale, const GradRow &g, int part, int parts, int lane, const Kept<T> &kept) {
  typedef Row<T> RW;
  constexpr int kPer = RW::kPer, kStep = 64 * kPer;
  auto exponent = [&](float f, float shift, float slo) {
    const float d = fmaf(f, scale, -shift);
    return (sizeof(T) == 4 ? d - slo : d) * kLog2e;
  };
  auto grad = [&](float f) {
    if (KEEP == 2) return f * g.coef;
    const float x = exponent(f, g.shift, g.slo), p = __builtin_amdgcn_exp2f(x);
    if (ENTROPY) return p * fmaf(-g.h, fmaxf(x, kFloor) + g.ent2, g.coef);
    return p * g.coef;
  };
  // elements first + 0 .. n - 1 of the lane, some of the wave's are listed
  auto listed = [&](const float *f, float *d, int n, int first, u64 hits) {
    if (TAIL)                                              // their own terms, not the tail's
      for (u64 h = hits; h; h &= h - 1) {
        const int at = __shfl(g.mine, (int)__ffsll((long long)h) - 1, 64) - first;
#pragma unroll
        for (int e = 0; e < n; ++e)
          if (e == at) d[e] = g.lcoef * (KEEP == 2 ? f[e] : __builtin_amdgcn_exp2f(exponent(f[e], g.lshift, g.lslo)));
      }
    for (u64 h = hits; h; h &= h - 1) {                    // what each mention adds, in the list's order
      const int src = (int)__ffsll((long long)h) - 1, at = __shfl(g.mine, src, 64) - first;
      const float add = __shfl(g.add, src, 64);
#pragma unroll
      for (int e = 0; e < n; ++e)
        if (e == at) d[e] += add;
    }
  };
  const int head = RW::template head<64>(z, V), tail = (V - head) % kPer, all = V;
  const T *row = z;
  T *drow = dz;
  z += head;
  dz += head;
  V -= head;
  const bool loose = (uintptr_t)dz & 15;
  const int steps = (V / kPer + 63) / 64;
  const int b0 = (int)((long long)steps * part / parts), b1 = (int)((long long)steps * (part + 1) / parts);
  auto steps_from = [&](int b) __attribute__((always_inline)) {
    float f[kUnroll][kPer];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int first = (b + u) * kStep + lane * kPer;
      if constexpr (KEEP) RW::spread(kept.v[b + u], f[u]);
      else if (b + u < b1 && first + kPer <= V) RW::load(z + first, f[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (b + u < b1) {
        const int base = head + (b + u) * kStep, first = (b + u) * kStep + lane * kPer;
        float d[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) d[e] = grad(f[u][e]);
        const u64 hits = __ballot(g.mine >= base && g.mine < base + kStep);
        if (hits) listed(f[u], d, kPer, head + first, hits);
        if (first + kPer <= V) {
          typename RW::Vec o;
#pragma unroll
          for (int e = 0; e < kPer; ++e) o[e] = (T)d[e];
          if (loose) *(typename RW::LooseVec *)(dz + first) = o;
          else if constexpr (STREAM) __builtin_nontemporal_store(o, (typename RW::Vec *)(dz + first));
          else *(typename RW::Vec *)(dz + first) = o;
        }
      }
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int b = 0; b < kKept; b += kUnroll)
      if (b < b1) steps_from(b);
  } else {
    for (int b = b0; b < b1; b += kUnroll) steps_from(b);
  }
  if (part == 0 && head + tail) {
    const int at = lane >= head + tail ? -1 : lane < head ? lane : all - tail + lane - head;
    const float f[1] = {KEEP ? kept.extra : at >= 0 ? (float)row[at] : -INFINITY};
    float d[1] = {grad(f[0])};
    const u64 hits = __ballot(g.mine >= 0 && (g.mine < head || g.mine >= all - tail));
    if (hits) listed(f, d, 1, at, hits);
    if (at >= 0) drow[at] = (T)d[0];
  }
}

// A row's lse from the one that was rounded to 32 bits.  Where probability and what is subtracted from it are close, that rounding is
// all that would be left of a gradient (fp32: rows of five classes, all of them listed: 1.7e-6 of its norm, 3e-7 so; 1585 classes, 20
// listed, student near its teacher: 1.6e-6, 3.8e-7).  The sum of the probabilities says how far it is off.  A wave that has its row to
// itself reads it once for both (us for 8200 rows of 1025, distillation / log probabilities: 17.7 / 14.5; without the sum 15.5 / 13.3, read
// twice 19.0 / 16.5); where a few rows are spread over waves each reads all of it.  Longer rows keep the rounded lse (their gradients are
// off by up to 8e-7).  16-bit gradients are rounded coarser than that.
template <typename T> __device__ __forceinline__ double exact_lse(const T *z, int V, float scale, float lse, int lane) {
  if constexpr (sizeof(T) == 4) {
    if (V <= kShort) {
      float sum = 0.0f;
      for (int v = lane; v < V; v += 256) {
        float f[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) f[u] = v + 64 * u < V ? z[v + 64 * u] : -INFINITY;
#pragma unroll
        for (int u = 0; u < 4; ++u) sum += __builtin_amdgcn_exp2f(fmaf(f[u], scale, -lse) * kLog2e);
      }
      return (double)lse + logf(row_sum<64>(sum));
    }
  }
  return lse;
}
// of a kept row: the sum of its probabilities by the rounded lse, which replace the scores if asked to (PROBS)
template <typename T, bool PROBS> __device__ __forceinline__ float kept_sum(Kept<T> &k, int V, float scale, float lse) {
  float sum = 0.0f;
  auto p_of = [&](float f) {
    const float p = __builtin_amdgcn_exp2f(fmaf(f, scale, -lse) * kLog2e);
    sum += p;
    return PROBS ? p : f;
  };
#pragma unroll
  for (int s = 0; s < kKept; ++s)
    if (256 * s < V)                                       // (the same for all lanes)
#pragma unroll
      for (int e = 0; e < Row<T>::kPer; ++e) k.v[s][e] = p_of(k.v[s][e]);
  k.extra = p_of(k.extra);
  return row_sum<64>(sum);
}

template <typename T, bool ENTROPY, bool STREAM, bool KEEP>
__global__ void __launch_bounds__(256) log_probs_backward_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int r = a.R - 1 - (int)(w / a.per_row), part = (int)(w % a.per_row);      // the last rows, read last by the forward pass, first
  if (r < 0) return;
  const T *z = (const T *)a.z + (long long)r * a.stride;
  Kept<T> kept;
  if constexpr (KEEP) kept = keep_row(z, a.V, lane);
  const float lse = a.lse[r];
  const bool empty = lse == -INFINITY;                    // no score to choose from: constant outputs, no gradient
  GradRow g = {};
  g.mine = -1;
  float own = 0.0f;
  if (lane < a.N) {
    g.mine = a.targets[(long long)r * a.N + lane];
    if (g.mine < 0 || g.mine >= a.V || empty) g.mine = -1;
    else own = a.g1[(long long)r * a.N + lane];
  }
  g.add = own * a.scale;
  double exact = empty ? 0.0 : lse;
  if constexpr (KEEP) exact += empty ? 0.0f : logf(kept_sum<T, false>(kept, a.V, a.scale, lse));
  else if (!empty) exact = exact_lse(z, a.V, a.scale, lse, lane);
  set_shift(g.shift, g.slo, exact);
  g.coef = empty ? 0.0f : -row_sum<64>(own) * a.scale;
  if (ENTROPY && !empty) {
    g.h = a.g2[r] * a.scale * kLn2;
    g.ent2 = a.entropy[r] * kLog2e;
  }
  grad_pass<T, ENTROPY, false, STREAM, KEEP ? 1 : 0>(z, (T *)a.dz + (long long)r * a.dz_stride, a.V, a.scale, g, part, a.per_row, lane, kept);
}

template <typename T, bool TAIL, bool STREAM, bool KEEP>
__global__ void __launch_bounds__(256) distill_backward_kernel(RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const long long w = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int r = a.R - 1 - (int)(w / a.per_row), part = (int)(w % a.per_row);      // the last rows, read last by the forward pass, first
  if (r < 0) return;
  const T *z = (const T *)a.z + (long long)r * a.stride;
  Kept<T> kept;
  if constexpr (KEEP) kept = keep_row(z, a.V, lane);
  const Teacher t = teacher_of<TAIL, 64>(a, r, lane);
  const double gs = (double)a.g1[r] * a.scale;
  const bool empty = a.lse[r] == -INFINITY;
  GradRow g = {};
  g.mine = empty ? -1 : t.index;
  g.add = (float)(-gs * t.p);
  T *dz = (T *)a.dz + (long long)r * a.dz_stride;
  double lse = empty ? 0.0 : a.lse[r];
  if constexpr (KEEP) {
    const float tail = TAIL ? a.log_tail[r] : 0.0f, sum = empty ? 1.0f : kept_sum<T, true>(kept, a.V, a.scale, (float)lse);
    // the probabilities are at hand unless the unlisted ones are too small next to the listed
    if (!empty && !(tail < -40.0f)) {
      g.lcoef = (float)(gs * t.mass / sum);
      g.coef = TAIL ? (float)(gs * (t.mass - t.rest * expf(-tail)) / sum) : g.lcoef;
      return grad_pass<T, false, TAIL, STREAM, 2>(z, dz, a.V, a.scale, g, part, a.per_row, lane, kept);
    }
    lse += logf(sum);
  } else if (!empty) {
    lse = exact_lse(z, a.V, a.scale, a.lse[r], lane);
  }
  set_shift(g.shift, g.slo, lse);
  g.coef = empty ? 0.0f : (float)(gs * t.mass);
  if (TAIL) {
    g.lshift = g.shift;
    g.lslo = g.slo;
    g.lcoef = g.coef;
    // unlisted v: mass q_v - rest q_v / q_tail = (mass q_tail - rest) exp(scale z - shift) with the tail's probability in the shift,
    // a probability within the tail: nothing overflows however small q_tail is
    const float tail = a.log_tail[r];
    if (!empty && tail != -INFINITY) {
      set_shift(g.shift, g.slo, lse + tail);
      g.coef = (float)(gs * (t.mass * expf(tail) - t.rest));
    }
  }
  grad_pass<T, false, TAIL, STREAM, 0>(z, dz, a.V, a.scale, g, part, a.per_row, lane, kept);
}

// ------------------------------------------------------------------ launches
// Waves per row.  One for short rows and, the more rows there are, for longer ones (what is done once per row, the alternatives most of
// all, costs every wave); sixteen for long rows where four would leave CUs with less than two workgroups.  bf16, us for the
// sums / with 8 alternatives / distillation: 512 rows of 3000: 4.5 / 8.5 / 4.8 with one wave, 4.3 / 9.9 / 4.9 with four, 8.5 / 23.8 / 7.8
// with sixteen; 8192 rows of 12000: 35 / 61 / 35, 39 / 76 / 40, 131 / 382 / 97; 1024 rows of 24000: 17.6 / 31 / 16.3, 13.9 / 22 / 13.8,
// 22 / 53 / 17; 256 rows of 131072: 73 / 109 / 65, 23 / 32 / 22, 20 / 27 / 19; 256 rows of 24000: 14 / 26 / 13, 6.1 / 12.4 / 6.4, 6.4 / 15 / 6.9.
inline int row_waves(int R, int V, int bytes) {
  const long long size = (long long)V * bytes, one = 16ll * R < 6144 ? 6144 : 16ll * R < 32768 ? 16ll * R : 32768;
  return size <= one ? 1 : R <= 256 && size > 96 * 1024 ? 16 : 4;
}
// Parts per row, two workgroups per CU and at least 8 KiB each; 0 = one workgroup does a row.  One launch against two, bf16, us
// without / with 20 alternatives: 1 row of 131072: 13.1 / 22.5 -> 5.1 / 13.0; 64: 13.9 / 23.7 -> 8.2 / 16.7; 128: 14.5 / 24.2 -> 11.9 / 22.8;
// 256: 21.0 / 27.8 -> 19.6 / 34.0; with 8 alternatives 32 rows of 48000: 9.3 / 15.6 -> 6.7 / 13.5; 128 of 24000: 6.0 / 11.2 -> 6.7 / 13.2.
// More parts cost their joining: 1 row of 131072 in 64 of 4 KiB: 5.0 / 14.8.
inline int row_parts(int R, int V, int bytes) {
  const long long size = (long long)V * bytes;
  if (size < 64 * 1024 || R > 128) return 0;
  const long long by_size = size / 8192, fill = 512 / R, n = by_size < fill ? by_size : fill;
  return n > kMostParts ? kMostParts : (int)n;
}
inline size_t log_probs_bytes(int R, int V, int bytes, int K) { return (size_t)R * row_parts(R, V, bytes) * (K * sizeof(u64) + sizeof(Stat)); }

// Gradients: a wave takes about 8 KiB of scores, less where that leaves waves to spare.  (2048 rows of 131072, bf16, log probabilities:
// 195 us with 4 KiB, 181 with 8, 193 with 16, 222 with 64; 8192 rows of 2500: 18.4, 16.9, 16.9, 16.9; one row of 131072: 3.0, 8.4 without the
// second rule.)
inline int grad_waves(int R, int V, int bytes) {
  const long long by_size = ((long long)V * bytes + 8191) / 8192, steps = (long long)V * bytes / 1024;
  const long long fill = (4096 + R - 1) / R, n = by_size > fill ? by_size : fill;
  return (int)(n < 1 || steps < 1 ? 1 : n > steps ? steps : n);
}

// A gradient beyond half of the 256 MB of the last-level cache is written past it: left there, its lines are written back while the
// next pass over scores reads (distillation and its gradient, 2048 rows of 131072 bf16 scores, 538 MB: 310 us instead of 281).
inline bool streams(const RowsArgs &a, int bytes) { return (long long)a.R * a.V * bytes > (128ll << 20); }

// Two rows a wave where they are short and many enough to fill the chip, and one lane is enough for each entry of their lists.  fp32, us
// for the sums / with 8 alternatives / distillation: 8192 rows of 1000: 7.5 / 13.4 / 8.2 against 8.2 / 17.3 / 10.0 with one; 30000 of 200:
// 7.9 / 21 / 12.8 against 13.0 / 39 / 22.6; 3000 of 2047: 8.0 / 14.9 / 8.2 against 5.8 / 10.5 / 6.2; bf16, 2048 of 1000: 3.8 / 7.3 / 4.3 against
// 4.1 / 8.0 / 4.5.
inline bool two_rows(int R, int V, int lists, int bytes) {
  const long long size = (long long)V * bytes;
  return R >= 2048 && size <= 6144 && 2 * size <= 3ll * R && lists <= 32;
}

// fp32 gradients: short rows that a wave has to itself are kept in its registers
inline bool keeps(const RowsArgs &a) { return a.V <= kShort && a.per_row == 1; }

template <typename T> hipError_t launch_log_probs(const RowsArgs &a, hipStream_t st) {
  if (a.parts) {
    auto part = a.K ? log_probs_part_kernel<T, true> : log_probs_part_kernel<T, false>;
    auto join = a.K ? log_probs_join_kernel<T, true> : log_probs_join_kernel<T, false>;
    hipLaunchKernelGGL(part, dim3(a.R * a.parts), dim3(256), 0, st, a);
    const hipError_t rc = hipGetLastError();
    if (rc != hipSuccess) return rc;
    hipLaunchKernelGGL(join, dim3(a.R), dim3(256), 0, st, a);
    return hipGetLastError();
  }
  const int W = row_waves(a.R, a.V, sizeof(T));
  const bool two = two_rows(a.R, a.V, a.K > a.N ? a.K : a.N, sizeof(T));
  const dim3 grid(W > 1 ? a.R : two ? (a.R + 7) / 8 : (a.R + 3) / 4), block(W == 16 ? 1024 : 256);
  auto kernel = two ? (a.K ? log_probs_kernel<T, 1, 32, true> : log_probs_kernel<T, 1, 32, false>)
              : W == 1 ? (a.K ? log_probs_kernel<T, 1, 64, true> : log_probs_kernel<T, 1, 64, false>)
              : W == 4 ? (a.K ? log_probs_kernel<T, 4, 64, true> : log_probs_kernel<T, 4, 64, false>)
                       : (a.K ? log_probs_kernel<T, 16, 64, true> : log_probs_kernel<T, 16, 64, false>);
  hipLaunchKernelGGL(kernel, grid, block, 0, st, a);
  return hipGetLastError();
}
template <typename T> hipError_t launch_distill(const RowsArgs &a, bool tail, hipStream_t st) {
  const int W = row_waves(a.R, a.V, sizeof(T));
  const bool two = two_rows(a.R, a.V, a.K, sizeof(T));
  const dim3 grid(W > 1 ? a.R : two ? (a.R + 7) / 8 : (a.R + 3) / 4), block(W == 16 ? 1024 : 256);
  auto kernel = two ? (tail ? distill_kernel<T, 1, 32, true> : distill_kernel<T, 1, 32, false>)
              : W == 1 ? (tail ? distill_kernel<T, 1, 64, true> : distill_kernel<T, 1, 64, false>)
              : W == 4 ? (tail ? distill_kernel<T, 4, 64, true> : distill_kernel<T, 4, 64, false>)
                       : (tail ? distill_kernel<T, 16, 64, true> : distill_kernel<T, 16, 64, false>);
  hipLaunchKernelGGL(kernel, grid, block, 0, st, a);
  return hipGetLastError();
}
template <typename T> hipError_t launch_log_probs_backward(RowsArgs a, hipStream_t st) {
  a.per_row = grad_waves(a.R, a.V, sizeof(T));
  const bool far = streams(a, sizeof(T));
  const dim3 grid((unsigned)(((long long)a.R * a.per_row + 3) / 4));
  auto kernel = a.g2 ? (far ? log_probs_backward_kernel<T, true, true, false> : log_probs_backward_kernel<T, true, false, false>)
                     : (far ? log_probs_backward_kernel<T, false, true, false> : log_probs_backward_kernel<T, false, false, false>);
  if constexpr (sizeof(T) == 4)
    if (keeps(a))
      kernel = a.g2 ? (far ? log_probs_backward_kernel<T, true, true, true> : log_probs_backward_kernel<T, true, false, true>)
                    : (far ? log_probs_backward_kernel<T, false, true, true> : log_probs_backward_kernel<T, false, false, true>);
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}
template <typename T> hipError_t launch_distill_backward(RowsArgs a, bool tail, hipStream_t st) {
  a.per_row = grad_waves(a.R, a.V, sizeof(T));
  const bool far = streams(a, sizeof(T));
  const dim3 grid((unsigned)(((long long)a.R * a.per_row + 3) / 4));
  auto kernel = tail ? (far ? distill_backward_kernel<T, true, true, false> : distill_backward_kernel<T, true, false, false>)
                     : (far ? distill_backward_kernel<T, false, true, false> : distill_backward_kernel<T, false, false, false>);
  if constexpr (sizeof(T) == 4)
    if (keeps(a))
      kernel = tail ? (far ? distill_backward_kernel<T, true, true, true> : distill_backward_kernel<T, true, false, true>)
                    : (far ? distill_backward_kernel<T, false, true, true> : distill_backward_kernel<T, false, false, true>);
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace urf
using namespace urf;

namespace {

#define URF_BY_TYPE(dtype, f, ...) \
  ((dtype) == URF_F32 ? f<float>(__VA_ARGS__) : (dtype) == URF_F16 ? f<_Float16>(__VA_ARGS__) : f<__bf16>(__VA_ARGS__))

int check_config(const urf_rows_config *c, const char *who) {
  URF_CHECK(c, "%s: null configuration", who);
  URF_CHECK(dtype_bytes(c->dtype), "%s: element type %d (URF_F32, URF_F16 or URF_BF16)", who, c->dtype);
  // a workgroup per row, and a launch takes fewer than 2^24 of them (of 256 threads)
  URF_CHECK(c->rows >= 0 && c->rows < (1 << 24) && c->classes >= 1 && c->classes <= (1 << 30), "%s: %d rows of %d classes", who, c->rows, c->classes);
  URF_CHECK(c->scale > 0.0f && c->scale < 0x1p127f, "%s: scale %g (positive)", who, (double)c->scale);      // (times log2(e) it is still finite)
  return 0;
}

// rows that far apart are still within 64 bits of bytes
bool stride_fits(long long stride, int rows) {
  const long long most = (1ll << 59) / (rows > 1 ? rows : 1);
  return rows <= 1 || (stride > -most && stride < most);
}

int check_rows(const urf_rows_config *c, const void *logits, const char *who) {
  if (check_config(c, who)) return -2;
  URF_CHECK(stride_fits(c->row_stride, c->rows), "%s: rows %lld elements apart", who, c->row_stride);
  URF_CHECK(c->rows == 0 || logits, "%s: logits is null", who);
  URF_CHECK(((uintptr_t)logits & (dtype_bytes(c->dtype) - 1)) == 0, "%s: logits is not aligned to its elements", who);
  return 0;
}

// the gradient's rows may not touch each other or the logits
int check_grad(const urf_rows_config *c, const void *logits, const void *d, long long stride, const char *who) {
  URF_CHECK(c->rows == 0 || d, "%s: d_logits is null", who);
  const long long b = dtype_bytes(c->dtype);
  URF_CHECK(((uintptr_t)d & (b - 1)) == 0, "%s: d_logits is not aligned to its elements", who);
  URF_CHECK(stride_fits(stride, c->rows), "%s: rows of d_logits %lld elements apart", who, stride);
  URF_CHECK(c->rows <= 1 || stride >= c->classes, "%s: the rows of d_logits overlap (stride %lld, %d classes)", who, stride, c->classes);
  if (c->rows == 0) return 0;
  const long long in = c->row_stride * (c->rows - 1), n = c->classes;
  const char *z = (const char *)logits, *z0 = z + (in < 0 ? in : 0) * b, *z1 = z + ((in > 0 ? in : 0) + n) * b;
  const char *d0 = (const char *)d, *d1 = d0 + (stride * (c->rows - 1) + n) * b;
  URF_CHECK(d1 <= z0 || z1 <= d0, "%s: d_logits overlaps the logits", who);
  return 0;
}

RowsArgs rows_of(const urf_rows_config *c, const void *logits) {
  RowsArgs a = {};
  a.z = logits;
  a.stride = c->row_stride;
  a.R = c->rows;
  a.V = c->classes;
  a.scale = c->scale;
  a.c = (float)((double)c->scale * kLog2eDouble);
  return a;
}

}  // namespace

static int check_top(const urf_rows_config *cfg, int top, const char *who) {
  URF_CHECK(top >= 0 && top <= URF_TOP_MAX && top <= cfg->classes, "%s: %d alternatives (0 .. %d, at most the %d classes)", who, top, URF_TOP_MAX, cfg->classes);
  return 0;
}

extern "C" int urf_log_probs_workspace(const urf_rows_config *cfg, int top, size_t *bytes) {
  const char *who = "urf_log_probs_workspace";
  if (check_config(cfg, who) || check_top(cfg, top, who)) return -2;
  URF_CHECK(bytes, "%s: null pointer", who);
  *bytes = cfg->rows ? log_probs_bytes(cfg->rows, cfg->classes, dtype_bytes(cfg->dtype), top) : 0;
  return 0;
}

extern "C" int urf_log_probs(const urf_rows_config *cfg, const void *logits, const int *d_targets, int n_targets, int top,
                             float *d_log_prob, float *d_entropy, float *d_lse, int *d_top_index, float *d_top_log_prob, void *d_work,
                             size_t work_bytes, void *stream) {
  const char *who = "urf_log_probs";
  if (check_rows(cfg, logits, who) || check_top(cfg, top, who)) return -2;
  URF_CHECK(n_targets >= 0 && n_targets <= URF_TOP_MAX, "%s: %d targets per row (0 .. %d)", who, n_targets, URF_TOP_MAX);
  if (cfg->rows == 0) return 0;
  const size_t need = log_probs_bytes(cfg->rows, cfg->classes, dtype_bytes(cfg->dtype), top);
  URF_CHECK(need == 0 || (d_work && work_bytes >= need && ((uintptr_t)d_work & 15) == 0), "%s: workspace of %zu bytes, %zu needed", who, work_bytes, need);
  URF_CHECK(d_entropy && d_lse && (n_targets == 0 || (d_targets && d_log_prob)) && (top == 0 || (d_top_index && d_top_log_prob)), "%s: null pointer", who);
  RowsArgs a = rows_of(cfg, logits);
  a.targets = d_targets; a.N = n_targets; a.K = top;
  a.log_prob = d_log_prob; a.entropy = d_entropy; a.lse = d_lse; a.top_index = d_top_index; a.top_log_prob = d_top_log_prob;
  a.parts = row_parts(cfg->rows, cfg->classes, dtype_bytes(cfg->dtype));
  a.part_keys = (u64 *)d_work;
  a.part_stats = (Stat *)(a.part_keys + (size_t)cfg->rows * a.parts * top);
  OnDevice on(cfg->device);
  URF_HIP(on.rc);
  URF_HIP(URF_BY_TYPE(cfg->dtype, launch_log_probs, a, (hipStream_t)stream));
  return 0;
}

extern "C" int urf_log_probs_backward(const urf_rows_config *cfg, const void *logits, const int *d_targets, int n_targets,
                                      const float *d_lse, const float *d_entropy, const float *d_d_log_prob,
                                      const float *d_d_entropy, void *d_logits, long long d_logits_stride, void *stream) {
  const char *who = "urf_log_probs_backward";
  if (check_rows(cfg, logits, who) || check_grad(cfg, logits, d_logits, d_logits_stride, who)) return -2;
  URF_CHECK(n_targets >= 0 && n_targets <= URF_TOP_MAX, "%s: %d targets per row (0 .. %d)", who, n_targets, URF_TOP_MAX);
  if (cfg->rows == 0) return 0;
  URF_CHECK(d_lse && (n_targets == 0 || (d_targets && d_d_log_prob)) && (!d_d_entropy || d_entropy), "%s: null pointer", who);
  RowsArgs a = rows_of(cfg, logits);
  a.targets = d_targets; a.N = n_targets;
  a.lse = (float *)d_lse; a.entropy = (float *)d_entropy; a.g1 = d_d_log_prob; a.g2 = d_d_entropy;
  a.dz = d_logits; a.dz_stride = d_logits_stride;
  OnDevice on(cfg->device);
  URF_HIP(on.rc);
  URF_HIP(URF_BY_TYPE(cfg->dtype, launch_log_probs_backward, a, (hipStream_t)stream));
  return 0;
}

static int distill_args(const urf_rows_config *cfg, const void *logits, const int *d_index, const float *d_value, int listed, int tail,
                        const char *who, RowsArgs *a) {
  if (check_rows(cfg, logits, who)) return -2;
  URF_CHECK(listed >= 1 && listed <= URF_TOP_MAX, "%s: %d listed alternatives (1 .. %d)", who, listed, URF_TOP_MAX);
  URF_CHECK(cfg->rows == 0 || (d_index && d_value), "%s: the teacher's alternatives are null", who);
  *a = rows_of(cfg, logits);
  a->t_index = d_index; a->t_value = d_value; a->K = listed;
  return 0;
}

extern "C" int urf_distill(const urf_rows_config *cfg, const void *logits, const int *d_index, const float *d_value, int listed,
                           int tail, float *d_loss, float *d_lse, float *d_log_tail, void *stream) {
  const char *who = "urf_distill";
  RowsArgs a;
  if (distill_args(cfg, logits, d_index, d_value, listed, tail, who, &a)) return -2;
  if (cfg->rows == 0) return 0;
  URF_CHECK(d_loss && d_lse && (!tail || d_log_tail), "%s: null pointer", who);
  a.loss = d_loss; a.lse = d_lse; a.log_tail = d_log_tail;
  OnDevice on(cfg->device);
  URF_HIP(on.rc);
  URF_HIP(URF_BY_TYPE(cfg->dtype, launch_distill, a, tail != 0, (hipStream_t)stream));
  return 0;
}

extern "C" int urf_distill_backward(const urf_rows_config *cfg, const void *logits, const int *d_index, const float *d_value, int listed,
                                    int tail, const float *d_lse, const float *d_log_tail, const float *d_d_loss, void *d_logits,
                                    long long d_logits_stride, void *stream) {
  const char *who = "urf_distill_backward";
  RowsArgs a;
  if (distill_args(cfg, logits, d_index, d_value, listed, tail, who, &a) || check_grad(cfg, logits, d_logits, d_logits_stride, who)) return -2;
  if (cfg->rows == 0) return 0;
  URF_CHECK(d_lse && d_d_loss && (!tail || d_log_tail), "%s: null pointer", who);
  a.lse = (float *)d_lse; a.log_tail = (float *)d_log_tail; a.g1 = d_d_loss;
  a.dz = d_logits; a.dz_stride = d_logits_stride;
  OnDevice on(cfg->device);
  URF_HIP(on.rc);
  URF_HIP(URF_BY_TYPE(cfg->dtype, launch_distill_backward, a, tail != 0, (hipStream_t)stream));
  return 0;
}
