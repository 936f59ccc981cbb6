// attention_api.hip -- the attention operator behind the C ABI: argument checks, the choice of the forward kernel's shape, the
// workspace.  The kernels: attention_op.h.
#include "attention_op.h"

#include <math.h>

#include <algorithm>

namespace urf {
hipError_t attn_forward_f32(const AttnArgs &, int, hipStream_t);
hipError_t attn_forward_f16(const AttnArgs &, int, hipStream_t);
hipError_t attn_forward_bf16(const AttnArgs &, int, hipStream_t);
hipError_t attn_backward_f32(const AttnArgs &, hipStream_t);
hipError_t attn_backward_f16(const AttnArgs &, hipStream_t);
hipError_t attn_backward_bf16(const AttnArgs &, hipStream_t);
}  // namespace urf
using namespace urf;

namespace {

struct Shape { int narrow, splits; };

// How the forward pass is cut.  128-row workgroups read the keys least often; where they are fewer than the 256 CUs, 32-row
// workgroups whose waves share the keys (8 x 4 heads of 1024 x 1024 x 64, bf16: 23 us with 256 of the former, 30 with 1024 of the latter; 2 x 4
// heads: 21 and 12.4); where those are fewer as well, the keys are split until there are two workgroups per CU, at least 256 keys each.  The
// join costs some 3 us and grows with the rows, so that short keys are left whole (1 x 4 heads of 1000 x 1000 x 64: 13.8 us in four ranges, 12.7
// whole; 512 x 512: 11.0 and 8.4; one row of 1 x 32 heads over 1000 keys: 9.2 and 12.8; fp32, whose products take longer, 512 x 512: 15.3 and
// 17.4).  Up to 32 rows (one token, some heads) over many keys their bytes are all there is: eight workgroups per CU even out lengths and
// keep loads in flight, at least 1024 keys each (32 sequences of up to 16384 keys, 8 key heads of 128, bf16: 427 us in 128-row workgroups, 344
// in 32-row ones, 320, 303 and 290 with 512, 1024 and 2048 of them; 64 sequences of 1000: 30 us with 2048, 18 with 512).
Shape forward_shape(const urf_attn_config &c) {
  const long long rows = (long long)c.q_len * (c.q_heads / c.kv_heads), groups = (long long)c.batch * c.kv_heads;
  const bool few = rows <= 32;
  if (!few && (rows + 127) / 128 * groups >= 256) return {0, 1};
  const long long blocks = (rows + 31) / 32 * groups;
  if ((!few && blocks >= 256) || c.k_len < (few || c.dtype == URF_F32 ? 512 : 1024)) return {1, 1};
  long long s = std::min<long long>((c.k_len + 255) / 256, (512 + blocks - 1) / blocks);
  if (few) s = std::max(s, std::min<long long>(c.k_len / 1024, (2048 + blocks - 1) / blocks));
  return {1, (int)std::min<long long>(std::max<long long>(s, 1), 64)};
}

size_t padded_dim(const urf_attn_config &c) { return ((size_t)c.head_dim + 31) / 32 * 32; }

size_t forward_bytes(const urf_attn_config &c) {
  const Shape sh = forward_shape(c);
  if (sh.splits == 1) return 0;
  const size_t rows = (size_t)c.q_len * c.q_heads * c.batch * sh.splits;
  return rows * (padded_dim(c) + 2) * sizeof(float);
}

// How the backward kernel is cut: 128 keys (or rows) a workgroup, over all rows (keys) or over `splits` ranges of them whose partial
// sums are added in fp32 afterwards.  Chosen by an estimate of its time, in ns: a workgroup's product of one row with its 128 keys
// takes 0.17 (16 bits) or 1.4 (fp32) per element of the head with two workgroups on every CU (four products for dk and dv, three for
// dq), a range costs two steps of 32 rows to begin with, and its partial sums are written and read at 4.7 TB/s.  Whole against this
// choice, us: 1 x 8 heads over 2 key heads of 4096 x 4096 x 64, bf16: 420, 165; 3 x 6 over 2 of 517 x 1333 x 128: 113, 59; 2 x 16 heads of 2048 x 2048 x 64:
// 153, 147; fp32, 4 x 4 heads of 1000 x 1000 x 64: 160, 138; 8 x 4 of 1024 x 1024: 242, 258.
void backward_shape(const urf_attn_config &c, int *kv_splits, int *q_splits) {
  const double rows = (double)c.q_len * (c.q_heads / c.kv_heads), keys = c.k_len, groups = (double)c.batch * c.kv_heads;
  const double dim = (c.head_dim + 31) / 32 * 32, step = dim * (c.dtype == URF_F32 ? 1.4 : 0.17), part = dim * 8 / 4700.0;
  const double kv_tiles = ceil(keys / 128), q_tiles = ceil(rows / 128), share = c.causal ? 0.5 : 1.0;
  double best = INFINITY;
  *kv_splits = *q_splits = 1;
  for (int k = 1; k <= 16 && (k == 1 || rows / k >= 64); ++k)
    for (int q = 1; q <= 16 && (q == 1 || keys / q >= 64); ++q) {
      const double units = groups * (kv_tiles * k + q_tiles * q), largest = step * fmax(4 * (rows / k + 64), 3 * (keys / q + 64));
      const double all = step * groups * (kv_tiles * 4 * (rows * share + 64 * k) + q_tiles * 3 * (keys * share + 64 * q));
      // equal units fill whole rounds of the 512 places; uneven ones (a causal mask's) even out
      const double rounds = c.causal ? all / 512 : ceil(units / 512) * (all / units);
      const double parts = (k > 1 ? 2 * k * groups * keys * part : 0.0) + (q > 1 ? q * groups * rows * part : 0.0) + (k > 1 || q > 1 ? 3000.0 : 0.0);
      const double t = fmax(largest, rounds) + parts;
      if (t < best) { best = t; *kv_splits = k; *q_splits = q; }
    }
}

size_t floats(size_t n) { return (n * sizeof(float) + 15) / 16 * 16; }
size_t delta_bytes(const urf_attn_config &c) { return floats((size_t)c.batch * c.q_heads * c.q_len); }
size_t norm_v_bytes(const urf_attn_config &c) { return floats((size_t)c.batch * c.kv_heads * c.k_len); }

// delta, f16: the norms of do's and v's rows, the parts of dk and dv, the parts of dq
size_t stat_bytes(const urf_attn_config &c) { return c.dtype == URF_F16 ? 2 * delta_bytes(c) + norm_v_bytes(c) : delta_bytes(c); }
size_t part_kv_bytes(const urf_attn_config &c, int splits) {
  return splits > 1 ? 2 * (size_t)splits * c.batch * c.kv_heads * c.k_len * padded_dim(c) * sizeof(float) : 0;
}
size_t part_q_bytes(const urf_attn_config &c, int splits) {
  return splits > 1 ? (size_t)splits * c.batch * c.q_heads * c.q_len * padded_dim(c) * sizeof(float) : 0;
}
size_t backward_bytes(const urf_attn_config &c, int kv, int q) { return stat_bytes(c) + part_kv_bytes(c, kv) + part_q_bytes(c, q); }

int check_config(const urf_attn_config *c, const char *who) {
  URF_CHECK(c, "%s: null configuration", who);
  URF_CHECK(dtype_bytes(c->dtype), "%s: element type %d (URF_F32, URF_F16 or URF_BF16)", who, c->dtype);
  URF_CHECK(c->batch >= 1 && c->q_len >= 1 && c->k_len >= 0, "%s: batch %d, %d rows, %d keys", who, c->batch, c->q_len, c->k_len);
  URF_CHECK(c->kv_heads >= 1 && c->q_heads >= 1 && c->q_heads % c->kv_heads == 0, "%s: %d query heads over %d key heads", who, c->q_heads, c->kv_heads);
  URF_CHECK(c->head_dim >= 8 && c->head_dim <= 128 && c->head_dim % 8 == 0, "%s: head size %d (a multiple of 8 up to 128)", who, c->head_dim);
  URF_CHECK(c->scale >= 0.0f && c->scale < 0x1p127f, "%s: scale %g", who, (double)c->scale);      // (times log2(e) it is still finite)
  // row and key indices are 32-bit, element offsets 64-bit; a launch takes fewer than 2^24 workgroups of 256 threads
  const long long most = 1ll << 23, rows = (long long)c->q_len * (c->q_heads / c->kv_heads);
  const bool few = (long long)c->batch * c->q_heads < most;
  const long long groups = few ? (long long)c->batch * c->kv_heads : most;
  URF_CHECK(few && rows < most * 32 && groups * ((rows + 31) / 32) < most && groups * (((long long)c->k_len + 31) / 32) < most &&
            (long long)c->batch * c->q_heads * c->q_len < most * 16, "%s: too many rows, keys or heads", who);
  return 0;
}

// `len` rows; without any there is nothing to point to
int check_tensor(const urf_attn_tensor *t, const urf_attn_config *c, int len, const char *who, const char *name) {
  URF_CHECK(t && (t->data || len == 0), "%s: %s is null", who, name);
  const long long per = 16 / dtype_bytes(c->dtype);
  URF_CHECK(((uintptr_t)t->data & 15) == 0 && t->batch_stride % per == 0 && t->row_stride % per == 0 && t->head_stride % per == 0,
            "%s: %s: base and strides have to be multiples of 16 bytes", who, name);
  return 0;
}

int check_out(const urf_attn_tensor *t, const urf_attn_config *c, int len, int heads, const char *who, const char *name) {
  if (check_tensor(t, c, len, who, name)) return -2;
  if (len == 0) return 0;
  // two elements of an output may not share memory: each dimension, from the smallest stride up, steps over all that is below it
  struct { long long stride, n; } dim[3] = {{llabs(t->batch_stride), c->batch}, {llabs(t->row_stride), len}, {llabs(t->head_stride), heads}};
  std::sort(dim, dim + 3, [](const auto &x, const auto &y) { return x.stride < y.stride; });
  long long extent = c->head_dim;
  for (const auto &d : dim) {
    if (d.n <= 1) continue;
    URF_CHECK(d.stride >= extent && d.stride < (1ll << 60) / d.n, "%s: the rows of output %s overlap", who, name);
    extent += d.stride * (d.n - 1);
  }
  return 0;
}

AttnView view(const urf_attn_tensor *t) { return {t->data, t->batch_stride, t->row_stride, t->head_stride}; }

AttnArgs args_of(const urf_attn_config *c, const urf_attn_tensor *q, const urf_attn_tensor *k, const urf_attn_tensor *v, const int *d_q_lens, const int *d_k_lens) {
  AttnArgs a = {};
  a.q = view(q); a.k = view(k); a.v = view(v);
  a.q_lens = d_q_lens; a.k_lens = d_k_lens;
  a.B = c->batch; a.Hq = c->q_heads; a.Hk = c->kv_heads; a.G = c->q_heads / c->kv_heads;
  a.Lq = c->q_len; a.Lk = c->k_len; a.D = c->head_dim; a.causal = c->causal != 0; a.splits = 1;
  a.scale = c->scale > 0.0f ? c->scale : 1.0f / sqrtf((float)c->head_dim);
  a.scale2 = (float)((double)a.scale * 1.4426950408889634);
  return a;
}

}  // namespace

extern "C" int urf_attn_workspace(const urf_attn_config *cfg, int backward, size_t *bytes) {
  if (check_config(cfg, "urf_attn_workspace")) return -2;
  URF_CHECK(bytes, "urf_attn_workspace: null pointer");
  int kv = 1, q = 1;
  if (backward) backward_shape(*cfg, &kv, &q);
  *bytes = backward ? backward_bytes(*cfg, kv, q) : forward_bytes(*cfg);
  return 0;
}

extern "C" int urf_attn_forward(const urf_attn_config *cfg, const urf_attn_tensor *q, const urf_attn_tensor *k, const urf_attn_tensor *v,
                                const int *d_q_lens, const int *d_k_lens, const urf_attn_tensor *o, float *d_lse, void *d_work,
                                size_t work_bytes, void *stream) {
  const char *who = "urf_attn_forward";
  if (check_config(cfg, who) || check_tensor(q, cfg, cfg->q_len, who, "q") || check_tensor(k, cfg, cfg->k_len, who, "k") || check_tensor(v, cfg, cfg->k_len, who, "v") ||
      check_out(o, cfg, cfg->q_len, cfg->q_heads, who, "o")) return -2;
  URF_CHECK(d_lse, "%s: lse is null", who);
  URF_CHECK(o->data != q->data && o->data != k->data && o->data != v->data, "%s: o may not be an input", who);
  const size_t need = forward_bytes(*cfg);
  URF_CHECK(need == 0 || (d_work && work_bytes >= need && ((uintptr_t)d_work & 15) == 0), "%s: workspace of %zu bytes, %zu needed", who, work_bytes, need);
  const Shape sh = forward_shape(*cfg);
  AttnArgs a = args_of(cfg, q, k, v, d_q_lens, d_k_lens);
  a.o = view(o);
  a.lse = d_lse;
  a.splits = sh.splits;
  if (sh.splits > 1) {
    const size_t rows = (size_t)a.Lq * a.Hq * a.B * sh.splits;
    a.part_o = (float *)d_work;
    a.part_ml = a.part_o + rows * padded_dim(*cfg);
  }
  OnDevice on(cfg->device);
  URF_HIP(on.rc);
  const hipStream_t st = (hipStream_t)stream;
  URF_HIP(cfg->dtype == URF_F32 ? attn_forward_f32(a, sh.narrow, st) : cfg->dtype == URF_F16 ? attn_forward_f16(a, sh.narrow, st) : attn_forward_bf16(a, sh.narrow, st));
  return 0;
}

extern "C" int urf_attn_backward(const urf_attn_config *cfg, const urf_attn_tensor *q, const urf_attn_tensor *k, const urf_attn_tensor *v,
                                 const urf_attn_tensor *o, const float *d_lse, const urf_attn_tensor *d_o, const int *d_q_lens,
                                 const int *d_k_lens, const urf_attn_tensor *dq, const urf_attn_tensor *dk, const urf_attn_tensor *dv,
                                 void *d_work, size_t work_bytes, void *stream) {
  const char *who = "urf_attn_backward";
  if (check_config(cfg, who) || check_tensor(q, cfg, cfg->q_len, who, "q") || check_tensor(k, cfg, cfg->k_len, who, "k") || check_tensor(v, cfg, cfg->k_len, who, "v") ||
      check_tensor(o, cfg, cfg->q_len, who, "o") || check_tensor(d_o, cfg, cfg->q_len, who, "the gradient of o") || check_out(dq, cfg, cfg->q_len, cfg->q_heads, who, "dq") ||
      check_out(dk, cfg, cfg->k_len, cfg->kv_heads, who, "dk") || check_out(dv, cfg, cfg->k_len, cfg->kv_heads, who, "dv")) return -2;
  URF_CHECK(d_lse, "%s: lse is null", who);
  const void *in[5] = {q->data, k->data, v->data, o->data, d_o->data}, *out[3] = {dq->data, dk->data, dv->data};
  for (int x = 0; x < 3; ++x) {
    for (int y = 0; y < 5; ++y) URF_CHECK(!out[x] || out[x] != in[y], "%s: an output may not be an input", who);
    for (int y = 0; y < x; ++y) URF_CHECK(!out[x] || out[x] != out[y], "%s: two outputs share a base", who);
  }
  int kv_splits, q_splits;
  backward_shape(*cfg, &kv_splits, &q_splits);
  const size_t need = backward_bytes(*cfg, kv_splits, q_splits);
  URF_CHECK(d_work && work_bytes >= need && ((uintptr_t)d_work & 15) == 0, "%s: workspace of %zu bytes, %zu needed", who, work_bytes, need);
  AttnArgs a = args_of(cfg, q, k, v, d_q_lens, d_k_lens);
  a.o = view(o); a.dout = view(d_o); a.dq = view(dq); a.dk = view(dk); a.dv = view(dv);
  a.lse = (float *)d_lse;
  a.delta = (float *)d_work;
  a.kv_splits = kv_splits; a.q_splits = q_splits;
  a.norm_do = (float *)((char *)d_work + delta_bytes(*cfg));
  a.norm_v = (float *)((char *)a.norm_do + delta_bytes(*cfg));
  a.part_kv = (float *)((char *)d_work + stat_bytes(*cfg));
  a.part_q = (float *)((char *)a.part_kv + part_kv_bytes(*cfg, a.kv_splits));
  OnDevice on(cfg->device);
  URF_HIP(on.rc);
  const hipStream_t st = (hipStream_t)stream;
  URF_HIP(cfg->dtype == URF_F32 ? attn_backward_f32(a, st) : cfg->dtype == URF_F16 ? attn_backward_f16(a, st) : attn_backward_bf16(a, st));
  return 0;
}
